// narrow_ce.hip -- linear_ce.hip's loss for a head of few outputs (action bins of an agent): up to 32
// outputs of 128 hidden elements, or 64 of 64.
//
// One kernel reads each hidden row once and writes its gradient once.  The weight is in LDS.  A wave
// takes 32 rows: z = W h^T has a row in a lane, sixteen outputs of it in either half of the wave, so
// the softmax is in registers; G = p - [target] is an operand of d h^T = W^T G^T as it lies, and goes
// through LDS to be one of d W = G^T h, whose sums stay in the wave's registers to the end.  A second
// kernel adds the workgroups' sums, in their order.
// bfloat16: G goes into both as two terms, 16 bits, so that what the gradients are off by is their own
// rounding (256000 x 64 x 25: d h 1.66e-3 of its size, 2.07e-3 with one term, and 1 us of 50).  The biases are in
// LDS to make room for that: with them in registers the wider heads spilled (256000 x 64 x 60: 89 us,
// now 76; float16 245, 155).
// Three products of 2 rows dim width operations: far below what the rows cost to read and write.
// 256000 rows of 64, 25 outputs, bfloat16: 34 us of the rows' kernel and 5 of adding up 512 workgroups' sums,
// 69 MB in all (14 us): what is left is a wave's chain through 32 rows, four of them each, and its first ones.
#include <math.h>

#include "narrow_ce.hpp"
#include "parts.hpp"

namespace {

using namespace part;
using learn::fail;
using learn::launched;
using learn::up;
using learn::wave_sum;

constexpr int BLOCK = 256, WAVES = BLOCK / 64, ROWS = 32;
constexpr int MOST_BLOCKS = 512;  // of the rows' kernel: two a compute unit, each leaves one set of sums
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN_2 = 0.69314718055994530942f;

struct Head {
    int64_t rows, inner, outer_stride, inner_stride;
    int dim, width, targets32, sum, skip_unit;
    const void *hidden, *weight, *bias, *targets;
    const uint8_t *mask;
    const int32_t *counts;
    int n_counts;
    const float *scale;    // upstream gradient, or NULL: 1
    float *logp, *loss;    // or NULL
    void *d_hidden;        // or NULL
    void *d_weight, *d_bias;
    float *sums;           // [grid][width * dim + width], or NULL: no gradient of the weight or the bias
    double *losses;        // [grid]
};

// What is multiplied: bfloat16, or float.
template <typename T> struct Mul { typedef float type; };
template <> struct Mul<bf16> { typedef bf16 type; };

template <typename T> __device__ __forceinline__ Part<typename Mul<T>::type> mul_of(const Part<T> &p)
{
    if constexpr (sizeof(Part<T>) == sizeof(Part<typename Mul<T>::type>)) return __builtin_bit_cast(Part<typename Mul<T>::type>, p);
}

// Rows that count, the same in every thread.
__device__ int64_t counted(const Head &c)
{
    if (!c.mask) return c.rows;
    __shared__ int64_t n;
    if (threadIdx.x < 64) {
        int64_t s = 0;
        for (int i = threadIdx.x; i < c.n_counts; i += 64) s += c.counts[i];
        s = wave_sum(s);
        if (threadIdx.x == 0) n = s;
    }
    __syncthreads();
    return n;
}
__device__ __forceinline__ bool skipped(const Head &c) { return c.skip_unit && *c.scale == 1.0f; }

template <typename T, int VT, int KT, int FIT> __global__ __launch_bounds__(BLOCK, 2) void k_rows(const Head c)
{
    typedef typename Mul<T>::type M;
    constexpr int KP = 32 * KT + 16 / (int)sizeof(T), GP = 32 * VT + 16 / (int)sizeof(M);
    constexpr int TERMS = Part<M>::TERMS ? 2 : 1;  // of G
    constexpr int EACH = 32 * (KP * (int)sizeof(T) + TERMS * GP * (int)sizeof(M));  // bytes of a wave
    constexpr int SUMS = 32 * VT * 32 * KT * 4, ROOM = WAVES * EACH;
    __shared__ __align__(16) T wx[32 * VT * KP];
    __shared__ __align__(16) char room[ROOM > SUMS ? ROOM : SUMS];
    __shared__ double red[WAVES];
    __shared__ __align__(16) float bx[32 * VT];
    if (skipped(c)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31, perm = swapped(col);
    const int D = c.dim, V = c.width;
    for (int x = threadIdx.x; x < 32 * VT * KP; x += BLOCK) {
        const int v = x / KP, d = x % KP;
        wx[x] = v < V && d < D ? ((const T *)c.weight)[v * D + d] : (T)0.0f;
    }
    // (those past the last output are -inf)
    if (threadIdx.x < 32 * VT)
        bx[threadIdx.x] = (int)threadIdx.x >= V ? -INFINITY : c.bias ? up(((const T *)c.bias)[threadIdx.x]) : 0.0f;
    const int64_t n_on = counted(c);
    const float up1 = c.scale ? *c.scale : 1.0f;
    const float weight = c.sum ? up1 : (float)((double)up1 / (double)(n_on > 1 ? n_on : 1));
    __syncthreads();
    T *const hx = (T *)(room + wave * EACH);
    M *const gx = (M *)(hx + 32 * KP);
    const bool grads = c.sums != nullptr;

    // register r of tile a is output 32 a + 16 (r / 8) + 8 half + r % 8
    f32x16 dw[VT][KT];
    float db[VT][16];
#pragma unroll
    for (int a = 0; a < VT; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            db[a][r] = 0.0f;
#pragma unroll
            for (int t = 0; t < KT; ++t) dw[a][t][r] = 0.0f;
        }
    double loss = 0.0;

    const int64_t tiles = (c.rows + ROWS - 1) / ROWS, step = (int64_t)gridDim.x * WAVES;
    int64_t tile = (int64_t)blockIdx.x * WAVES + wave;
    // a row of the next tile, its target and whether it counts; where it does not the first row is
    // read in its place, and taken as zeros
    Raw<T> hr[2 * KT];
    int64_t target = 0;
    bool on = false;
    auto load = [&](int64_t tile) {
        const int64_t i = tile * ROWS + col;
        on = i < c.rows && (!c.mask || c.mask[i]);
        const int64_t row = on ? i : 0;
        target = c.targets32 ? (int64_t)((const int32_t *)c.targets)[row] : ((const int64_t *)c.targets)[row];
        const uint32_t o = (uint64_t)c.inner >= (uint64_t)c.rows ? 0 : (uint32_t)((uint32_t)row / (uint32_t)c.inner);
        const T *const x = (const T *)c.hidden + o * c.outer_stride + (row - o * c.inner) * c.inner_stride;
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) hr[t] = row_of<T, FIT>(x, 16 * t + 8 * half, D, true);
    };
    if (tile < tiles) load(tile);
    for (; tile < tiles; tile += step) {
        const int64_t i = tile * ROWS + col;
        const bool counts = on;
        const int64_t at = target;
        Part<T> hf[2 * KT];
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) {
#pragma unroll
            for (int k = 0; k < (int)(2 * sizeof(T)); ++k) hr[t].w[k] = counts ? hr[t].w[k] : 0;
            hf[t] = part_of(hr[t]);
            if (grads) *(Raw<T> *)(hx + col * KP + 16 * t + 8 * half) = hr[t];
        }
        if (tile + step < tiles) load(tile + step);
        f32x16 z[VT] = {};
#pragma unroll
        for (int a = 0; a < VT; ++a)
#pragma unroll
            for (int t = 0; t < 2 * KT; ++t)
                mma<M>(z[a], mul_of<T>(part_of(*(const Raw<T> *)(wx + (32 * a + perm) * KP + 16 * t + 8 * half))), mul_of<T>(hf[t]));
        float m = -INFINITY, s = 0.0f, zt = 0.0f;
        const bool in = at >= 0 && at < V;
        const int own = in ? (int)at - 8 * half : -1;  // this half's place of the target
        int b0 = 8 * half;
        asm volatile("" : "+v"(b0));  // (read here, not kept in registers throughout)
#pragma unroll
        for (int a = 0; a < VT; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                z[a][r] += bx[32 * a + 16 * (r >> 3) + (r & 7) + b0];
                m = z[a][r] > m ? z[a][r] : m;
            }
        const float m2 = __shfl_xor(m, 32, 64);
        m = m2 > m ? m2 : m;
#pragma unroll
        for (int a = 0; a < VT; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                // (the difference first: logits at the type's lowest value neither overflow nor differ)
                const float y = z[a][r] - m;
                zt = own == 32 * a + 16 * (r >> 3) + (r & 7) ? y : zt;
                z[a][r] = __builtin_amdgcn_exp2f(y * LOG2E);
                s += z[a][r];
            }
        s += __shfl_xor(s, 32, 64);
        zt += __shfl_xor(zt, 32, 64);
        // (no such target: NaN, and so is all that comes of it)
        const float logp = in ? zt - __builtin_amdgcn_logf(s) * LN_2 : NAN;
        if (half == 0 && i < c.rows) {
            if (c.logp) c.logp[i] = counts ? logp : 0.0f;
            if (counts) loss += (double)logp;
        }
        if (!grads && !c.d_hidden) continue;
        const float inv = counts ? (in ? 1.0f / s : NAN) : 0.0f, one = counts ? 1.0f : 0.0f;
#pragma unroll
        for (int a = 0; a < VT; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = counts ? z[a][r] * inv : 0.0f;
                z[a][r] = own == 32 * a + 16 * (r >> 3) + (r & 7) ? p - one : p;
                db[a][r] += z[a][r];
            }
        Part<M> gf[VT][2], gl[VT][2];
#pragma unroll
        for (int a = 0; a < VT; ++a)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float y[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) y[r] = z[a][8 * x + r];
                gf[a][x] = term_of<M>(y, true);
                if (Part<M>::TERMS) gl[a][x] = term_of<M>(y, false);
                if (grads) {
                    *(Raw<M> *)(gx + col * GP + 32 * a + 16 * x + 8 * half) = __builtin_bit_cast(Raw<M>, gf[a][x]);
                    if (Part<M>::TERMS) *(Raw<M> *)(gx + (32 + col) * GP + 32 * a + 16 * x + 8 * half) = __builtin_bit_cast(Raw<M>, gl[a][x]);
                }
            }
        if (c.d_hidden) {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                f32x16 o = {};
#pragma unroll
                for (int a = 0; a < VT; ++a)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const Part<M> wc = mul_of<T>(column_of<T>(wx, KP, 32 * a + 16 * x, 32 * t, lane));
                        mma<M>(o, wc, gf[a][x]);
                        if (Part<M>::TERMS) mma<M>(o, wc, gl[a][x]);
                    }
                if (i < c.rows) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int d = 32 * t + 16 * x + 8 * half;
                        T *const to = (T *)c.d_hidden + i * D + d;
                        Span<T, 8> e;
#pragma unroll
                        for (int r = 0; r < 8; ++r) e.e[r] = (T)(counts ? o[8 * x + r] * weight : 0.0f);
                        if (FIT == FULL || d + 8 <= D) *(Span<T, 8> *)to = e;
                        else if constexpr (FIT <= ANY) {
#pragma unroll
                            for (int r = 0; r < 8; ++r)
                                if (d + r < D) to[r] = e.e[r];
                        }
                    }
                }
            }
        }
        if (grads) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                Part<M> gc[VT][TERMS];
#pragma unroll
                for (int a = 0; a < VT; ++a)
#pragma unroll
                    for (int n = 0; n < TERMS; ++n) gc[a][n] = column_of<M>(gx, GP, 32 * n + 16 * x, 32 * a, lane);
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    const Part<M> hc = mul_of<T>(column_of<T>(hx, KP, 16 * x, 32 * t, lane));
#pragma unroll
                    for (int a = 0; a < VT; ++a)
#pragma unroll
                        for (int n = 0; n < TERMS; ++n) mma<M>(dw[a][t], gc[a][n], hc);
                }
            }
        }
    }
    loss = wave_sum(loss);
    if (lane == 0) red[wave] = loss;
    __syncthreads();
    if (c.losses && threadIdx.x == 0) c.losses[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
    if (!grads) return;
    // the waves' sums, one after the other
    float *const sums = (float *)room;
    for (int w = 0; w < WAVES; ++w) {
        if (w == wave) {
#pragma unroll
            for (int a = 0; a < VT; ++a)
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int v = 32 * a + 16 * (r >> 3) + 8 * half + (r & 7);
                        float *const y = sums + v * (32 * KT) + 32 * t + perm;
                        *y = dw[a][t][r] + (w ? *y : 0.0f);
                    }
        }
        __syncthreads();
    }
    float *const to = c.sums + (int64_t)blockIdx.x * (V * D + V);
    for (int x = threadIdx.x; x < V * D; x += BLOCK) to[x] = sums[x / D * (32 * KT) + x % D];
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) {
        if (w == wave) {
#pragma unroll
            for (int a = 0; a < VT; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float y = db[a][r];
                    for (int d = 16; d > 0; d >>= 1) y += __shfl_xor(y, d, 64);
                    const int v = 32 * a + 16 * (r >> 3) + 8 * half + (r & 7);
                    if (col == 0) sums[v] = y + (w ? sums[v] : 0.0f);
                }
        }
        __syncthreads();
    }
    for (int x = threadIdx.x; x < V; x += BLOCK) to[V * D + x] = sums[x];
}

// The workgroups' sums: 32 elements of the gradients a workgroup, in eight shares; the loss by the last.
template <typename T> __global__ __launch_bounds__(BLOCK) void k_finish(const Head c, int grid)
{
    __shared__ float red[8][32];
    __shared__ double reds[WAVES];
    if (skipped(c)) return;
    const int64_t n_on = counted(c);
    if (blockIdx.x == gridDim.x - 1) {
        if (!c.loss) return;
        double s = 0;
        for (int k = threadIdx.x; k < grid; k += BLOCK) s += c.losses[k];
        s = wave_sum(s);
        if ((threadIdx.x & 63) == 0) reds[threadIdx.x >> 6] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            s = (reds[0] + reds[1]) + (reds[2] + reds[3]);
            *c.loss = (float)(n_on ? -s * (c.sum ? 1.0 : 1.0 / (double)n_on) : 0.0);
        }
        return;
    }
    const float up1 = c.scale ? *c.scale : 1.0f;
    const float weight = c.sum ? up1 : (float)((double)up1 / (double)(n_on > 1 ? n_on : 1));
    const int n = c.width * c.dim, all = n + c.width, share = threadIdx.x >> 5;
    const int x = blockIdx.x * 32 + (threadIdx.x & 31);
    float s = 0.0f;
    if (x < all)
        for (int k0 = share; k0 < grid; k0 += 8 * 16) {  // (asked for together: latency is all of this)
            float y[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) y[q] = k0 + 8 * q < grid ? c.sums[(int64_t)(k0 + 8 * q) * all + x] : 0.0f;
#pragma unroll
            for (int q = 0; q < 16; ++q) s += y[q];
        }
    red[share][threadIdx.x & 31] = s;
    __syncthreads();
    if (share || x >= all) return;
    s = 0.0f;
    for (int k = 0; k < 8; ++k) s += red[k][threadIdx.x];
    if (x < n) {
        if (c.d_weight) ((T *)c.d_weight)[x] = (T)(s * weight);
    } else if (c.d_bias) ((T *)c.d_bias)[x - n] = (T)(s * weight);
}

uint64_t up_to(uint64_t n, uint64_t k) { return (n + k - 1) / k * k; }
int grid_of(int64_t rows)
{
    const int64_t n = (rows + ROWS * WAVES - 1) / (ROWS * WAVES);
    return (int)(n < 1 ? 1 : n > MOST_BLOCKS ? MOST_BLOCKS : n);
}

template <typename T, int VT, int KT> void rows(const Head &c, int grid, hipStream_t st)
{
    if (c.dim == 32 * KT) hipLaunchKernelGGL((k_rows<T, VT, KT, FULL>), dim3(grid), dim3(BLOCK), 0, st, c);
    else if (c.dim % 8 == 0) hipLaunchKernelGGL((k_rows<T, VT, KT, EIGHTS>), dim3(grid), dim3(BLOCK), 0, st, c);
    else if (c.dim >= 8) hipLaunchKernelGGL((k_rows<T, VT, KT, ANY>), dim3(grid), dim3(BLOCK), 0, st, c);
    else if constexpr (KT == 1) hipLaunchKernelGGL((k_rows<T, VT, KT, SHORT>), dim3(grid), dim3(BLOCK), 0, st, c);
}

template <typename T> void call(const Head &c, int grid, hipStream_t st)
{
    if (c.width <= 32) {
        if (c.dim <= 32) rows<T, 1, 1>(c, grid, st);
        else if (c.dim <= 64) rows<T, 1, 2>(c, grid, st);
        else rows<T, 1, 4>(c, grid, st);
    } else {
        if (c.dim <= 32) rows<T, 2, 1>(c, grid, st);
        else rows<T, 2, 2>(c, grid, st);
    }
    const int blocks = c.sums ? (c.width * c.dim + c.width + 31) / 32 : 0;
    if (c.loss || c.sums) hipLaunchKernelGGL((k_finish<T>), dim3(blocks + 1), dim3(BLOCK), 0, st, c, grid);
}

}  // namespace

namespace narrow {

bool fits(const swarp_linear_ce_t *a)
{
    return (a->width <= 32 && a->dim <= 128) || (a->width <= 64 && a->dim <= 64);
}

uint64_t work_bytes(const swarp_linear_ce_t *a)
{
    return up_to(4 * (a->mask ? counts_of(a->rows) : 0), 256) + MOST_BLOCKS * 8 +
           up_to((uint64_t)grid_of(a->rows) * (a->width * a->dim + a->width) * 4, 256);
}

int run(const swarp_linear_ce_t *a, int skip_unit, const float *scale, void *d_hidden, void *d_weight, void *d_bias,
        hipStream_t st)
{
    Head c = {};
    c.rows = a->rows;
    c.inner = a->inner;
    c.outer_stride = a->outer_stride;
    c.inner_stride = a->inner_stride;
    c.dim = a->dim;
    c.width = a->width;
    c.targets32 = a->targets32;
    c.sum = a->sum;
    c.skip_unit = skip_unit;
    c.hidden = a->hidden;
    c.weight = a->weight;
    c.bias = a->bias;
    c.targets = a->targets;
    c.mask = a->mask;
    c.scale = scale;
    c.d_hidden = d_hidden;
    c.d_weight = d_weight;
    c.d_bias = d_bias;
    const int grid = grid_of(a->rows);
    char *mem = (char *)a->work;
    c.losses = (double *)mem;
    mem += MOST_BLOCKS * 8;
    c.sums = d_weight || d_bias ? (float *)mem : nullptr;
    mem += up_to((uint64_t)grid * (a->width * a->dim + a->width) * 4, 256);
    if (!scale) {
        c.logp = a->logp;
        c.loss = a->loss;
    }
    if (a->mask && a->rows) {
        c.counts = (int32_t *)mem;
        c.n_counts = (int)counts_of(a->rows);
        count(a->rows, a->mask, (int32_t *)c.counts, st);
    }
    switch (a->dtype) {
    case SWARP_F32: call<float>(c, grid, st); break;
    case SWARP_BF16: call<bf16>(c, grid, st); break;
    default: call<f16>(c, grid, st); break;
    }
    return launched();
}

}  // namespace narrow
