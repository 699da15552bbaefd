// linear_ce.hip -- softmax cross entropy of a linear head, from the hidden states and the head's
// weight, without the logits (swarp_linear_ce).
//
// Per decision i with the hidden state h, target t and the head's rows W_j (and biases b_j):
//   z_j = h W_j + b_j;   logp = z_t - log sum_j exp z_j;   loss = -w sum of logp;
//   G_ij = p_ij - [j = t];   d h_i = w G_i W,  d W = w G^T h,  d b = w sum_i G_i.
//
// Three matrix products of 2 rows dim width operations each: the logits, which are formed tile by
// tile in the matrix cores' registers and leave them as exponentials, and the two gradients, which
// need all of a row's exponentials.  Those are kept for as many rows as 1 GiB holds (a piece); then
// comes the next piece.  They are relative to the target's logit r, which is known beforehand (one dot
// product a row):
//   E_ij = exp(z_j - r_i),  s_i = sum_j E_ij,  logp = -log(s_i / E_it),  G_ij = E_ij / s_i - [j = t],
// so that a tile of them can be written before the row's sum is known.  Where some logit of a piece is above
// its target's by more than REACH the piece is done again, relative to the rows' maxima (the kernels of that
// second pass are always launched, look at a flag, and mostly end).
// A dot product adds in another order than the matrix cores: r is off z_t by some 2^-24 of their terms, which
// may be more than 1 - p.  So the target's own exponential, and G there, come of the logit that its tile has:
// s_i is a sum with E_it in it, never less, and logp never above 0.
//
// float32: 1 / s_i goes into the rows of d h and into E, or into h beside E^T, whichever is less.
//
// 16 bits: h / s beside E^T would be a second rounding of d W's terms (8 x 1023 decisions of 50001 logits,
// 1024 wide, bfloat16, a quarter masked: 2.9e-3 of its size off, where its own rounding makes 1.7e-3),
// and float16 has not the range.  So 24 bits of an exponential are kept, in two places, and become G,
// normalised and rounded once, in a pass of their own (0.32 ms there: 5 bytes a logit at 4.8 TB/s), beside
// which h stands as it is: 2.45 ms in all; it was 2.17 with the second rounding, and 2.83 with the sums from a
// product of their own.  d h of few columns, which p - 1 does not lead, is 2.1e-3 off where its own rounding makes 1.7e-3
// (10038 x 414, 15 columns, bfloat16): a second term of G would be a second product of each kind.
//
// Decisions whose mask is not set are left out of the products: the rows that count are gathered
// first, and every kernel goes by their number on the device.
#include <math.h>

#include <atomic>

#include "matrix.hpp"
#include "narrow_ce.hpp"

namespace {

using namespace mat;
using learn::fail;
using learn::launched;
using learn::up;
using learn::wave_sum;

constexpr int BLOCK = 256;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN_2 = 0.69314718055994530942f;
constexpr float REACH = 40.0f;        // e^40 times 2^21 logits, times any weight, is far from overflow
constexpr int KEPT_BITS = 14;         // 16-bit exponentials are kept times 2^14: float16's 2^-38 is not lost
using narrow::COUNT_ROWS;
constexpr uint64_t PIECE = 1ull << 30;  // bytes of exponentials at a time (but for their lower 8 bits)

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
__device__ __forceinline__ float log_of(float x) { return __builtin_amdgcn_logf(x) * LN_2; }

// What every kernel of a call may read.  Rows are the counted ones, in order; `n_on` of them.
struct Call {
    int64_t rows;             // of the call; at most as many count
    int64_t inner, outer_stride, inner_stride;
    int dim, width;
    int dim_p;                // elements of a padded row of h
    int pitch_w;              // bytes of a row of W
    int64_t wide;             // elements of a row of E
    int64_t first;            // row that the piece starts with
    int piece;                // rows that it has room for
    int targets32, sum;
    const void *hidden, *weight, *bias, *targets;
    const int32_t *index;     // which rows count, or NULL: all
    const int32_t *n_on;      // how many, or NULL: all
    float *logp, *loss;
    // of all rows
    void *h;
    float *z_t, *ref, *top;   // target's logit (NaN: none); what E is relative to; largest logit
    float *inv, *inv_h;       // of d h's rows; what h, or E (16 bits), is multiplied by: k_scale, k_norm
    float *one;               // normed: G / weight times 2^KEPT_BITS at the target
    int32_t *target;          // or -1
    double *sums;             // of logp, one for `few` rows
    int few;                  // rows of a workgroup that joins: 1 or 64
    int64_t pieces;
    int normed;               // E becomes G in a pass of its own, and h stands beside it as it is
    // of the piece
    int32_t *flag;            // (of all of them, one behind the other)
    float2 *parts;            // [n_parts][piece]: largest logit and sum of a part of a row
    int n_parts;
    void *e, *hs;             // exponentials; h as it goes beside them
    uint8_t *low;             // of a 24-bit exponential, the bits that E has not room for
    const void *w;            // padded weight
};

// Rows of the piece that count.
__device__ __forceinline__ int rows_of(const Call &c)
{
    const int64_t n = (c.n_on ? (int64_t)*c.n_on : c.rows) - c.first;
    return (int)(n < 0 ? 0 : n < c.piece ? n : c.piece);
}

// Weight of a row in the loss.
__device__ __forceinline__ float weight_of(const Call &c)
{
    const int64_t n = c.n_on ? (int64_t)*c.n_on : c.rows;
    return c.sum || n < 1 ? 1.0f : (float)(1.0 / (double)n);
}

// ------------------------------------------------------------------ which rows count

__global__ __launch_bounds__(BLOCK) void k_count(int64_t rows, const uint8_t *mask, int32_t *counts)
{
    __shared__ int red[BLOCK / 64];
    int n = 0;
    for (int k = threadIdx.x; k < COUNT_ROWS; k += BLOCK) {
        const int64_t i = (int64_t)blockIdx.x * COUNT_ROWS + k;
        n += i < rows && mask[i];
    }
    n = wave_sum(n);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// index[j] is the j-th row that counts, place[i] the j of row i or -1; logp of the others is 0.
__global__ __launch_bounds__(BLOCK) void k_place(int64_t rows, const uint8_t *mask, const int32_t *counts,
                                                 int32_t *index, int32_t *place, int32_t *n_on, float *logp)
{
    __shared__ int red[BLOCK / 64];
    int before = 0;
    for (int k = threadIdx.x; k < (int)blockIdx.x; k += BLOCK) before += counts[k];
    before = wave_sum(before);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = before;
    __syncthreads();
    int at = red[0] + red[1] + red[2] + red[3];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int k = 0; k < COUNT_ROWS; k += BLOCK) {
        const int64_t i = (int64_t)blockIdx.x * COUNT_ROWS + k + threadIdx.x;
        const bool on = i < rows && mask[i];
        const uint64_t votes = __ballot(on);
        __syncthreads();
        if (lane == 0) red[w] = __popcll(votes);
        __syncthreads();
        int j = at + __popcll(votes & ((1ull << lane) - 1));
        for (int v = 0; v < w; ++v) j += red[v];
        if (on) index[j] = (int32_t)i;
        if (i < rows) {
            place[i] = on ? j : -1;
            if (!on) logp[i] = 0.0f;
        }
        at += red[0] + red[1] + red[2] + red[3];
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *n_on = at;
}

// ------------------------------------------------------------------ rows made ready

// Eight neighbouring elements, anywhere.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T e[8];
};

// Row i of the hidden states, padded with zeros, its target, and (of a call that keeps exponentials) what those
// will be relative to.  A wave a row.
template <typename T> __global__ __launch_bounds__(BLOCK) void k_rows(const Call c)
{
    const int lane = threadIdx.x & 63;
    const int64_t n = c.n_on ? *c.n_on : c.rows;
    for (int64_t k = (int64_t)blockIdx.x * BLOCK + threadIdx.x; k < c.pieces; k += (int64_t)gridDim.x * BLOCK) c.flag[k] = 0;
    for (int64_t j = (int64_t)blockIdx.x * (BLOCK / 64) + (threadIdx.x >> 6); j < (n + 31) / 32 * 32;
         j += (int64_t)gridDim.x * (BLOCK / 64)) {
        if (j >= n) {  // the last step of a product over the rows ends with zeros
            for (int k = lane * 8; k < c.dim_p; k += 64 * 8) *(Eight<T> *)((T *)c.h + j * c.dim_p + k) = Eight<T>{};
            continue;
        }
        const int64_t i = c.index ? c.index[j] : j;
        const uint64_t o = (uint64_t)i / (uint64_t)c.inner;
        const T *const x = (const T *)c.hidden + (int64_t)o * c.outer_stride + (i - (int64_t)o * c.inner) * c.inner_stride;
        const int64_t t = c.targets32 ? (int64_t)((const int32_t *)c.targets)[i] : ((const int64_t *)c.targets)[i];
        const bool in = t >= 0 && t < c.width;
        const T *const w = (const T *)c.weight + (in ? t : 0) * c.dim;
        T *const h = (T *)c.h + j * c.dim_p;
        float z = 0.0f;
        for (int k = lane * 8; k < c.dim_p; k += 64 * 8) {  // (a padded row is a multiple of eight)
            Eight<T> v = {}, y = {};
            if (k + 8 <= c.dim) {
                v = *(const Eight<T> *)(x + k);
                if (c.e) y = *(const Eight<T> *)(w + k);
            } else {
                for (int q = 0; q < 8; ++q)
                    if (k + q < c.dim) {
                        v.e[q] = x[k + q];
                        if (c.e) y.e[q] = w[k + q];
                    }
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) z = __builtin_fmaf(up(v.e[q]), up(y.e[q]), z);
            *(Eight<T> *)(h + k) = v;
        }
        z = wave_sum(z);
        if (lane == 0) {
            if (c.bias) z += up(((const T *)c.bias)[in ? t : 0]);
            c.z_t[j] = NAN;  // (k_logits has it where there is such a target)
            c.ref[j] = in ? z : NAN;
            c.target[j] = in ? (int32_t)t : -1;
        }
    }
}

// out [rows][pitch] = in [rows][n], the rest zero.
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_pad(const T *in, int64_t rows, int n, T *out, int pitch)
{
    const int64_t all = rows * pitch;
    for (int64_t k = (int64_t)blockIdx.x * BLOCK + threadIdx.x; k < all; k += (int64_t)gridDim.x * BLOCK) {
        const int64_t r = k / pitch;
        const int i = (int)(k - r * pitch);
        out[k] = i < n ? in[r * n + i] : (T)0.0f;
    }
}

// The piece's rows of h times inv_h, which the weight's gradient is made of, and zeros up to a whole
// step (where E has none).  A wave a row.
__global__ __launch_bounds__(BLOCK) void k_scale(const Call c)
{
    const int rows = rows_of(c), all = (rows + 31) / 32 * 32, lane = threadIdx.x & 63;
    for (int r = blockIdx.x * (BLOCK / 64) + (threadIdx.x >> 6); r < all; r += gridDim.x * (BLOCK / 64)) {
        const float *const x = (const float *)c.h + (c.first + (r < rows ? r : 0)) * c.dim_p;
        const float f = r < rows ? c.inv_h[c.first + r] : 0.0f;
        for (int k = lane * 8; k < c.dim_p; k += 64 * 8) {
            Eight<float> v = *(const Eight<float> *)(x + k);
#pragma unroll
            for (int q = 0; q < 8; ++q) v.e[q] = r < rows ? v.e[q] * f : 0.0f;
            *(Eight<float> *)((float *)c.hs + (int64_t)r * c.dim_p + k) = v;
        }
    }
}

// ------------------------------------------------------------------ logits

// A tile of logits, width along the tile's rows and decisions along its columns, so that a lane has
// many logits of one decision.  Leaves the largest and the sum of the exponentials of each wave's
// part of a row; with STORE relative to ref[row], and the exponentials themselves; else the sum is
// relative to the part's largest.  With `again` only where the piece's flag is set.
// 6138 x 50001 logits of 1024 terms, bfloat16: 0.83 ms, 760 TFLOP/s with the exponentials written (0.9 GB); the
// products alone run at some 950, the rest is what a tile's end (exponentials, two trips through LDS) does not
// overlap with the next tile's products: a compute unit has room for one workgroup of 256 x 256.
// 16 x 131072 logits, bfloat16: 44 us for 268 MB of weight, 6.1 TB/s.
template <typename T, typename C, bool STORE>
__global__ __launch_bounds__(C::THREADS) void k_logits(const Call c, int nm, int nn, int again)
{
    extern __shared__ __align__(16) char lds[];
    if (again && !*c.flag) return;
    const int rows = rows_of(c);
    int tm, tn;
    tile_of(blockIdx.x, gridDim.x, nm, nn, tm, tn);
    const int v0 = tm * C::BM, r0 = tn * C::BN;
    if (r0 >= rows) return;
    const int lane = threadIdx.x & 63, w = C::wave(), wm = w / C::WN, wn = w % C::WN;
    C t;
    t.clear();
    const int64_t pitch = (int64_t)c.dim_p * sizeof(T);
    const Operand a = {(const char *)c.w + v0 * (int64_t)c.pitch_w, c.pitch_w, c.width - v0, c.pitch_w};
    const Operand b = {(const char *)c.h + (c.first + r0) * pitch, pitch, rows - r0, (int)pitch};
    t.run(lds, a, b, 0, c.dim_p / C::KE);
    if (c.bias || v0 + C::BM > c.width) {
        // -inf past the last column
        float *const bias = (float *)lds;
        for (int k = threadIdx.x; k < C::BM; k += C::THREADS)
            bias[k] = v0 + k >= c.width ? -INFINITY : c.bias ? up(((const T *)c.bias)[v0 + k]) : 0.0f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float y = bias[(wm * C::TM + i) * 32 + acc_row(r, lane)];
#pragma unroll
                for (int j = 0; j < C::TN; ++j) t.acc[i][j][r] += y;
            }
    }
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
        const int row = r0 + (wn * C::TN + j) * 32 + acc_col(lane);
        const bool mine = row < rows;
        float m = -INFINITY, s = 0.0f;
        // (few tiles of a wide head hold a target of theirs)
        const uint32_t own = mine ? (uint32_t)(c.target[c.first + row] - (v0 + wm * C::TM * 32)) : ~0u;
        if (__ballot(own < C::TM * 32u)) {
            float zt = 0.0f;
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) zt = own == (uint32_t)(i * 32 + acc_row(r, lane)) ? t.acc[i][j][r] : zt;
            if (own < C::TM * 32u && (own >> 2 & 1) == (uint32_t)lane >> 5) c.z_t[c.first + row] = zt;
        }
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) m = fmaxf(m, t.acc[i][j][r]);  // (a NaN is passed over here and shows in the sum)
        const float ref = STORE ? (again ? c.top : c.ref)[c.first + (mine ? row : 0)] : (m == -INFINITY ? 0.0f : m);
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = exp_of(t.acc[i][j][r] - ref);
                s += e;
                t.acc[i][j][r] = e;
            }
        if constexpr (STORE) {
            s += __shfl_xor(s, 32, 64);
            const float y = __shfl_xor(m, 32, 64);
            m = y > m ? y : m;
        } else {
            const float ms = __shfl_xor(m, 32, 64), ss = __shfl_xor(s, 32, 64);
            const float hi = ms > m ? ms : m, at = hi == -INFINITY ? 0.0f : hi;
            s = (m == -INFINITY && s == 0.0f ? 0.0f : s * exp_of(m - at)) +
                (ms == -INFINITY && ss == 0.0f ? 0.0f : ss * exp_of(ms - at));
            m = hi;
        }
        if (lane < 32 && mine) c.parts[(int64_t)(tm * C::WM + wm) * c.piece + row] = make_float2(m, s);
    }
    if constexpr (STORE) {
        // through LDS, so that a row's are written together: 32 decisions of a wave's columns at a time
        constexpr int PITCH = C::TM * 32 + 16 / (int)sizeof(T), PIECES = C::TM * 32 * (int)sizeof(T) / 16;
        constexpr bool LOW = sizeof(T) == 2;
        constexpr int PITCH_LOW = C::TM * 32 + 16;
        static_assert(C::WAVES * 32 * (PITCH * (int)sizeof(T) + (LOW ? PITCH_LOW : 0)) <= C::LDS, "a wave's part of a tile fits");
        T *const mine = (T *)lds + w * 32 * PITCH;
        uint8_t *const low = (uint8_t *)lds + C::WAVES * 32 * PITCH * sizeof(T) + w * 32 * PITCH_LOW;
        __syncthreads();  // (every wave has read its last operands)
        const int64_t v = v0 + wm * C::TM * 32;
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int at = i * 32 + acc_row(r, lane);
                    if constexpr (LOW) {
                        // the upper 24 bits, rounded: 16 and 8
                        uint32_t u[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float x = t.acc[i][j][r + q];  // (a vector's element has no address to cast from)
                            u[q] = __builtin_bit_cast(uint32_t, x) + 0x80u;
                        }
                        const uint2 y = {__builtin_amdgcn_perm(u[1], u[0], 0x07060302u), __builtin_amdgcn_perm(u[3], u[2], 0x07060302u)};
                        *(uint2 *)(mine + acc_col(lane) * PITCH + at) = y;
                        const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0501u), b = __builtin_amdgcn_perm(u[3], u[2], 0x05010c0cu);
                        *(uint32_t *)(low + acc_col(lane) * PITCH_LOW + at) = a | b;
                    } else {
                        *(f32x4 *)(mine + acc_col(lane) * PITCH + at) =
                            f32x4{t.acc[i][j][r], t.acc[i][j][r + 1], t.acc[i][j][r + 2], t.acc[i][j][r + 3]};
                    }
                }
            __builtin_amdgcn_wave_barrier();
            const int row0 = r0 + (wn * C::TN + j) * 32;
#pragma unroll
            for (int k = 0; k < 32 * PIECES / 64; ++k) {
                const int at = k * 64 + lane, r = at / PIECES, e = at % PIECES * (16 / (int)sizeof(T));
                if (row0 + r < rows && v + e < c.wide)
                    *(u32x4 *)((T *)c.e + (int64_t)(row0 + r) * c.wide + v + e) = *(const u32x4 *)(mine + r * PITCH + e);
            }
            if constexpr (LOW) {
                constexpr int LOWS = C::TM * 32 / 16;
#pragma unroll
                for (int k = 0; k < 32 * LOWS / 64; ++k) {
                    const int at = k * 64 + lane, r = at / LOWS, e = at % LOWS * 16;
                    if (row0 + r < rows && v + e < c.wide)
                        *(u32x4 *)(c.low + (int64_t)(row0 + r) * c.wide + v + e) = *(const u32x4 *)(low + r * PITCH_LOW + e);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// How a row's parts are joined.
enum { SUMS = 0,     // from parts relative to their largest: logp
       KEPT = 1,     // from parts relative to ref, which E is too: logp, 1 / s, G at the target
       KEPT2 = 2 };  // the same after a second pass

// A workgroup takes ROWS rows, its threads every (BLOCK / ROWS)-th part of one.
template <typename T, int ROWS> __global__ __launch_bounds__(BLOCK) void k_join(const Call c, int how)
{
    constexpr int WAYS = BLOCK / ROWS, AHEAD = 8;
    auto of = [](float part, float all) { return part == -INFINITY ? 1.0f : exp_of(part - all); };
    __shared__ float red[2][WAYS][ROWS];
    __shared__ double total[ROWS];
    if (how == KEPT2 && !*c.flag) return;
    const int rows = rows_of(c), lane = threadIdx.x % ROWS, w = threadIdx.x / ROWS;
    const int row = blockIdx.x * ROWS + lane;
    const bool mine = row < rows;
    const int64_t j = c.first + (mine ? row : 0);
    if (blockIdx.x * ROWS >= rows) return;
    const float ref = how == KEPT2 ? c.top[j] : c.ref[j], zt = c.z_t[j];
    float s = 0.0f, m = -INFINITY;
    if (mine) {
        // (asked for together: a row's parts are few enough that latency is all of this)
        for (int k0 = w; k0 < c.n_parts; k0 += AHEAD * WAYS) {
            float2 p[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int k = k0 + q * WAYS;
                p[q] = k < c.n_parts ? c.parts[(int64_t)k * c.piece + row] : make_float2(-INFINITY, 0.0f);
            }
            float hi = m;
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) hi = p[q].x > hi ? p[q].x : hi;
            const float at = hi == -INFINITY ? 0.0f : hi;
            if (how == SUMS) s *= of(m, at);
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                s += how == SUMS ? p[q].y * of(p[q].x, at) : p[q].y;
            m = hi;
        }
    }
    red[0][w][lane] = m;
    red[1][w][lane] = s;
    __syncthreads();
    float hi = m;
    if constexpr (ROWS == 1) {
        if (w >= 64) return;
        for (int k = w + 64; k < WAYS; k += 64) hi = red[0][k][0] > hi ? red[0][k][0] : hi;
        hi = learn::wave_max(hi);
        s = 0.0f;
        for (int k = w; k < WAYS; k += 64) s += red[1][k][0] * (how == SUMS ? of(red[0][k][0], hi) : 1.0f);
        s = wave_sum(s);
        if (w) return;
    } else {
        if (w) return;
        for (int k = 1; k < WAYS; ++k) hi = red[0][k][lane] > hi ? red[0][k][lane] : hi;
        s = 0.0f;
        for (int k = 0; k < WAYS; ++k) s += red[1][k][lane] * (how == SUMS ? of(red[0][k][lane], hi) : 1.0f);
    }
    const int64_t i = c.index ? c.index[j] : j;
    float logp;
    const float et = exp_of(zt - ref);  // as E has it
    if (how == SUMS) {
        logp = (zt - hi) - log_of(s);
    } else {
        // (s is not below et, which is one of its terms)
        logp = et > 0.5f ? -log_of(s / et) : (zt - ref) - log_of(s);
        if (how == KEPT && mine) {
            if (hi - ref > REACH || ref == -INFINITY) *c.flag = 1;
            c.top[j] = hi;
        }
    }
    // (no logit above -inf, or no such target: in a second pass its row's exponentials are finite)
    const bool none = hi == -INFINITY || zt != zt;
    if (none) logp = NAN;
    if (mine && how != SUMS) {
        if (!c.normed) {
            c.inv[j] = c.inv_h[j] = none ? NAN : weight_of(c) / s;
            if (c.target[j] >= 0) ((float *)c.e)[(int64_t)row * c.wide + c.target[j]] = et - s;
        } else {
            const float f = none ? NAN : (1 << KEPT_BITS) / s;
            c.inv[j] = weight_of(c) / (1 << KEPT_BITS);
            c.inv_h[j] = f;
            c.one[j] = (et - s) * f;
        }
    }
    if (mine) c.logp[i] = logp;
    total[lane] = mine ? (double)logp : 0.0;
    __builtin_amdgcn_wave_barrier();  // (w == 0: one wave at most)
    if (lane == 0) {
        double sum = 0;
        for (int k = 0; k < ROWS; ++k) sum += total[k];
        c.sums[c.first / ROWS + blockIdx.x] = sum;
    }
}

// An exponential as it is kept.
__device__ __forceinline__ float exponential(float e, uint8_t) { return e; }
template <typename T> __device__ __forceinline__ float exponential(T e, uint8_t low)
{
    return __builtin_bit_cast(float, (uint32_t)__builtin_bit_cast(uint16_t, e) << 16 | (uint32_t)low << 8);
}

// G / weight times 2^KEPT_BITS, in E's place.  A thread takes eight neighbours at a time (a row is of whole
// steps, so they are of one row), NORMS times, which it asks for ahead.
constexpr int NORMS = 4;
template <typename T> __global__ __launch_bounds__(BLOCK) void k_norm(const Call c)
{
    const uint32_t eights = (uint32_t)(c.wide / 8), n = (uint32_t)rows_of(c) * eights;  // (at most 2^26)
    struct __attribute__((aligned(16))) Whole { T e[8]; };
    struct __attribute__((aligned(8))) Low { uint8_t e[8]; };
    Whole x[NORMS];
    Low y[NORMS];
    float f[NORMS];
    int32_t t[NORMS];
    const uint32_t first = blockIdx.x * NORMS * BLOCK + threadIdx.x;
#pragma unroll
    for (int k = 0; k < NORMS; ++k) {
        const uint32_t at = first + k * BLOCK;
        if (at >= n) break;
        x[k] = ((const Whole *)c.e)[at];
        if constexpr (sizeof(T) == 2) y[k] = ((const Low *)c.low)[at];
        const uint32_t row = at / eights;
        f[k] = c.inv_h[c.first + row];
        t[k] = c.target[c.first + row] - (int32_t)(at - row * eights) * 8;
    }
#pragma unroll
    for (int k = 0; k < NORMS; ++k) {
        const uint32_t at = first + k * BLOCK;
        if (at >= n) break;
        Whole z;
#pragma unroll
        for (int q = 0; q < 8; ++q) z.e[q] = (T)(exponential(x[k].e[q], y[k].e[q]) * f[k]);
        if ((uint32_t)t[k] < 8u) {
            const T one = (T)c.one[c.first + at / eights];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q == t[k]) z.e[q] = one;
        }
        ((Whole *)c.e)[at] = z;
    }
}

// ------------------------------------------------------------------ products of the gradients

// out [m][n] (+)= scale[m] sum_k A[m][k] B[n][k].  B lies along k ([k][n]), A too where AK ([k][m]).
struct Product {
    const void *a, *b;
    int64_t a_pitch, b_pitch;  // bytes
    int64_t m, n;              // rows of A and of B
    int k;                     // how many there are
    int rows_m, rows_k;        // 1: m, or k, is the piece's rows instead
    int add;
    float times;               // with `weigh` times the rows' weight
    int weigh;
    const float *scale;        // of the rows of A, or NULL
    float *out;                // [m][n]
    float *parts;              // sums of splits
};

// How a product's tiles go over the workgroups, one for each place on the chip: whole tiles in rounds,
// one a workgroup, and what is left of the last round along k, into as many splits as end soonest.
// (8184 decisions of 50001 logits, a quarter of them masked, 1024 wide: 96 tiles for 256 places.)
struct Share {
    int nm, nn, steps;
    int64_t whole;        // tiles that a workgroup does alone
    int rest, splits;     // of the others
};

// What a split of one tile costs, in steps of a round: a step of 256 x 256 in 16 bits takes some 0.45 us, of 128 x 128
// or 64 x 256 in float32 1, of 64 x 256 in 16 bits as long as of 256 x 256 (it waits for memory); a tile's
// sums to memory and back 0.1 and 0.03 (all chip).
template <typename C> constexpr float split_cost() { return (C::BM * C::BN == 256 * 256 ? 0.25f : 0.06f) * (C::KE == 32 ? 1.0f : 0.5f); }

template <typename C> __host__ __device__ __forceinline__ Share share_of(int64_t m, int64_t n, int steps, int places)
{
    Share s;
    s.nm = (int)((m + C::BM - 1) / C::BM);
    s.nn = (int)((n + C::BN - 1) / C::BN);
    s.steps = steps;
    const int64_t tiles = (int64_t)s.nm * s.nn;
    s.rest = (int)(tiles % places);
    s.whole = tiles - s.rest;
    s.splits = 1;
    float least = (float)steps;
    constexpr int WAYS[] = {2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64, 96, 128, 192, 256};
    for (int w : WAYS) {
        if (!s.rest || s.rest * w > 2 * places || w * 4 > steps) break;
        const float cost = (float)((s.rest * w + places - 1) / places) * (float)((steps + w - 1) / w) + split_cost<C>() * (float)(s.rest * w);
        if (cost < least) {
            least = cost;
            s.splits = w;
        }
    }
    return s;
}
// The m and n of a tile: groups of eight rows of tiles share what they read of B while it is in L2.
__device__ __forceinline__ void place_of(const Share &s, int64_t t, int &m, int &n)
{
    const int per = 8 * s.nn, group = (int)(t / per), first = group * 8, size = s.nm - first < 8 ? s.nm - first : 8;
    const int at = (int)(t - (int64_t)group * per);
    m = first + at % size;
    n = at / size;
}

// 6138 rows, 50001 columns, 1024 terms, bfloat16: d h and d W 0.65 ms each, 960 TFLOP/s, with the splits' joining
// 0.03 more (a plain library product of the same sizes: 860 to 1020).  96 rows, 131072 columns, float32: 0.33 and
// 0.40 ms, 79 and 64 TFLOP/s of 154: six steps a tile, whose first loads and 64 KiB of output nothing covers.
template <typename T, typename C, bool AK>
__global__ __launch_bounds__(C::THREADS, 2) void k_product(const Call c, const Product p)
{
    extern __shared__ __align__(16) char lds[];
    const int rows = rows_of(c), places = gridDim.x;
    const int64_t M = p.rows_m ? rows : p.m;
    const int k = p.rows_k ? rows : p.k;
    const Share s = share_of<C>(M, p.n, (k + C::KE - 1) / C::KE, places);
    const float times = p.weigh ? p.times * weight_of(c) : p.times;
    const int lane = threadIdx.x & 63, w = C::wave(), wm = w / C::WN, wn = w % C::WN;
    // (workgroups go round the eight dies one by one: each die, with its own L2, has neighbouring tiles)
    const int mine = places % 8 ? blockIdx.x : (blockIdx.x & 7) * (places / 8) + (blockIdx.x >> 3);
    for (int64_t u = mine; u < s.whole + (int64_t)s.rest * s.splits; u += places) {
        const bool whole = u < s.whole || s.splits == 1;
        const int64_t part = u - s.whole;
        int first = 0, last = s.steps, tm, tn;
        if (!whole) {
            const int each = (s.steps + s.splits - 1) / s.splits;
            first = (int)(part / s.rest) * each;
            last = first + each < s.steps ? first + each : s.steps;
        }
        place_of(s, whole ? u : s.whole + part % s.rest, tm, tn);
        const int64_t m0 = (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
        C t;
        t.clear();
        const Operand a = {(const char *)p.a + (AK ? m0 * (int64_t)sizeof(T) : m0 * p.a_pitch), p.a_pitch,
                           (int)(M - m0 < C::BM ? M - m0 : C::BM), AK ? k : (int)p.a_pitch};
        const Operand b = {(const char *)p.b + n0 * (int64_t)sizeof(T), p.b_pitch, (int)(p.n - n0 < C::BN ? p.n - n0 : C::BN),
                           p.rows_k ? (k + 31) / 32 * 32 : k};  // (h beside E^T ends with zeros)
        t.template run<AK, true>(lds, a, b, first, last);
        // (where each element goes is worked out here, and not kept in registers from tile to tile)
        int at = lane;
        asm volatile("" : "+v"(at));
        const int i0 = wm * C::TM * 32 + acc_row(0, at), j0 = wn * C::TN * 32 + acc_col(at);
        if (whole) {
            float *const out = p.out + (m0 + i0) * p.n + n0 + j0;
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = 32 * i + acc_row(r, 0);
                    if (m0 + i0 + row >= M) continue;
                    const float f = p.scale ? times * p.scale[m0 + i0 + row] : times;
#pragma unroll
                    for (int j = 0; j < C::TN; ++j)
                        if (n0 + j0 + 32 * j < p.n) {
                            float *const y = out + row * p.n + 32 * j;
                            *y = f * t.acc[i][j][r] + (p.add ? *y : 0.0f);
                        }
                }
        } else {
            float *const sums = p.parts + part * (C::BM * C::BN) + i0 * C::BN + j0;
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
#pragma unroll
                    for (int j = 0; j < C::TN; ++j) sums[(32 * i + acc_row(r, 0)) * C::BN + 32 * j] = t.acc[i][j][r];
        }
    }
}

// The tiles whose sums lie in splits.
template <typename C> __global__ __launch_bounds__(BLOCK) void k_splits(const Call c, const Product p, int ke, int places)
{
    const int rows = rows_of(c), k = p.rows_k ? rows : p.k;
    const int64_t M = p.rows_m ? rows : p.m;
    const Share s = share_of<C>(M, p.n, (k + ke - 1) / ke, places);
    if (s.splits == 1) return;
    const float times = p.weigh ? p.times * weight_of(c) : p.times;
    constexpr int AREA = C::BM * C::BN;
    for (int64_t x = (int64_t)blockIdx.x * BLOCK + threadIdx.x; x < (int64_t)s.rest * AREA; x += (int64_t)gridDim.x * BLOCK) {
        const int at = (int)(x % AREA), i = (int)(x / AREA);
        int tm, tn;
        place_of(s, s.whole + i, tm, tn);
        const int64_t m = (int64_t)tm * C::BM + at / C::BN, n = (int64_t)tn * C::BN + at % C::BN;
        if (m >= M || n >= p.n) continue;
        float y = 0.0f;
        for (int w0 = 0; w0 < s.splits; w0 += 16) {  // (asked for together: there may be no other wave to wait for)
            float part[16];
#pragma unroll
            for (int w = 0; w < 16; ++w) part[w] = w0 + w < s.splits ? p.parts[((int64_t)(w0 + w) * s.rest + i) * AREA + at] : 0.0f;
#pragma unroll
            for (int w = 0; w < 16; ++w) y += part[w];
        }
        float *const out = p.out + m * p.n + n;
        *out = y * (p.scale ? times * p.scale[m] : times) + (p.add ? *out : 0.0f);
    }
}

// d b = sum_i inv_i E_ij, from E before it is rounded: where an action is as often right as it is likely the
// sum is small beside its terms.  A workgroup takes 64 lanes' 16 bytes of columns and one of BIAS_WAYS shares of
// the rows, its waves every fourth of these; the shares are added by k_bias_sum.
constexpr int BIAS_WAYS = 32;

template <typename T> __global__ __launch_bounds__(BLOCK) void k_bias(const Call c, float *parts)
{
    constexpr int V = 16 / sizeof(T);
    struct __align__(16) Line { T e[V]; };
    struct __align__(V) Low { uint8_t e[V]; };
    __shared__ float red[4][64 * V];
    const int rows = rows_of(c), lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int each = (rows + BIAS_WAYS - 1) / BIAS_WAYS, first = each * blockIdx.y, last = first + each < rows ? first + each : rows;
    const int64_t v = (int64_t)blockIdx.x * (64 * V) + lane * V;
    float s[V] = {};
    if (v < c.wide)
        for (int r = first + w; r < last; r += 4) {
            const int64_t j = c.first + r, at = (int64_t)r * c.wide + v;
            const Line y = *(const Line *)((const T *)c.e + at);
            Low low = {};
            if constexpr (sizeof(T) == 2) low = *(const Low *)(c.low + at);
            const float inv = c.inv[j], f = c.normed ? c.inv_h[j] : 1.0f;
            const float one = c.normed ? c.one[j] : 0.0f;
            const int64_t t = c.normed ? c.target[j] - v : -1;
#pragma unroll
            for (int k = 0; k < V; ++k) s[k] = __builtin_fmaf(inv, k == t ? one : exponential(y.e[k], low.e[k]) * f, s[k]);
        }
#pragma unroll
    for (int k = 0; k < V; ++k) red[w][lane * V + k] = s[k];
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * V; k += BLOCK) {
        const int64_t at = (int64_t)blockIdx.x * (64 * V) + k;
        if (at < c.width) parts[(int64_t)blockIdx.y * c.width + at] = (red[0][k] + red[1][k]) + (red[2][k] + red[3][k]);
    }
}
__global__ __launch_bounds__(BLOCK) void k_bias_sum(int width, const float *parts, float *out, int add)
{
    const int v = blockIdx.x * BLOCK + threadIdx.x;
    if (v >= width) return;
    float s = 0.0f;
    for (int k = 0; k < BIAS_WAYS; ++k) s += parts[(int64_t)k * width + v];
    out[v] = s + (add ? out[v] : 0.0f);
}

__global__ __launch_bounds__(BLOCK) void k_loss(const Call c)
{
    __shared__ double red[BLOCK / 64];
    const int64_t n = c.n_on ? *c.n_on : c.rows;
    double s = 0;
    for (int64_t k = threadIdx.x; k < (n + c.few - 1) / c.few; k += BLOCK) s += c.sums[k];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = (red[0] + red[1]) + (red[2] + red[3]);
        *c.loss = (float)(n ? -s * (c.sum ? 1.0 : 1.0 / (double)n) : 0.0);
    }
}

// The gradients as the caller has them: times the upstream gradient, rounded once; in place (floats) only
// where that is not 1.  place: of the rows that count, or NULL.
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_give(const float *from, T *to, int64_t n, int dim, const int32_t *place,
                                                const float *up1)
{
    const float f = *up1;
    if ((const void *)from == (const void *)to && f == 1.0f) return;
    if (!place) {
        struct __align__(16) F4 { float e[4]; };
        struct __attribute__((aligned(4 * sizeof(T)))) T4 { T e[4]; };
        for (int64_t k = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) * 4; k < n; k += (int64_t)gridDim.x * BLOCK * 4) {
            if (k + 4 <= n) {
                const F4 x = *(const F4 *)(from + k);
                T4 y;
#pragma unroll
                for (int q = 0; q < 4; ++q) y.e[q] = (T)(f * x.e[q]);
                *(T4 *)(to + k) = y;
            } else {
                for (int64_t q = k; q < n; ++q) to[q] = (T)(f * from[q]);
            }
        }
        return;
    }
    for (int64_t k = (int64_t)blockIdx.x * BLOCK + threadIdx.x; k < n; k += (int64_t)gridDim.x * BLOCK) {
        const int64_t i = k / dim, j = place[i];
        to[k] = j < 0 ? (T)0.0f : (T)(f * from[j * dim + (k - i * dim)]);
    }
}

// ------------------------------------------------------------------ host

template <typename T> struct Tiles;
template <> struct Tiles<bf16> { typedef Tile<bf16, 4, 2, 2, 4> Wide; typedef Tile<bf16, 2, 1, 4, 1> Few; typedef Tile<bf16, 2, 2, 1, 4> Thin; typedef Tile<bf16, 1, 1, 2, 1> Slim; };
template <> struct Tiles<f16> { typedef Tile<f16, 4, 2, 2, 4> Wide; typedef Tile<f16, 2, 1, 4, 1> Few; typedef Tile<f16, 2, 2, 1, 4> Thin; typedef Tile<f16, 1, 1, 2, 1> Slim; };
template <> struct Tiles<float> { typedef Tile<float, 2, 2, 2, 2> Wide; typedef Tile<float, 2, 1, 4, 1> Few; typedef Tile<float, 2, 2, 1, 4> Thin; typedef Tile<float, 1, 1, 2, 1> Slim; };
constexpr int FEW = 32;            // rows of a Few tile
constexpr int THIN_MOST = 64;      // columns of a Thin one (82305 x 1261 float32, 22 columns: 0.77 ms, 1.17 with Wide ones)
constexpr int SLIM_MOST = 64 * 256;  // rows of Slim tiles of logits (3205 x 2038 float32, 3 columns: 159 us, 253 with
                                      // Thin ones, of 256 rows; 20000 rows: alike)
enum { WIDE, FEWER, THIN, SLIM };
constexpr int FEW_JOINED = 2048;   // fewer rows: a workgroup joins the parts of one

int64_t up_to(int64_t n, int64_t k) { return (n + k - 1) / k * k; }

// Where everything lies in the work memory.
struct Plan {
    int size;                 // bytes of an element
    int64_t dim_p, wide, piece, n_parts;
    int shape;
    int64_t pieces;
    bool pad_w, grad, normed;
    uint64_t index, counts, h, z_t, ref, top, inv, inv_h, one, target, sums, flag, parts, e, low, hs, w, split, bias, bytes;
};

// Workgroups of a product: one a compute unit with 128 KiB of LDS, two with 64.
int places(int size) { return size == 2 ? 256 : 512; }

Plan plan_of(const swarp_linear_ce_t *a)
{
    Plan p = {};
    p.size = a->dtype == SWARP_F32 ? 4 : 2;
    const int64_t ke = STEP / p.size, V = a->width, N = a->rows < 1 ? 1 : a->rows, D = a->dim;
    const bool dh = a->d_hidden, dw = a->d_weight;
    p.grad = dh || dw || a->d_bias;
    p.dim_p = up_to(D, ke);
    p.wide = up_to(V, ke);
    p.shape = N <= FEW ? FEWER : V > THIN_MOST ? WIDE : N < SLIM_MOST ? SLIM : THIN;
    const int64_t bm = p.shape >= THIN ? 64 : p.shape == FEWER || p.size == 2 ? 256 : 128;
    const int64_t wm = p.shape == THIN ? 1 : p.shape == FEWER ? 4 : 2;
    // (float32: what there is less of is multiplied, E or h)
    p.normed = p.size == 2 || V < D;
    p.n_parts = (V + bm - 1) / bm * wm;
    // (a piece's parts of sums stay below its exponentials)
    int64_t piece = p.grad ? (int64_t)(PIECE / (uint64_t)(p.wide * p.size)) : (int64_t)(PIECE / 8 / (uint64_t)p.n_parts);
    piece = piece / 256 * 256;
    if (piece < 256) piece = 256;
    if (piece >= N) piece = up_to(N, N < 256 ? 32 : 256);
    p.piece = piece;
    p.pad_w = D * p.size % 16 || ((uintptr_t)a->weight & 15);
    uint64_t at = 0;
    auto room = [&](bool need, uint64_t bytes) {
        const uint64_t here = at;
        if (need) at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.pieces = (N + piece - 1) / piece;
    p.flag = room(true, 4 * p.pieces);
    p.index = room(a->mask, 4 * N);
    p.counts = room(a->mask, 4 * (N / COUNT_ROWS + 1));
    p.h = room(true, (uint64_t)(N + 31) * p.dim_p * p.size);
    p.z_t = room(true, 4 * N);
    p.ref = room(true, 4 * N);
    p.top = room(true, 4 * N);
    p.inv = room(true, 4 * N);
    p.inv_h = room(true, 4 * N);
    p.one = room(p.grad && p.normed, 4 * N);
    p.target = room(true, 4 * N);
    p.sums = room(true, 8 * (N / (piece < FEW_JOINED ? 1 : 64) + 1));
    p.parts = room(true, 8ull * p.n_parts * piece);
    p.w = room(p.pad_w, (uint64_t)V * p.dim_p * p.size);
    p.e = room(p.grad, (uint64_t)piece * p.wide * p.size);
    p.low = room(p.grad && p.size == 2, (uint64_t)piece * p.wide);
    p.hs = room(dw && !p.normed, (uint64_t)piece * p.dim_p * p.size);
    // (twice as many splits as places, of whole tiles: share_of)
    p.split = room(dh || dw, p.size == 2 ? 2ull * places(2) * 256 * 256 * 4 : 2ull * places(4) * 128 * 128 * 4);
    p.bias = room(a->d_bias, 4ull * BIAS_WAYS * V);
    p.bytes = at;
    return p;
}

int blocks_of(int64_t n) { return (int)(n < 1 ? 1 : n > 4096 ? 4096 : n); }

// A kernel may have more LDS than a launch without asking gives; once a device.
bool lds_limit(const void *kernel, int bytes, std::atomic<uint64_t> &done)
{
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return true;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
    done.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

template <typename T, typename C, bool STORE> bool logits(const Call &c, int again, hipStream_t st)
{
    static std::atomic<uint64_t> done{0};
    const bool ok = lds_limit((const void *)k_logits<T, C, STORE>, C::LDS, done);
    const int nm = (c.width + C::BM - 1) / C::BM, nn = (c.piece + C::BN - 1) / C::BN;
    hipLaunchKernelGGL((k_logits<T, C, STORE>), dim3(nm * nn), dim3(C::THREADS), C::LDS, st, c, nm, nn, again);
    return ok;
}
template <typename T, bool STORE> bool logits(const Call &c, int shape, int again, hipStream_t st)
{
    switch (shape) {
    case FEWER: return logits<T, typename Tiles<T>::Few, STORE>(c, again, st);
    case THIN: return logits<T, typename Tiles<T>::Thin, STORE>(c, again, st);
    case SLIM: return logits<T, typename Tiles<T>::Slim, STORE>(c, again, st);
    default: return logits<T, typename Tiles<T>::Wide, STORE>(c, again, st);
    }
}

template <typename T, typename C, bool AK> bool product(const Call &c, const Product &p, int n, hipStream_t st)
{
    static std::atomic<uint64_t> done{0};
    const bool ok = lds_limit((const void *)k_product<T, C, AK>, C::LDS, done);
    hipLaunchKernelGGL((k_product<T, C, AK>), dim3(n), dim3(C::THREADS), C::LDS, st, c, p);
    const int64_t left = c.rows - c.first, rows = left < c.piece ? left : c.piece;
    if (c.n_on || share_of<C>(p.rows_m ? rows : p.m, p.n, (int)(((p.rows_k ? rows : p.k) + C::KE - 1) / C::KE), n).splits > 1)
        hipLaunchKernelGGL((k_splits<C>), dim3(1024), dim3(BLOCK), 0, st, c, p, C::KE, n);
    return ok;
}
template <typename T, bool AK> bool product(const Call &c, const Product &p, bool thin, hipStream_t st)
{
    if constexpr (AK) {
        if (thin) return product<T, typename Tiles<T>::Thin, AK>(c, p, 512, st);
    }
    return product<T, typename Tiles<T>::Wide, AK>(c, p, places(sizeof(T)), st);
}

template <typename T> void join(const Call &c, int how, hipStream_t st)
{
    if (c.few == 1) hipLaunchKernelGGL((k_join<T, 1>), dim3((unsigned)c.piece), dim3(BLOCK), 0, st, c, how);
    else hipLaunchKernelGGL((k_join<T, 64>), dim3((unsigned)((c.piece + 63) / 64)), dim3(BLOCK), 0, st, c, how);
}

template <typename T> int run(const swarp_linear_ce_t *a, hipStream_t st)
{
    const Plan p = plan_of(a);
    char *const mem = (char *)a->work;
    Call c = {};
    c.rows = a->rows;
    c.inner = a->inner;
    c.outer_stride = a->outer_stride;
    c.inner_stride = a->inner_stride;
    c.dim = a->dim;
    c.width = a->width;
    c.dim_p = (int)p.dim_p;
    c.pitch_w = (int)((p.pad_w ? p.dim_p : a->dim) * p.size);
    c.wide = p.wide;
    c.piece = (int)p.piece;
    c.targets32 = a->targets32;
    c.sum = a->sum;
    c.hidden = a->hidden;
    c.weight = a->weight;
    c.bias = a->bias;
    c.targets = a->targets;
    c.logp = a->logp;
    c.loss = a->loss;
    c.h = mem + p.h;
    c.z_t = (float *)(mem + p.z_t);
    c.ref = (float *)(mem + p.ref);
    c.top = (float *)(mem + p.top);
    c.inv = (float *)(mem + p.inv);
    c.inv_h = (float *)(mem + p.inv_h);
    c.one = (float *)(mem + p.one);
    c.target = (int32_t *)(mem + p.target);
    c.sums = (double *)(mem + p.sums);
    c.flag = (int32_t *)(mem + p.flag);
    c.pieces = p.grad ? p.pieces : 0;
    c.normed = p.normed;
    c.parts = (float2 *)(mem + p.parts);
    c.n_parts = (int)p.n_parts;
    c.few = p.piece < FEW_JOINED ? 1 : 64;
    c.w = p.pad_w ? mem + p.w : (const char *)a->weight;
    c.e = p.grad ? mem + p.e : nullptr;
    c.low = (uint8_t *)mem + p.low;
    c.hs = mem + p.hs;
    if (a->mask && a->rows) {
        c.index = (int32_t *)(mem + p.index);
        c.n_on = a->place + a->rows;
        int32_t *const counts = (int32_t *)(mem + p.counts);
        const int blocks = (int)((a->rows + COUNT_ROWS - 1) / COUNT_ROWS);
        hipLaunchKernelGGL(k_count, dim3(blocks), dim3(BLOCK), 0, st, a->rows, a->mask, counts);
        hipLaunchKernelGGL(k_place, dim3(blocks), dim3(BLOCK), 0, st, a->rows, a->mask, counts, (int32_t *)c.index,
                           a->place, (int32_t *)c.n_on, a->logp);
    }
    hipLaunchKernelGGL((k_rows<T>), dim3(blocks_of((a->rows + 3) / 4)), dim3(BLOCK), 0, st, c);
    if (p.pad_w)
        hipLaunchKernelGGL((k_pad<T>), dim3(blocks_of(c.width * p.dim_p / BLOCK)), dim3(BLOCK), 0, st,
                           (const T *)a->weight, (int64_t)c.width, c.dim, (T *)c.w, c.dim_p);
    bool ok = true;
    // (without a row too: the gradients are zeros)
    for (int64_t first = 0, n = 0; n == 0 || first < a->rows; first += p.piece, ++n) {
        c.first = first;
        const dim3 block(BLOCK);
        if (!p.grad) {
            ok &= logits<T, false>(c, p.shape, 0, st);
            join<T>(c, SUMS, st);
            continue;
        }
        c.flag = (int32_t *)(mem + p.flag) + n;
        ok &= logits<T, true>(c, p.shape, 0, st);
        join<T>(c, KEPT, st);
        ok &= logits<T, true>(c, p.shape, 1, st);
        join<T>(c, KEPT2, st);
        if (a->d_bias) {
            float *const sums = (float *)(mem + p.bias);
            const int per = 64 * 16 / sizeof(T);
            hipLaunchKernelGGL((k_bias<T>), dim3((c.width + per - 1) / per, BIAS_WAYS), block, 0, st, c, sums);
            hipLaunchKernelGGL(k_bias_sum, dim3((c.width + BLOCK - 1) / BLOCK), block, 0, st, c.width, sums, a->d_bias, (int)(n > 0));
        }
        if (c.normed) {
            const int64_t n = p.piece * p.wide / 8, each = NORMS * BLOCK;
            hipLaunchKernelGGL((k_norm<T>), dim3((unsigned)((n + each - 1) / each)), block, 0, st, c);
        }
        float *const parts = (float *)(mem + p.split);
        const int64_t pitch_e = c.wide * (int64_t)sizeof(T), pitch_h = c.dim_p * (int64_t)sizeof(T);
        if (a->d_hidden) {
            const Product y = {c.e, c.w, pitch_e, c.pitch_w, p.piece, c.dim, c.width, 1, 0, 0, 1.0f, 0, c.inv + first,
                               a->d_hidden + first * c.dim, parts};
            ok &= product<T, false>(c, y, false, st);
        }
        if (a->d_weight) {
            if (!c.normed) hipLaunchKernelGGL(k_scale, dim3(blocks_of(p.piece / 4)), block, 0, st, c);
            const void *const h = c.normed ? (const char *)c.h + first * pitch_h : c.hs;
            const Product y = {c.e, h, pitch_e, pitch_h, c.width, c.dim, 0, 0, 1, n > 0,
                               c.normed ? 1.0f / (1 << KEPT_BITS) : 1.0f, c.normed, nullptr, a->d_weight, parts};
            ok &= product<T, true>(c, y, p.shape >= THIN, st);
        }
    }
    hipLaunchKernelGGL(k_loss, dim3(1), dim3(BLOCK), 0, st, c);
    const int rc = launched();
    return ok ? rc : fail("the LDS of the matrix products was refused");
}

int check(const swarp_linear_ce_t *a)
{
    swarp::set_error("");
    if (!a) return fail("arguments must be set");
    if (a->dtype != SWARP_F32 && a->dtype != SWARP_BF16 && a->dtype != SWARP_F16) return fail("unknown dtype");
    if (a->rows < 0 || a->rows >= 1ll << 31 || a->dim < 1 || a->dim > 65536 || a->width < 1 || a->width > 1 << 21)
        return fail("bad sizes");
    return 0;
}

template <typename T> void give(const swarp_linear_ce_t *a, const float *scale, void *h, void *w, void *b, hipStream_t st)
{
    const int64_t nh = a->rows * a->dim, nw = (int64_t)a->width * a->dim;
    if (h && nh)
        hipLaunchKernelGGL((k_give<T>), dim3(blocks_of(nh / BLOCK)), dim3(BLOCK), 0, st, (const float *)a->d_hidden, (T *)h,
                           nh, a->dim, (const int32_t *)(a->mask ? a->place : nullptr), scale);
    if (w)
        hipLaunchKernelGGL((k_give<T>), dim3(blocks_of(nw / BLOCK)), dim3(BLOCK), 0, st, (const float *)a->d_weight, (T *)w,
                           nw, a->dim, (const int32_t *)nullptr, scale);
    if (b)
        hipLaunchKernelGGL((k_give<T>), dim3(blocks_of(a->width / BLOCK)), dim3(BLOCK), 0, st, (const float *)a->d_bias,
                           (T *)b, (int64_t)a->width, 1, (const int32_t *)nullptr, scale);
}

// Of a call without gradients, or of one with them.
uint64_t work_of(const swarp_linear_ce_t *a) { return narrow::fits(a) ? narrow::work_bytes(a) : plan_of(a).bytes; }

int ready(const swarp_linear_ce_t *a)
{
    if (!a->work || a->work_bytes < work_of(a)) return fail("work must be set, swarp_linear_ce_work_bytes() long");
    if ((uintptr_t)a->work & 255u) return fail("work must be 256-byte aligned");
    if (!a->weight || a->inner < 1 || (a->rows && (!a->hidden || !a->targets))) return fail("pointer arguments must be set");
    return 0;
}

}  // namespace

extern "C" {

int32_t swarp_linear_ce_complete(const swarp_linear_ce_t *a) { return !check(a) && narrow::fits(a); }

uint64_t swarp_linear_ce_work_bytes(const swarp_linear_ce_t *a)
{
    if (check(a)) return 0;
    return work_of(a);
}

int swarp_linear_ce(const swarp_linear_ce_t *a, void *stream)
{
    if (check(a)) return -1;
    if (!a->loss) return fail("loss must be set");
    if (ready(a)) return -1;
    if (a->rows && !a->logp) return fail("pointer arguments must be set");
    hipStream_t st = (hipStream_t)stream;
    if (narrow::fits(a)) return narrow::run(a, 0, nullptr, a->d_hidden, a->d_weight, a->d_bias, st);
    if (a->rows && a->mask && !a->place) return fail("a mask needs place");
    switch (a->dtype) {
    case SWARP_F32: return run<float>(a, st);
    case SWARP_BF16: return run<bf16>(a, st);
    default: return run<f16>(a, st);
    }
}

int swarp_linear_ce_bwd(const swarp_linear_ce_t *a, int32_t skip_unit, const void *scale, void *d_hidden, void *d_weight,
                        void *d_bias, void *stream)
{
    if (check(a)) return -1;
    if (!scale) return fail("pointer arguments must be set");
    hipStream_t st = (hipStream_t)stream;
    if (narrow::fits(a))
        return ready(a) ? -1 : narrow::run(a, skip_unit, (const float *)scale, d_hidden, d_weight, d_bias, st);
    if ((d_hidden && !a->d_hidden) || (d_weight && !a->d_weight) || (d_bias && !a->d_bias))
        return fail("pointer arguments must be set");
    if (a->rows && a->mask && !a->place) return fail("a mask needs place");
    if (a->dtype != SWARP_F32 && ((d_hidden && d_hidden == a->d_hidden) || (d_weight && d_weight == a->d_weight) ||
                                  (d_bias && d_bias == a->d_bias)))
        return fail("only float gradients are scaled in place");
    if (a->mask && d_hidden && d_hidden == a->d_hidden) return fail("the rows that count are moved, not in place");
    switch (a->dtype) {
    case SWARP_F32: give<float>(a, (const float *)scale, d_hidden, d_weight, d_bias, st); break;
    case SWARP_BF16: give<bf16>(a, (const float *)scale, d_hidden, d_weight, d_bias, st); break;
    default: give<f16>(a, (const float *)scale, d_hidden, d_weight, d_bias, st); break;
    }
    return launched();
}

uint64_t swarp_capture_id(void *stream)
{
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
        (void)hipGetLastError();
        return 0;
    }
    return status == hipStreamCaptureStatusActive ? id + 1 : 0;
}

}  // extern "C"

namespace narrow {

void count(int64_t rows, const uint8_t *mask, int32_t *counts, hipStream_t st)
{
    hipLaunchKernelGGL(k_count, dim3((unsigned)counts_of(rows)), dim3(BLOCK), 0, st, rows, mask, counts);
}

}  // namespace narrow
