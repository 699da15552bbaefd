// decay.hip -- linear attention with a decay for each head, along a rollout (swarp_decay_fwd,
// swarp_decay_bwd, swarp_decay_step).
//
// Per batch entry and head, with the state S [dk, dv] and lambda = exp(log_decay):
//   S_t = (starts_t ? 0 : lambda S_{t-1}) + k_t v_t^T,   o_t = scale q_t S_t.
// Over a chunk of 32 steps that S enters (0 <= t, i < 32, both of one episode where they meet):
//   o_t = scale (sum_{i <= t} lambda^(t-i) (q_t k_i) v_i + lambda^(t+1) q_t S),
//   S' = lambda^32 S + sum_i lambda^(31-i) k_i v_i^T:
// four small matrix products, all powers at most 1.
//
// The gradients are scans of the same kind with the parts exchanged:
//   dq_t = scale sum_{i <= t} lambda^(t-i) (do_t v_i) k_i + ...     forwards,  (do, v, k), state S^T
//   dk_i = scale sum_{t >= i} lambda^(t-i) (v_i do_t) q_t + ...     backwards, (v, do, q), state dS^T
//   dv_i = scale sum_{t >= i} lambda^(t-i) (k_i q_t) do_t + ...     backwards, (k, q, do), state dS
// so that one kernel does all four; below, q, k and v are a scan's own parts.
#include <math.h>

#include "learn.hpp"

namespace {

using namespace learn;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int BLOCK = 256, WAVES = BLOCK / 64;
constexpr int CHUNK = 32;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr int MOST_DIM = 128;

template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Span {
    T e[N];
};

// One of a call's scans.
struct Scan {
    const void *q, *k, *v;
    void *out;
    int64_t qs[3], ks[3], vs[3], os[3];  // elements: step, batch, head
    int dk, dv;                          // of this scan
    int back;                            // from the last step to the first
    int slices;                          // of 32 columns of v
    float score, grow, carry;            // factors of the scores, of k v^T in the state, of q S in the output
    const float *state;                  // element (i, j) at i si + j sj of a head's
    float *state_out;
    int si, sj;
};

struct Call {
    Scan scan[3];
    int scans, slices;     // slices of all scans
    int64_t units;         // waves: batch * heads * slices
    int64_t steps, batch, group;
    int heads, area;       // area: dk dv of a state
    const float *log_decay;
    const uint8_t *starts;
};

// What a lane gives to a product of 32 x 32 over 16 k: row (or column) l % 32, the eight k from
// 8 (l / 32) on.  bfloat16 goes into the matrix cores as it is, sums of it and what is rounded from
// float as two or three terms; the others are multiplied in float (float16 has not the range for the
// states).
template <typename T> struct Part {
    float x[8];
    static constexpr int TERMS = 1;
};
template <> struct Part<bf16> {
    u32x4 w;
    static constexpr int TERMS = 3;
};

__device__ __forceinline__ void mma(f32x16 &acc, const Part<float> &a, const Part<float> &b)
{
#pragma unroll
    for (int k = 0; k < 8; ++k) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x[k], b.x[k], acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16 &acc, const Part<f16> &a, const Part<f16> &b)
{
#pragma unroll
    for (int k = 0; k < 8; ++k) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x[k], b.x[k], acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16 &acc, const Part<bf16> &a, const Part<bf16> &b)
{
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.w), __builtin_bit_cast(bf16x8, b.w),
                                                  acc, 0, 0, 0);
}

template <typename T> __device__ __forceinline__ Part<T> part_of(const T (&e)[8])
{
    Part<T> p;
    if constexpr (sizeof(p) == 16) p.w = __builtin_bit_cast(u32x4, *(const Span<T, 8> *)e);
    else {
#pragma unroll
        for (int k = 0; k < 8; ++k) p.x[k] = (float)e[k];
    }
    return p;
}
// The next term of x, which is left with what remains of it.
template <typename T> __device__ __forceinline__ Part<T> term_of(float (&x)[8])
{
    Part<T> p;
    if constexpr (Part<T>::TERMS == 1) {
#pragma unroll
        for (int k = 0; k < 8; ++k) p.x[k] = x[k];
    } else {
        T e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            e[k] = (T)x[k];
            x[k] -= (float)e[k];
        }
        p = part_of<T>(e);
    }
    return p;
}

// n elements of a row from x on, zero past them.
template <typename T> __device__ __forceinline__ Part<T> row_of(const T *x, int n)
{
    T e[8];
    if (n >= 8) *(Span<T, 8> *)e = *(const Span<T, 8> *)x;
    else {
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = k < n ? x[k] : (T)0.0f;
    }
    return part_of<T>(e);
}

// Row m of a 32 x 32 accumulator is what operand row m was; swapping two bits of the operand's
// rows makes a lane's registers 8 s .. 8 s + 7 stand for the rows 16 s + 8 (l / 32) + 0 .. 7, which is
// how it holds an operand: accumulators go into the next product as they are.
__device__ __forceinline__ int swapped(int m) { return (m & 0x13) | (m & 4) << 1 | (m & 8) >> 1; }

// One wave: one head of a batch entry, 32 columns of v, all steps.  The state's columns stay in its
// registers; KT: 32s of dk.
template <typename T, int KT> __global__ __launch_bounds__(BLOCK) void k_scan(const Call c)
{
    const int64_t unit = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= c.units) return;
    const int64_t bh = unit / c.slices, b = bh / c.heads;
    const int h = (int)(bh - b * c.heads);
    int slice = (int)(unit - bh * c.slices), which = 0;
    while (slice >= c.scan[which].slices) slice -= c.scan[which++].slices;
    const Scan &s = c.scan[which];
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, perm = swapped(col);
    const int64_t steps = c.steps, last = s.back ? steps - 1 : 0, way = s.back ? -1 : 1;
    const int64_t qt = way * s.qs[0], kt = way * s.ks[0], vt = way * s.vs[0], ot = way * s.os[0];
    const T *const q = (const T *)s.q + b * s.qs[1] + h * s.qs[2] + last * s.qs[0];
    const T *const k = (const T *)s.k + b * s.ks[1] + h * s.ks[2] + last * s.ks[0];
    const T *const v = (const T *)s.v + b * s.vs[1] + h * s.vs[2] + last * s.vs[0];
    T *const out = (T *)s.out + b * s.os[1] + h * s.os[2] + last * s.os[0];
    const int dk = s.dk, dv = s.dv, j0 = 32 * slice, j = j0 + perm;
    const bool back = s.back;
    const uint8_t *const starts = c.starts ? c.starts + b / c.group : nullptr;
    const int64_t groups = c.batch / c.group;

    // the state: element (32 t + 16 (r / 8) + 8 half + r % 8, j) in register r of tile t
    f32x16 S[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = 32 * t + 16 * (r >> 3) + 8 * half + (r & 7);
            S[t][r] = s.state && i < dk && j < dv ? s.state[bh * c.area + (int64_t)i * s.si + (int64_t)j * s.sj] : 0.0f;
        }
    // (a product with 0 is not 0 where the state is not finite)
    auto finite = [&]() {
        float z = 0.0f;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) z = __builtin_fmaf(S[t][r], 0.0f, z);
        return __ballot(!(z == 0.0f)) == 0;
    };
    bool plain = finite();

    // powers: of the decay between the steps of a lane's scores, of what a step leaves in the state
    float a2 = c.log_decay[h] * LOG2E;
    a2 = a2 < -1e30f ? -1e30f : a2;  // (-inf times 0 steps is no decay)
    const float lambda = __builtin_amdgcn_exp2f(a2);
    float D[16], u[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int i = 16 * (r >> 3) + 8 * half + (r & 7);
        D[r] = col >= i ? s.score * __builtin_amdgcn_exp2f(a2 * (float)(col - i)) : 0.0f;
    }
    const float w0 = s.carry * __builtin_amdgcn_exp2f(a2 * (float)(col + (back ? 0 : 1)));
    float whole = 0.0f;
    int width = 0;  // of the chunk that u and whole are for

    for (int64_t c0 = 0; c0 < steps; c0 += CHUNK) {
        const int L = (int)(steps - c0 < CHUNK ? steps - c0 : CHUNK);
        if (L != width) {
            width = L;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = 16 * (r >> 3) + 8 * half + (r & 7);
                u[r] = i < L ? s.grow * __builtin_amdgcn_exp2f(a2 * (float)(L - 1 - i + (back ? 1 : 0))) : 0.0f;
            }
            whole = __builtin_amdgcn_exp2f(a2 * (float)L);
        }
        // steps that nothing before them enters
        uint32_t cut = 0;
        if (starts) {
            const int64_t t = back ? steps - (c0 + col) : c0 + col;
            cut = (uint32_t)__ballot(half == 0 && col < L && (!back || c0 + col > 0) && starts[t * groups]);
        }
        const uint32_t upto = cut & (0xffffffffu >> (31 - col));
        const int since = upto ? 31 - __clz(upto) : -1;               // first step that enters step `col`
        const int kept = cut ? 31 - __clz(cut) : -1;                  // ... the leaving state

        Part<T> qf[2 * KT], vf[2];
        f32x16 p = {};
        const T *const qr = q + (c0 + (col < L ? col : 0)) * qt, *const kr = k + (c0 + (perm < L ? perm : 0)) * kt;
#pragma unroll
        for (int x = 0; x < 2 * KT; ++x) {
            const int at = 16 * x + 8 * half;
            qf[x] = row_of<T>(qr + at, col < L ? dk - at : 0);
            const Part<T> kf = row_of<T>(kr + at, perm < L ? dk - at : 0);
            mma(p, kf, qf[x]);
        }
        float vx[16], odd = 0.0f;
        {
            T e[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = 16 * (r >> 3) + 8 * half + (r & 7);
                e[r] = i < L && j < dv ? v[(c0 + i) * vt + j] : (T)0.0f;
                vx[r] = (float)e[r];
                odd = __builtin_fmaf(vx[r], 0.0f, odd);
            }
            vf[0] = part_of<T>(*(const T(*)[8])e);
            vf[1] = part_of<T>(*(const T(*)[8])(e + 8));
        }
        // (a score is not finite wherever its q or k is not)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd = __builtin_fmaf(p[r], 0.0f, odd);
        Part<T> kc[KT][2];  // columns of k
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                T e[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int i = 16 * x + 8 * half + r;
                    e[r] = i < L && 32 * t + perm < dk ? k[(c0 + i) * kt + 32 * t + perm] : (T)0.0f;
                }
                kc[t][x] = part_of<T>(e);
            }
        if (plain && __ballot(!(odd == 0.0f)) == 0) {
            f32x16 o = {};
#pragma unroll
            for (int x = 0; x < 2 * KT; ++x) {
                float y[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) y[r] = S[x >> 1][8 * (x & 1) + r];
#pragma unroll
                for (int n = 0; n < (Part<T>::TERMS + 1) / 2; ++n) mma(o, term_of<T>(y), qf[x]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) o[r] = since < 0 ? o[r] * w0 : 0.0f;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float y[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int i = 16 * x + 8 * half + r;
                    // (a select: a step that is not open may hold anything)
                    y[r] = i <= col && i >= since ? p[8 * x + r] * D[8 * x + r] : 0.0f;
                }
#pragma unroll
                for (int n = 0; n < (Part<T>::TERMS + 1) / 2; ++n) mma(o, vf[x], term_of<T>(y));
            }
            if (col < L) {
                T *const to = out + (c0 + col) * ot + j0;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int at = 16 * x + 8 * half, n = dv - j0 - at;
                    T e[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) e[r] = (T)o[8 * x + r];
                    if (n >= 8) *(Span<T, 8> *)(to + at) = *(const Span<T, 8> *)e;
                    else {
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (r < n) to[at + r] = e[r];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[t][r] = cut ? 0.0f : S[t][r] * whole;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float y[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) y[r] = 16 * x + 8 * half + r >= kept ? vx[8 * x + r] * u[8 * x + r] : 0.0f;
#pragma unroll
                for (int n = 0; n < Part<T>::TERMS; ++n) {
                    const Part<T> w = term_of<T>(y);
#pragma unroll
                    for (int t = 0; t < KT; ++t) mma(S[t], kc[t][x], w);
                }
            }
        } else {
            // something is not finite: step by step, as the definition has it
            for (int i = 0; i < L; ++i) {
                const float vi = j < dv ? (float)v[(c0 + i) * vt + j] : 0.0f;
                const bool fresh = cut >> i & 1;
                float o = 0.0f;
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int at = 32 * t + 16 * (r >> 3) + 8 * half + (r & 7);
                        if (at < dk) {
                            const float kv = (float)k[(c0 + i) * kt + at] * vi * s.grow;
                            const float y = fresh ? kv : __builtin_fmaf(back ? 1.0f : lambda, S[t][r], kv);
                            o = __builtin_fmaf((float)q[(c0 + i) * qt + at], y, o);
                            S[t][r] = back ? lambda * y : y;
                        }
                    }
                o += __shfl_xor(o, 32, 64);
                if (half == 0 && j < dv) out[(c0 + i) * ot + j] = (T)(o * s.carry);
            }
            plain = finite();
        }
    }
    if (s.state_out) {
        // (backwards: what an episode that starts with the first step leaves of the state before it)
        const bool none = back && starts && steps > 0 && starts[0];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = 32 * t + 16 * (r >> 3) + 8 * half + (r & 7);
                if (i < dk && j < dv)
                    s.state_out[bh * c.area + (int64_t)i * s.si + (int64_t)j * s.sj] = none ? 0.0f : S[t][r];
            }
    }
}

// One step: a thread a column of v, all of dk in turn; the state is read and written once.
template <typename T> __global__ __launch_bounds__(BLOCK) void k_step(const swarp_decay_t a, int64_t n)
{
    for (int64_t x = (int64_t)blockIdx.x * BLOCK + threadIdx.x; x < n; x += (int64_t)gridDim.x * BLOCK) {
        const int64_t bh = x / a.dv, b = bh / a.heads;
        const int j = (int)(x - bh * a.dv), h = (int)(bh - b * a.heads);
        const T *const q = (const T *)a.q + b * a.q_stride[1] + h * a.q_stride[2];
        const T *const k = (const T *)a.k + b * a.k_stride[1] + h * a.k_stride[2];
        const float v = (float)((const T *)a.v)[b * a.v_stride[1] + h * a.v_stride[2] + j];
        const bool fresh = !a.state || (a.starts && a.starts[b / a.group]);
        const float lambda = __builtin_amdgcn_exp2f(a.log_decay[h] * LOG2E);
        const int64_t at = bh * a.dk * a.dv + j;
        float o = 0.0f;
        for (int i = 0; i < a.dk; ++i) {
            const int64_t e = at + (int64_t)i * a.dv;
            const float kv = (float)k[i] * v;
            const float s = fresh ? kv : __builtin_fmaf(lambda, a.state[e], kv);
            a.state_out[e] = s;
            o = __builtin_fmaf((float)q[i], s, o);
        }
        ((T *)a.out)[x] = (T)(o * (float)a.scale);
    }
}

int check(const swarp_decay_t *a)
{
    swarp::set_error("");
    if (!a) return fail("arguments must be set");
    if (a->dtype != SWARP_F32 && a->dtype != SWARP_BF16 && a->dtype != SWARP_F16) return fail("unknown dtype");
    if (a->steps < 0 || a->batch < 0 || a->heads < 1 || a->dk < 1 || a->dk > MOST_DIM || a->dv < 1 ||
        a->dv > MOST_DIM || a->group < 1 || a->batch % a->group)
        return fail("bad sizes");
    if (a->batch * a->heads > 1ll << 31 || a->steps > 1ll << 40) return fail("bad sizes");
    return 0;
}

void strides(int64_t (&to)[3], const swarp_decay_t *a, int d)
{
    to[0] = a->batch * a->heads * d;
    to[1] = (int64_t)a->heads * d;
    to[2] = d;
}
void copy(int64_t (&to)[3], const int64_t *from)
{
    for (int i = 0; i < 3; ++i) to[i] = from[i];
}

Call call_of(const swarp_decay_t *a)
{
    Call c = {};
    c.steps = a->steps;
    c.batch = a->batch;
    c.group = a->group;
    c.heads = a->heads;
    c.area = a->dk * a->dv;
    c.log_decay = a->log_decay;
    c.starts = a->starts;
    return c;
}

template <typename T> void launch(Call &c, hipStream_t st)
{
    int kt = 0;
    c.slices = 0;
    for (int i = 0; i < c.scans; ++i) {
        c.scan[i].slices = (c.scan[i].dv + 31) / 32;
        c.slices += c.scan[i].slices;
        if ((c.scan[i].dk + 31) / 32 > kt) kt = (c.scan[i].dk + 31) / 32;
    }
    c.units = c.batch * c.heads * c.slices;
    const dim3 grid((unsigned)((c.units + WAVES - 1) / WAVES));
    if (kt == 1) hipLaunchKernelGGL((k_scan<T, 1>), grid, dim3(BLOCK), 0, st, c);
    else if (kt == 2) hipLaunchKernelGGL((k_scan<T, 2>), grid, dim3(BLOCK), 0, st, c);
    else hipLaunchKernelGGL((k_scan<T, 4>), grid, dim3(BLOCK), 0, st, c);
}

int launch(const swarp_decay_t *a, Call &c, hipStream_t st)
{
    switch (a->dtype) {
    case SWARP_F32: launch<float>(c, st); break;
    case SWARP_BF16: launch<bf16>(c, st); break;
    default: launch<f16>(c, st); break;
    }
    return launched();
}

}  // namespace

extern "C" {

uint64_t swarp_decay_work_bytes(const swarp_decay_t *a) { return check(a) ? 0 : 256; }

int swarp_decay_fwd(const swarp_decay_t *a, void *stream)
{
    if (check(a)) return -1;
    if (!a->batch) return 0;
    if (!a->log_decay || (a->steps && (!a->q || !a->k || !a->v || !a->out))) return fail("pointer arguments must be set");
    Call c = call_of(a);
    Scan &s = c.scan[0];
    s.q = a->q;
    s.k = a->k;
    s.v = a->v;
    s.out = a->out;
    copy(s.qs, a->q_stride);
    copy(s.ks, a->k_stride);
    copy(s.vs, a->v_stride);
    strides(s.os, a, a->dv);
    s.dk = a->dk;
    s.dv = a->dv;
    s.score = s.carry = (float)a->scale;
    s.grow = 1.0f;
    s.state = a->state;
    s.state_out = a->state_out;
    s.si = a->dv;
    s.sj = 1;
    c.scans = 1;
    return launch(a, c, (hipStream_t)stream);
}

int swarp_decay_bwd(const swarp_decay_t *a, void *stream)
{
    if (check(a)) return -1;
    if (!a->batch) return 0;
    if (!a->log_decay || (a->steps && (!a->q || !a->k || !a->v || !a->adj_out)))
        return fail("pointer arguments must be set");
    if (!a->d_q != !a->d_k || !a->d_q != !a->d_v) return fail("d_q, d_k and d_v are set together");
    Call c = call_of(a);
    const float scale = (float)a->scale;
    Scan q = {}, k = {}, v = {};
    q.q = k.k = v.v = a->adj_out;
    strides(q.qs, a, a->dv);
    strides(k.ks, a, a->dv);
    strides(v.vs, a, a->dv);
    q.k = k.q = a->v;
    copy(q.ks, a->v_stride);
    copy(k.qs, a->v_stride);
    q.v = v.q = a->k;
    copy(q.vs, a->k_stride);
    copy(v.qs, a->k_stride);
    k.v = v.k = a->q;
    copy(k.vs, a->q_stride);
    copy(v.ks, a->q_stride);
    q.out = a->d_q;
    k.out = a->d_k;
    v.out = a->d_v;
    strides(q.os, a, a->dk);
    strides(k.os, a, a->dk);
    strides(v.os, a, a->dv);
    q.dk = k.dk = v.dv = a->dv;
    q.dv = k.dv = v.dk = a->dk;
    q.score = k.score = v.score = scale;
    q.carry = k.grow = v.grow = scale;
    q.grow = k.carry = v.carry = 1.0f;
    k.back = v.back = 1;
    q.state = a->state;
    k.state = v.state = a->adj_state;
    v.state_out = a->d_state;
    q.si = k.si = v.sj = 1;
    q.sj = k.sj = v.si = a->dv;
    c.scan[0] = q;
    c.scan[1] = k;
    c.scan[2] = v;
    c.scans = 3;
    return launch(a, c, (hipStream_t)stream);
}

int swarp_decay_step(const swarp_decay_t *a, void *stream)
{
    if (check(a)) return -1;
    if (!a->batch) return 0;
    if (a->steps != 1) return fail("a step is one step");
    if (!a->log_decay || !a->q || !a->k || !a->v || !a->out || !a->state_out)
        return fail("pointer arguments must be set");
    hipStream_t st = (hipStream_t)stream;
    const int64_t n = a->batch * a->heads * a->dv;
    const dim3 grid((unsigned)((n + BLOCK - 1) / BLOCK < 16384 ? (n + BLOCK - 1) / BLOCK : 16384));
    switch (a->dtype) {
    case SWARP_F32: hipLaunchKernelGGL((k_step<float>), grid, dim3(BLOCK), 0, st, *a, n); break;
    case SWARP_BF16: hipLaunchKernelGGL((k_step<bf16>), grid, dim3(BLOCK), 0, st, *a, n); break;
    default: hipLaunchKernelGGL((k_step<f16>), grid, dim3(BLOCK), 0, st, *a, n); break;
    }
    return launched();
}

}  // extern "C"
