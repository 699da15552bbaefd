// adamw.hip -- an AdamW step over many tensors (swarp_adamw), its 8-bit moments as floats
// (swarp_adamw_unpack) and the norm of all gradients (swarp_grad_norm).
//
// The tensors of a launch travel in its arguments, up to MOST_TENSORS of them; a workgroup finds
// its own from a running count of chunks.
//
// 8-bit moments.  A group of 256 elements shares a base; a code is the float's bits from the
// third bit of the mantissa up, less the base's exponent: all integer work, the same on any
// machine.  beta2 = 0.999 moves v by a thousandth a step, and a code's step is an eighth: rounded
// to nearest, v would never fall and hardly rise.  Rounded up or down at random in proportion
// (16 random bits from the element's place and the step's seed), its mean is right.
#include <math.h>

#include "learn.hpp"

namespace {

using namespace learn;

constexpr int GROUP = SWARP_ADAMW_GROUP;
constexpr int BLOCK = GROUP;
constexpr int CHUNK = 8 * GROUP;         // elements of a workgroup
constexpr int MOST_TENSORS = 64;         // of a launch
constexpr uint32_t MOST_CHUNKS = (1u << 24) - 1;  // of a step's launch: below 2^32 threads
constexpr int NORM_BLOCKS = 1024;

struct Tensors {
    void *param[MOST_TENSORS];
    const void *grad[MOST_TENSORS];
    int64_t n[MOST_TENSORS], slot[MOST_TENSORS];
    uint32_t first[MOST_TENSORS];  // the tensor's first chunk
    int count;
};

// The tensor of chunk `c`.
__device__ __forceinline__ int tensor_of(const Tensors &t, uint32_t c)
{
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int m = (lo + hi) / 2;
        if (t.first[m] <= c) lo = m;
        else hi = m;
    }
    return lo;
}

struct Step {
    float b1, a1, b2, a2;     // beta1, 1 - beta1, beta2, 1 - beta2
    float lr_t, v_t, eps, keep;  // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), eps, 1 - lr wd
    uint32_t seed;
    int careful;  // whether the root of a v below the smallest normal number counts beside eps
    void *m, *v;
    uint8_t *m_base, *v_base;
    float *master;
    const float *scale;
};

// One round of multiply and shift; the multipliers here and below are the odd integers at 2^32
// times the fractional parts of sqrt(3), sqrt(7), the golden ratio and sqrt(5).
__device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x *= 0xBB67AE85u;
    x ^= x >> 15;
    x *= 0xA54FF53Bu;
    return x ^ (x >> 16);
}
// 32 random bits of element i of the flat state are mix(place_of(i, seed)); i + 1 of the same 2^32
// is a PLACE further.
constexpr uint32_t PLACE = 0x9E3779B1u;
__device__ __forceinline__ uint32_t place_of(uint64_t i, uint32_t seed)
{
    return (uint32_t)i * PLACE + seed + (uint32_t)(i >> 32) * 0x3C6EF373u;
}

__device__ __forceinline__ uint32_t bits_of(float x) { return (uint32_t)__float_as_int(x); }
__device__ __forceinline__ float float_of(uint32_t b) { return __int_as_float((int)b); }

// The base of a group whose largest magnitude, rounded up to a code, has the exponent e.
__device__ __forceinline__ uint32_t base_of(uint32_t e, uint32_t reach) { return e > reach ? e - reach : 0; }
__device__ __forceinline__ uint32_t magnitude(float x)
{
    const uint32_t m = bits_of(x) & 0x7fffffffu;
    return m < 0x7ff00000u ? m : 0x7ff00000u;
}
__device__ __forceinline__ uint32_t encode(uint32_t mag, uint32_t base, uint32_t r16)
{
    const int k = (int)((mag + (r16 << 4 | 8u)) >> 20) - (int)(base << 3);
    return (uint32_t)(k > 0 ? k : 0);
}
__device__ __forceinline__ float decode(uint32_t q, uint32_t base)
{
    const uint32_t b = (q + (base << 3)) << 20;
    return float_of(q ? b : 0u);
}
__device__ __forceinline__ float decode_m(uint32_t c, uint32_t base)
{
    const float x = decode(c & 127u, base);
    return float_of(bits_of(x) | (c & 128u) << 24);
}

// Both exponents of a group's largest magnitudes, rounded up to a code: one reduction over the wave
// for the two, as halves of a word.
typedef unsigned short Pair __attribute__((ext_vector_type(2)));
__device__ __forceinline__ Pair wave_max(Pair e)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
        e = __builtin_elementwise_max(e, __builtin_bit_cast(Pair, __shfl_xor(__builtin_bit_cast(int, e), d, 64)));
    return e;
}
__device__ __forceinline__ uint32_t exponent(uint32_t mag) { return (mag + 0xfffffu) >> 23; }

// A parameter without a master copy: bfloat16 at random, in proportion (a NaN stays one).
template <typename P> __device__ __forceinline__ P rounded(float x, uint32_t r)
{
    if constexpr (__is_same(P, bf16)) {
        const uint32_t b = x != x ? 0x7fc00000u : bits_of(x);
        return __builtin_bit_cast(bf16, (uint16_t)((b + (mix(r) & 0xffffu)) >> 16));
    } else {
        return (P)x;
    }
}

template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Span {
    T e[N];
};
// The four elements from p[i] on, those below n; 0 for the others.
template <typename T> __device__ __forceinline__ void get(float (&x)[4], const T *p, uint32_t i, int64_t n)
{
    if ((int64_t)i + 4 <= n) {
        const Span<T, 4> y = *(const Span<T, 4> *)(p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (float)y.e[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (int64_t)i + k < n ? (float)p[i + k] : 0.0f;
    }
}

// A workgroup takes a chunk of a tensor, a wave two groups of it, a thread four neighbouring
// elements of each group: all loads of both groups are in flight before the first is used, and a
// group's largest exponents are found without LDS or barriers.  (100 M float32 parameters with two
// groups a wave 490 us, with four 504; 150 M bfloat16 with 8-bit moments 378 and 405.)
// What bounds it: 32-bit moments, memory: 28 bytes a parameter at 5.6 TB/s (100 M in 490 to 504 us,
// by the card).  8-bit ones, the vector units, which are busy 0.9 of the time: some 80 instructions a
// parameter, the random bits' multiplications, the root and the reciprocal at a quarter of the
// rate; 10 bytes a parameter at 3.9 TB/s.  100 M bfloat16 parameters with 32-bit moments take 414 us,
// with a master copy 526; float16 ones with a master copy and 8-bit moments 324.
struct Yes {
    constexpr operator bool() const { return true; }
};
struct No {
    constexpr operator bool() const { return false; }
};
constexpr int WAVE_GROUPS = CHUNK / GROUP / (BLOCK / 64);

template <typename P, typename G, int BITS>
__global__ __launch_bounds__(BLOCK) void k_adamw(const Step s, const Tensors t)
{
    const int k = tensor_of(t, blockIdx.x);
    P *const param = (P *)t.param[k];
    const G *const grad = (const G *)t.grad[k];
    const int64_t n = t.n[k], slot = t.slot[k];
    const int wave = threadIdx.x >> 6;
    const uint32_t at = 4 * (threadIdx.x & 63);
    const int64_t begin = (int64_t)(blockIdx.x - t.first[k]) * CHUNK + wave * (WAVE_GROUPS * GROUP);
    const float scale = s.scale ? *s.scale : 1.0f;
    float g[WAVE_GROUPS][4], m[WAVE_GROUPS][4], v[WAVE_GROUPS][4], w[WAVE_GROUPS][4];
    uint32_t mc[WAVE_GROUPS], vc[WAVE_GROUPS], mb[WAVE_GROUPS], vb[WAVE_GROUPS];
#pragma unroll
    for (int u = 0; u < WAVE_GROUPS; ++u) {
        const int64_t i0 = begin + u * GROUP, j0 = slot + i0;
        if (i0 >= n) break;
        get(g[u], grad + i0, at, n - i0);
        if (BITS == 8) {
            mc[u] = *(const uint32_t *)((const uint8_t *)s.m + j0 + at);
            vc[u] = *(const uint32_t *)((const uint8_t *)s.v + j0 + at);
            mb[u] = s.m_base[j0 / GROUP];
            vb[u] = s.v_base[j0 / GROUP];
        } else {
            // (the state goes on to the end of the group)
            const float4 a = *(const float4 *)((const float *)s.m + j0 + at);
            const float4 b = *(const float4 *)((const float *)s.v + j0 + at);
            m[u][0] = a.x, m[u][1] = a.y, m[u][2] = a.z, m[u][3] = a.w;
            v[u][0] = b.x, v[u][1] = b.y, v[u][2] = b.z, v[u][3] = b.w;
        }
        if (s.master) {
            const float4 a = *(const float4 *)(s.master + j0 + at);
            w[u][0] = a.x, w[u][1] = a.y, w[u][2] = a.z, w[u][3] = a.w;
        } else {
            get(w[u], param + i0, at, n - i0);
        }
    }
    // One group, whose last elements may be past the tensor's end where it is not `whole`.
    const auto one = [&](int u, auto whole) {
        const int64_t i0 = begin + u * GROUP, j0 = slot + i0;
        const int left = whole ? GROUP : (int)(n - i0);
        uint32_t r[4], mt = 0, vt = 0;
        const uint32_t place = place_of((uint64_t)j0, s.seed) + at * PLACE;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (BITS == 8) {
                m[u][e] = decode_m(mc[u] >> 8 * e & 255u, mb[u]);
                v[u][e] = decode(vc[u] >> 8 * e & 255u, vb[u]);
            }
            const float x = s.scale ? g[u][e] * scale : g[u][e];
            m[u][e] = m[u][e] * s.b1 + x * s.a1;
            v[u][e] = v[u][e] * s.b2 + x * x * s.a2;
        }
        // (the root and the quotient to an ulp or two: a fraction of an update that is itself a
        // thousandth of the parameter; the moments, which accumulate, are exact.  The instruction
        // takes a v below the smallest normal number for 0: one it matters for is scaled)
        float root[4];
        if (s.careful) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool tiny = v[u][e] < 0x1p-96f;
                root[e] = __builtin_amdgcn_sqrtf(tiny ? v[u][e] * 0x1p32f : v[u][e]) * (tiny ? 0x1p-16f : 1.0f);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) root[e] = __builtin_amdgcn_sqrtf(v[u][e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float den = __builtin_fmaf(root[e], s.v_t, s.eps);
            w[u][e] = __builtin_fmaf(-s.lr_t, m[u][e] * __builtin_amdgcn_rcpf(den), w[u][e] * s.keep);
            r[e] = mix(place + (uint32_t)e * PLACE);
            if (BITS == 8 && (whole || (int)at + e < left)) {
                const uint32_t a = magnitude(m[u][e]), b = magnitude(v[u][e]);
                mt = a > mt ? a : mt;
                vt = b > vt ? b : vt;
            }
        }
        if (BITS == 8) {
            const Pair top = wave_max(Pair{(unsigned short)exponent(mt), (unsigned short)exponent(vt)});
            const uint32_t mbase = base_of(top.x, 15), vbase = base_of(top.y, 31);
            uint32_t a = 0, b = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t vm = magnitude(v[u][e]);
                const uint32_t x = encode(magnitude(m[u][e]), mbase, r[e] >> 16) | (bits_of(m[u][e]) >> 24 & 128u);
                const uint32_t c = encode(vm, vbase, r[e] & 0xffffu), least = vm < 1u ? vm : 1u;
                const uint32_t y = c > least ? c : least;
                if (whole || (int)at + e < left) {
                    a |= x << 8 * e;
                    b |= y << 8 * e;
                }
            }
            *(uint32_t *)((uint8_t *)s.m + j0 + at) = a;
            *(uint32_t *)((uint8_t *)s.v + j0 + at) = b;
            if (at == 0) {
                s.m_base[j0 / GROUP] = (uint8_t)mbase;
                s.v_base[j0 / GROUP] = (uint8_t)vbase;
            }
        } else {
            *(float4 *)((float *)s.m + j0 + at) = make_float4(m[u][0], m[u][1], m[u][2], m[u][3]);
            *(float4 *)((float *)s.v + j0 + at) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
        }
        Span<P, 4> o;
        if (s.master) {
            *(float4 *)(s.master + j0 + at) = make_float4(w[u][0], w[u][1], w[u][2], w[u][3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o.e[e] = (P)w[u][e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o.e[e] = rounded<P>(w[u][e], r[e]);
        }
        if (whole || (int)at + 4 <= left) {
            *(Span<P, 4> *)(param + i0 + at) = o;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((int)at + e < left) param[i0 + at + e] = o.e[e];
        }
    };
#pragma unroll
    for (int u = 0; u < WAVE_GROUPS; ++u) {
        const int64_t i0 = begin + u * GROUP;
        if (i0 >= n) break;
        if (i0 + GROUP <= n) one(u, Yes());
        else one(u, No());
    }
}

// A thread writes four neighbouring elements of each moment, so that a wave writes whole lines.
__global__ __launch_bounds__(BLOCK) void k_unpack(int64_t groups, const uint8_t *m, const uint8_t *v,
                                                  const uint8_t *m_base, const uint8_t *v_base,
                                                  float *avg, float *sq)
{
    const int lane = threadIdx.x & 63;
    for (int64_t q = (int64_t)blockIdx.x * (BLOCK / 64) + (threadIdx.x >> 6); q < groups;
         q += (int64_t)gridDim.x * (BLOCK / 64)) {
        const int64_t j = q * GROUP + 4 * lane;
        const uint32_t a = *(const uint32_t *)(m + j), b = *(const uint32_t *)(v + j);
        const uint32_t mb = m_base[q], vb = v_base[q];
        *(float4 *)(avg + j) = make_float4(decode_m(a & 255u, mb), decode_m(a >> 8 & 255u, mb),
                                           decode_m(a >> 16 & 255u, mb), decode_m(a >> 24, mb));
        *(float4 *)(sq + j) = make_float4(decode(b & 255u, vb), decode(b >> 8 & 255u, vb),
                                          decode(b >> 16 & 255u, vb), decode(b >> 24, vb));
    }
}

template <typename G>
__global__ __launch_bounds__(BLOCK) void k_norm(const Tensors t, uint32_t chunks, double *sums, int set)
{
    __shared__ double red[BLOCK / 64];
    double s = 0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        const G *const grad = (const G *)t.grad[k];
        const int64_t begin = (int64_t)(c - t.first[k]) * CHUNK;
        const int64_t end = begin + CHUNK < t.n[k] ? begin + CHUNK : t.n[k];
        float part = 0;
#pragma unroll
        for (int u = 0; u < CHUNK / (4 * BLOCK); ++u) {
            const int64_t i = begin + (u * BLOCK + threadIdx.x) * 4;
            float g[4];
            get(g, grad + begin, (uint32_t)(i - begin), end - begin);
            part += g[0] * g[0] + g[1] * g[1] + (g[2] * g[2] + g[3] * g[3]);
        }
        s += part;
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < BLOCK / 64; ++w) s += red[w];
        sums[blockIdx.x] = (int)blockIdx.x < set ? sums[blockIdx.x] + s : s;
    }
}

__global__ __launch_bounds__(BLOCK) void k_norm_finish(int blocks, const double *sums, float most, float *out)
{
    __shared__ double red[BLOCK / 64];
    double s = 0;
    for (int b = threadIdx.x; b < blocks; b += BLOCK) s += sums[b];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < BLOCK / 64; ++w) s += red[w];
        const float norm = (float)sqrt(s);
        const float c = most / (norm + 1e-6f);
        out[0] = norm;
        out[1] = c > 1.0f ? 1.0f : c;
    }
}

// ------------------------------------------------------------------------------ host side

int check(const swarp_adamw_t *a)
{
    if (!a) return fail("arguments must be set");
    if (a->bits != 32 && a->bits != 8) return fail("bits must be 32 or 8");
    if (a->state_len < 0 || a->state_len % GROUP) return fail("state_len must be a multiple of 256");
    if (a->state_len && (!a->exp_avg || !a->exp_avg_sq)) return fail("the moments must be set");
    if (((uintptr_t)a->exp_avg | (uintptr_t)a->exp_avg_sq | (uintptr_t)a->master) & 15u)
        return fail("the state must be 16-byte aligned");
    if (a->bits == 8 && a->state_len && (!a->avg_base || !a->sq_base))
        return fail("8-bit moments need their bases");
    return 0;
}

int check(const swarp_tensor_t *t, int n)
{
    if (n < 0 || (n && !t)) return fail("tensors must be set");
    for (int k = 0; k < n; ++k) {
        if (t[k].n < 0 || t[k].n > (int64_t)CHUNK << 30) return fail("a tensor's size is out of range");
        if (t[k].n && !t[k].grad) return fail("a tensor has no gradient");
        const int d = t[k].grad_dtype;
        if (d != SWARP_F32 && d != SWARP_BF16 && d != SWARP_F16)
            return fail("gradients are float32, bfloat16 or float16");
    }
    return 0;
}

// Fills the table with the tensors from `k` on that `take` accepts, as many as it holds and `most`
// chunks (none has more by itself); returns where to go on.
template <typename Take>
int fill(Tensors &t, uint32_t &chunks, const swarp_tensor_t *x, int n, int k, uint32_t most, Take take)
{
    t.count = 0;
    chunks = 0;
    for (; k < n && t.count < MOST_TENSORS; ++k) {
        if (x[k].n == 0 || !take(x[k])) continue;
        const uint64_t c = (uint64_t)((x[k].n + CHUNK - 1) / CHUNK);
        if (chunks + c > most) break;
        t.param[t.count] = x[k].param;
        t.grad[t.count] = x[k].grad;
        t.n[t.count] = x[k].n;
        t.slot[t.count] = x[k].slot;
        t.first[t.count] = chunks;
        chunks += (uint32_t)c;
        ++t.count;
    }
    return k;
}

template <typename P, typename G>
void steps(const Step &s, int bits, const swarp_tensor_t *x, int n, int pd, int gd, hipStream_t st)
{
    Tensors t;
    uint32_t chunks;
    for (int k = 0; k < n;) {
        k = fill(t, chunks, x, n, k, MOST_CHUNKS, [&](const swarp_tensor_t &y) { return y.param_dtype == pd && y.grad_dtype == gd; });
        if (!t.count) continue;
        if (bits == 8)
            hipLaunchKernelGGL((k_adamw<P, G, 8>), dim3(chunks), dim3(BLOCK), 0, st, s, t);
        else
            hipLaunchKernelGGL((k_adamw<P, G, 32>), dim3(chunks), dim3(BLOCK), 0, st, s, t);
    }
}

}  // namespace

extern "C" {

int swarp_adamw(const swarp_adamw_t *a, const swarp_tensor_t *tensors, int32_t n_tensors, void *stream)
{
    swarp::set_error("");
    if (check(a) || check(tensors, n_tensors)) return -1;
    if (a->step < 1) return fail("step must be >= 1");
    for (int k = 0; k < n_tensors; ++k) {
        const swarp_tensor_t &x = tensors[k];
        if (x.n == 0) continue;
        if (!x.param) return fail("a tensor has no parameter");
        if (x.n > (int64_t)CHUNK * MOST_CHUNKS) return fail("a tensor's size is out of range");
        if (x.param_dtype != SWARP_F32 && x.param_dtype != SWARP_BF16 && x.param_dtype != SWARP_F16)
            return fail("parameters are float32, bfloat16 or float16");
        if (x.grad_dtype != x.param_dtype && x.grad_dtype != SWARP_F32)
            return fail("a gradient has its parameter's type, or float32");
        if (x.param_dtype == SWARP_F16 && !a->master) return fail("float16 parameters need a master copy");
        if (x.slot < 0 || x.slot % GROUP || x.slot > a->state_len || (x.n + GROUP - 1) / GROUP > (a->state_len - x.slot) / GROUP)
            return fail("a tensor's slot is outside the state");
    }
    Step s;
    const double c1 = 1.0 - pow(a->beta1, (double)a->step), c2 = 1.0 - pow(a->beta2, (double)a->step);
    s.b1 = (float)a->beta1;
    s.a1 = (float)(1.0 - a->beta1);
    s.b2 = (float)a->beta2;
    s.a2 = (float)(1.0 - a->beta2);
    s.lr_t = (float)(a->lr / c1);
    s.v_t = (float)(1.0 / sqrt(c2));
    s.eps = (float)a->eps;
    s.careful = s.v_t * 0x1p-63f > s.eps * 0x1p-25f;
    s.keep = (float)(1.0 - a->lr * a->weight_decay);
    s.seed = a->seed;
    s.m = a->exp_avg;
    s.v = a->exp_avg_sq;
    s.m_base = a->avg_base;
    s.v_base = a->sq_base;
    s.master = a->master;
    s.scale = a->grad_scale;
    hipStream_t st = (hipStream_t)stream;
    const int b = a->bits, n = n_tensors;
    steps<float, float>(s, b, tensors, n, SWARP_F32, SWARP_F32, st);
    steps<bf16, bf16>(s, b, tensors, n, SWARP_BF16, SWARP_BF16, st);
    steps<bf16, float>(s, b, tensors, n, SWARP_BF16, SWARP_F32, st);
    steps<f16, f16>(s, b, tensors, n, SWARP_F16, SWARP_F16, st);
    steps<f16, float>(s, b, tensors, n, SWARP_F16, SWARP_F32, st);
    return launched();
}

int swarp_adamw_unpack(const swarp_adamw_t *a, float *avg, float *sq, void *stream)
{
    swarp::set_error("");
    if (check(a)) return -1;
    if (a->bits != 8) return fail("only 8-bit moments are unpacked");
    if (a->state_len == 0) return 0;
    if (!avg || !sq) return fail("pointer arguments must be set");
    if (((uintptr_t)avg | (uintptr_t)sq) & 15u) return fail("avg and sq must be 16-byte aligned");
    const int64_t groups = a->state_len / GROUP;
    hipLaunchKernelGGL(k_unpack, dim3((unsigned)(groups < 65536 ? (groups + 3) / 4 : 16384)), dim3(BLOCK), 0,
                       (hipStream_t)stream, groups, (const uint8_t *)a->exp_avg,
                       (const uint8_t *)a->exp_avg_sq, (const uint8_t *)a->avg_base,
                       (const uint8_t *)a->sq_base, avg, sq);
    return launched();
}

int swarp_grad_norm(const swarp_tensor_t *tensors, int32_t n_tensors, double max_norm,
                    float *norm_scale, void *work, void *stream)
{
    swarp::set_error("");
    if (check(tensors, n_tensors)) return -1;
    if (!norm_scale || !work || (uintptr_t)work & 15u) return fail("norm_scale and aligned work must be set");
    hipStream_t st = (hipStream_t)stream;
    double *const sums = (double *)work;
    Tensors t;
    uint32_t chunks;
    int blocks = 0;  // sums set so far: a launch adds to those and sets the others of its grid
    for (int d : {SWARP_F32, SWARP_BF16, SWARP_F16})
        for (int k = 0; k < n_tensors;) {
            k = fill(t, chunks, tensors, n_tensors, k, 0x7fffffffu, [&](const swarp_tensor_t &y) { return y.grad_dtype == d; });
            if (!t.count) continue;
            const int grid = (int)(chunks < NORM_BLOCKS ? chunks : NORM_BLOCKS);
            const dim3 g(grid), b(BLOCK);
            if (d == SWARP_F32) hipLaunchKernelGGL((k_norm<float>), g, b, 0, st, t, chunks, sums, blocks);
            else if (d == SWARP_BF16) hipLaunchKernelGGL((k_norm<bf16>), g, b, 0, st, t, chunks, sums, blocks);
            else hipLaunchKernelGGL((k_norm<f16>), g, b, 0, st, t, chunks, sums, blocks);
            blocks = grid > blocks ? grid : blocks;
        }
    hipLaunchKernelGGL(k_norm_finish, dim3(1), dim3(BLOCK), 0, st, blocks, (const double *)sums,
                       (float)max_norm, norm_scale);
    return launched();
}

}  // extern "C"
