// gae.hip -- generalised advantage estimation and its adjoint (swarp_gae_fwd / _bwd).
//
//   A_t = d_t + c_t A_{t+1},  d_t = r_t + gamma n_t - V_t,  c_t = 0 at an episode's end, else
//   gamma lam;  G_t = (gA_t + gR_t) + c_{t-1} G_{t-1} is the adjoint of d_t.
//
// Both are first-order recurrences, run over tiles: a stretch of SEG steps is one thread's, held in
// registers; every thread forms the value its stretch ends in with nothing carried in, and the
// product of its factors; a scan of those pairs gives each thread what is carried into it, and a
// tile what it hands to the next.  So each array is read once and written once whatever the
// lengths, and a long axis is spread over a workgroup where there are few columns.
//   Time first: a wave has 64 neighbouring columns, its rows of 64 are whole lines; the workgroup's
//   1 to 16 waves have consecutive stretches, joined through LDS.  16 waves where the columns do
//   not fill the card by themselves, fewer where there are fewer steps.
//   Time last: the threads of a wave (of 1 to 4, by the length) have consecutive stretches of one
//   column, joined by a scan over the lanes; a column's arrays are read in spans of SEG steps,
//   which start anywhere (a column of values is one longer than one of rewards).
// What bounds it: many columns, memory: 32 x 16000 x 16 float32 in 24 us, 132 MB at 5.5 TB/s (a
// thread that walks its column alone: 52 us), its adjoint in 30; half as many columns of float64 in
// 26 and 27.  Few, the latency of two tiles' loads and scans: 96 columns of 4095 steps in 10 us,
// their adjoint in 10 (alone: 3 ms each), 13 and 12 in float64.
#include "learn.hpp"

namespace {

using namespace learn;

template <typename T> struct Args {
    int64_t steps, columns, group;
    T gamma, carry, carries;  // gamma, gamma * lam, the product of a stretch's SEG such factors
    const T *r, *v, *fin;
    const uint8_t *term, *trunc;
    T *adv, *ret;
    const T *g_adv, *g_ret;
    T *d_r, *d_v, *d_fin;
    int has_fin;
};

// x -> a + c x, and one such map after another.  An end of an episode is a factor of -0, which
// stops NaN and infinities too; every other factor is +0 (lam = 0) or above, and a product of such
// ones that would underflow is held at the smallest number, so that what is not finite reaches
// as far through a scan as it does step by step.
template <typename T> struct Map {
    T a, c;
};
__device__ __forceinline__ bool ends(float c) { return (uint32_t)__float_as_int(c) == 0x80000000u; }
__device__ __forceinline__ bool ends(double c) { return (uint64_t)__double_as_longlong(c) == (uint64_t)1 << 63; }
constexpr float least(float) { return 0x1p-149f; }
constexpr double least(double) { return 0x1p-1074; }
template <typename T> __host__ __device__ __forceinline__ T product(T f, T c)
{
    return f > T(0) && c > T(0) && !(f * c > T(0)) ? least(T(0)) : f * c;
}
template <typename T> __device__ __forceinline__ Map<T> after(const Map<T> &f, const Map<T> &first)
{
    return {ends(f.c) ? f.a : f.a + f.c * first.a, ends(f.c) ? f.c : product(f.c, first.c)};
}
template <typename T> __device__ __forceinline__ T apply(const Map<T> &f, T x)
{
    return ends(f.c) ? f.a : f.a + f.c * x;
}

constexpr int SEG = 8;       // steps of a stretch
constexpr int MOST_WAVES = 16;
constexpr int ROWS_BLOCK = 256;

template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Span {
    T e[N];
};

// A stretch of steps t0 .. t0 + SEG - 1 of one column.  One that reaches past the first or the last
// step is the last in the recurrence's order: nothing is done with its map, and of its steps out
// there nothing is stored.  q: two bits a step, terminated and truncated.
template <typename T> struct Stretch {
    T x[SEG], y[SEG + 1];
    uint32_t q;

    __device__ __forceinline__ T factor(const Args<T> &a) const { return q & (1u << 2 * SEG) - 1u ? T(-0.0) : a.carries; }
    // Advantages: x holds the rewards, y the values; leaves x the d_t.
    template <typename Fin> __device__ __forceinline__ Map<T> rewards(const Args<T> &a, int64_t t0, Fin fin)
    {
        T A = T(0);
#pragma unroll
        for (int k = SEG - 1; k >= 0; --k) {
            const uint32_t e = q >> 2 * k & 3u;
            T next = y[k + 1];
            if (a.has_fin && e == 2u && t0 + k >= 0) next = fin(k);
            x[k] = x[k] + (e & 1u ? T(0) : a.gamma * next) - y[k];
            A = e ? x[k] : x[k] + a.carry * A;
        }
        return {A, factor(a)};
    }
    // ... and with A of the step behind carried in, x the advantages, y the returns.
    __device__ __forceinline__ void advantages(const Args<T> &a, T in)
    {
#pragma unroll
        for (int k = SEG - 1; k >= 0; --k) {
            in = q >> 2 * k & 3u ? x[k] : x[k] + a.carry * in;
            x[k] = in;
            y[k] += in;
        }
    }
    // The adjoint: x holds gA, y gR (both 0 past the end); q begins one step earlier.
    __device__ __forceinline__ Map<T> adjoints(const Args<T> &a)
    {
        T G = T(0);
#pragma unroll
        for (int k = 0; k < SEG; ++k) {
            x[k] += y[k];
            G = q >> 2 * k & 3u ? x[k] : x[k] + a.carry * G;
        }
        return {G, factor(a)};
    }
    // ... and with G of the step before carried in, x the adjoints of the rewards, y those of the
    // values (of step L, too, where the stretch reaches it), z those of the final values.
    __device__ __forceinline__ void slopes(const Args<T> &a, int64_t t0, T in, T (&z)[SEG])
    {
#pragma unroll
        for (int k = 0; k <= SEG; ++k) {
            const uint32_t e = q >> 2 * k & 3u;
            const T into = t0 + k == 0 || (e & 1u) || (e == 2u && a.has_fin) ? T(0) : a.gamma * in;
            if (k == SEG) {
                y[k] = into;
                break;
            }
            const T G = e ? x[k] : x[k] + a.carry * in;
            x[k] = G;
            y[k] = t0 + k < a.steps ? y[k] - G + into : into;
            z[k] = (q >> 2 * (k + 1) & 3u) == 2u ? a.gamma * G : T(0);
            in = G;
        }
    }
};

// ------------------------------------------------------------------------------ time first

// Joins the stretches of the workgroup's waves: `in` is what is carried into the thread's own,
// `carry` what the tile hands on.  Wave 0 is the first in the recurrence's order.
template <typename T>
__device__ __forceinline__ void join_waves(const Map<T> &m, Map<T> (*maps)[64], T &carry, T &in)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    in = carry;
    if (waves == 1) {
        carry = apply(m, carry);
        return;
    }
    __syncthreads();
    maps[wave][lane] = m;
    __syncthreads();
    for (int w = 0; w < waves; ++w) {
        if (w == wave) in = carry;
        carry = apply(maps[w][lane], carry);
    }
}

template <typename T> __global__ __launch_bounds__(64 * MOST_WAVES) void k_gae_fwd_time(const Args<T> a)
{
    __shared__ Map<T> maps[MOST_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int64_t N = a.columns, F = N / a.group;
    const int64_t n = (int64_t)blockIdx.x * 64 + lane < N ? (int64_t)blockIdx.x * 64 + lane : N - 1;
    const bool mine = (int64_t)blockIdx.x * 64 + lane < N;  // (the others repeat the last column)
    const int64_t f = n / a.group;
    T carry = 0, in;
    for (int64_t end = a.steps; end > 0; end -= (int64_t)waves * SEG) {
        const int64_t t0 = end - (int64_t)(wave + 1) * SEG;  // (may lie before the first step)
        Stretch<T> s;
        s.q = 0;
        Map<T> m = {T(0), T(1)};
        if (t0 > -SEG) {
            // steps before the first read its place and do nothing
            uint8_t te[SEG] = {}, tr[SEG] = {};
#pragma unroll
            for (int k = 0; k < SEG; ++k) s.x[k] = a.r[(t0 + k < 0 ? 0 : t0 + k) * N + n];
#pragma unroll
            for (int k = 0; k <= SEG; ++k) s.y[k] = a.v[(t0 + k < 0 ? 0 : t0 + k) * N + n];
            if (a.term) {
#pragma unroll
                for (int k = 0; k < SEG; ++k) te[k] = a.term[(t0 + k < 0 ? 0 : t0 + k) * F + f];
            }
            if (a.trunc) {
#pragma unroll
                for (int k = 0; k < SEG; ++k) tr[k] = a.trunc[(t0 + k < 0 ? 0 : t0 + k) * F + f];
            }
#pragma unroll
            for (int k = 0; k < SEG; ++k) s.q |= (uint32_t)((te[k] ? 1 : 0) | (tr[k] ? 2 : 0)) << 2 * k;
            m = s.rewards(a, t0, [&](int k) { return a.fin[(t0 + k) * N + n]; });
        }
        join_waves(m, maps, carry, in);
        if (t0 > -SEG) {
            s.advantages(a, in);
#pragma unroll
            for (int k = 0; k < SEG; ++k)
                if (mine && t0 + k >= 0) {
                    a.adv[(t0 + k) * N + n] = s.x[k];
                    a.ret[(t0 + k) * N + n] = s.y[k];
                }
        }
    }
}

template <typename T> __global__ __launch_bounds__(64 * MOST_WAVES) void k_gae_bwd_time(const Args<T> a)
{
    __shared__ Map<T> maps[MOST_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int64_t L = a.steps, N = a.columns, F = N / a.group;
    const int64_t n = (int64_t)blockIdx.x * 64 + lane < N ? (int64_t)blockIdx.x * 64 + lane : N - 1;
    const bool mine = (int64_t)blockIdx.x * 64 + lane < N;
    const int64_t f = n / a.group;
    if (L == 0 && mine && wave == 0 && a.d_v) a.d_v[n] = T(0);
    T carry = 0, in;
    for (int64_t start = 0; start < L; start += (int64_t)waves * SEG) {
        const int64_t t0 = start + (int64_t)wave * SEG;
        Stretch<T> s;
        Map<T> m = {T(0), T(1)};
        if (t0 < L) {
            uint8_t te[SEG + 1] = {}, tr[SEG + 1] = {};
#pragma unroll
            for (int k = 0; k < SEG; ++k) s.x[k] = s.y[k] = T(0);
            if (a.g_adv) {
#pragma unroll
                for (int k = 0; k < SEG; ++k) s.x[k] = a.g_adv[(t0 + k < L ? t0 + k : L - 1) * N + n];
            }
            if (a.g_ret) {
#pragma unroll
                for (int k = 0; k < SEG; ++k) s.y[k] = a.g_ret[(t0 + k < L ? t0 + k : L - 1) * N + n];
            }
            if (a.term) {
#pragma unroll
                for (int k = 0; k <= SEG; ++k) te[k] = a.term[(t0 + k - 1 < 0 ? 0 : t0 + k - 1 < L ? t0 + k - 1 : L - 1) * F + f];
            }
            if (a.trunc) {
#pragma unroll
                for (int k = 0; k <= SEG; ++k) tr[k] = a.trunc[(t0 + k - 1 < 0 ? 0 : t0 + k - 1 < L ? t0 + k - 1 : L - 1) * F + f];
            }
            s.q = 0;
#pragma unroll
            for (int k = 0; k <= SEG; ++k) s.q |= (uint32_t)((te[k] ? 1 : 0) | (tr[k] ? 2 : 0)) << 2 * k;
            if (t0 == 0) s.q |= 1u;  // (nothing comes before the first step)
            m = s.adjoints(a);
        }
        join_waves(m, maps, carry, in);
        if (t0 < L && mine) {
            T z[SEG];
            s.slopes(a, t0, in, z);
#pragma unroll
            for (int k = 0; k < SEG; ++k)
                if (t0 + k < L) {
                    if (a.d_r) a.d_r[(t0 + k) * N + n] = s.x[k];
                    if (a.d_v) a.d_v[(t0 + k) * N + n] = s.y[k];
                    if (a.d_fin) a.d_fin[(t0 + k) * N + n] = z[k];
                }
#pragma unroll
            for (int k = 1; k <= SEG; ++k)
                if (t0 + k == L && a.d_v) a.d_v[L * N + n] = s.y[k];
        }
    }
}

// ------------------------------------------------------------------------------- time last

// Joins the stretches of the `per` threads (a power of two up to ROWS_BLOCK) of a column; thread 0
// of them is the first in the recurrence's order.
template <typename T>
__device__ __forceinline__ void join_lanes(Map<T> m, int per, Map<T> *totals, T &carry, T &in)
{
    const int lanes = per < 64 ? per : 64, lane = threadIdx.x % lanes;
    for (int d = 1; d < lanes; d <<= 1) {
        const Map<T> p = {__shfl_up(m.a, d, lanes), __shfl_up(m.c, d, lanes)};
        if (lane >= d) m = after(m, p);
    }
    const Map<T> all = {__shfl(m.a, lanes - 1, lanes), __shfl(m.c, lanes - 1, lanes)};
    Map<T> mine = {__shfl_up(m.a, 1, lanes), __shfl_up(m.c, 1, lanes)};
    if (lane == 0) mine = {T(0), T(1)};
    T before = carry;
    if (per > 64) {
        const int wave = threadIdx.x >> 6, first = wave / (per / 64) * (per / 64);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) totals[wave] = all;
        __syncthreads();
        for (int w = 0; w < per / 64; ++w) {
            if (first + w == wave) before = carry;
            carry = apply(totals[first + w], carry);
        }
    } else {
        carry = apply(all, carry);
    }
    in = apply(mine, before);
}

// Elements lo .. SEG - 1 or 0 .. hi - 1 of a span: whole where it can be.
template <typename T, int N>
__device__ __forceinline__ void get(T (&x)[N], const T *p, int lo, int hi)
{
    if (lo <= 0 && hi >= N) {
        const Span<T, N> y = *(const Span<T, N> *)p;
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = y.e[k];
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = k >= lo && k < hi ? p[k] : T(0);
    }
}
template <typename T, int M>
__device__ __forceinline__ void put(const T (&x)[M], T *p, int lo, int hi)
{
    if (lo <= 0 && hi >= SEG) {
        Span<T, SEG> y;
#pragma unroll
        for (int k = 0; k < SEG; ++k) y.e[k] = x[k];
        *(Span<T, SEG> *)p = y;
    } else {
#pragma unroll
        for (int k = 0; k < SEG; ++k)
            if (k >= lo && k < hi) p[k] = x[k];
    }
}

template <typename T>
__global__ __launch_bounds__(ROWS_BLOCK) void k_gae_fwd_rows(const Args<T> a, int per)
{
    __shared__ Map<T> totals[ROWS_BLOCK / 64];
    const int64_t L = a.steps, n0 = ((int64_t)blockIdx.x * ROWS_BLOCK + threadIdx.x) / per;
    const bool mine = n0 < a.columns;
    const int64_t n = mine ? n0 : a.columns - 1, f = n / a.group;
    const int p = threadIdx.x % per;
    T carry = 0, in;
    for (int64_t end = L; end > 0; end -= (int64_t)per * SEG) {
        const int64_t t0 = end - (int64_t)(p + 1) * SEG;
        const bool some = mine && t0 > -SEG;
        const int lo = t0 < 0 ? (int)-t0 : 0;
        Stretch<T> s;
        Map<T> m = {T(0), T(1)};
        if (some) {
            uint8_t te[SEG] = {}, tr[SEG] = {};
            get(s.x, a.r + n * L + t0, lo, SEG);
            get(s.y, a.v + n * (L + 1) + t0, lo, SEG + 1);
            if (a.term) get(te, a.term + f * L + t0, lo, SEG);
            if (a.trunc) get(tr, a.trunc + f * L + t0, lo, SEG);
            s.q = 0;
#pragma unroll
            for (int k = 0; k < SEG; ++k) s.q |= (uint32_t)((te[k] ? 1 : 0) | (tr[k] ? 2 : 0)) << 2 * k;
            m = s.rewards(a, t0, [&](int k) { return a.fin[n * L + t0 + k]; });
        }
        join_lanes(m, per, totals, carry, in);
        if (some) {
            s.advantages(a, in);
            put(s.x, a.adv + n * L + t0, lo, SEG);
            put(s.y, a.ret + n * L + t0, lo, SEG);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(ROWS_BLOCK) void k_gae_bwd_rows(const Args<T> a, int per)
{
    __shared__ Map<T> totals[ROWS_BLOCK / 64];
    const int64_t L = a.steps, n0 = ((int64_t)blockIdx.x * ROWS_BLOCK + threadIdx.x) / per;
    const bool mine = n0 < a.columns;
    const int64_t n = mine ? n0 : a.columns - 1, f = n / a.group;
    const int p = threadIdx.x % per;
    if (L == 0 && mine && p == 0 && a.d_v) a.d_v[n] = T(0);
    T carry = 0, in;
    for (int64_t start = 0; start < L; start += (int64_t)per * SEG) {
        const int64_t t0 = start + (int64_t)p * SEG;
        const bool some = mine && t0 < L;
        const int hi = L - t0 < SEG ? (int)(L - t0) : SEG;
        Stretch<T> s;
        Map<T> m = {T(0), T(1)};
        if (some) {
            uint8_t te[SEG] = {}, tr[SEG] = {};
            T gr[SEG] = {};
#pragma unroll
            for (int k = 0; k < SEG; ++k) s.x[k] = T(0);
            if (a.g_adv) get(s.x, a.g_adv + n * L + t0, 0, hi);
            if (a.g_ret) get(gr, a.g_ret + n * L + t0, 0, hi);
            if (a.term) get(te, a.term + f * L + t0, 0, hi);
            if (a.trunc) get(tr, a.trunc + f * L + t0, 0, hi);
            const int64_t j = f * L + t0 - 1;
            s.q = t0 == 0 ? 1u : (uint32_t)((a.term && a.term[j] ? 1 : 0) | (a.trunc && a.trunc[j] ? 2 : 0));
#pragma unroll
            for (int k = 0; k < SEG; ++k) {
                s.q |= (uint32_t)((te[k] ? 1 : 0) | (tr[k] ? 2 : 0)) << 2 * (k + 1);
                s.y[k] = gr[k];
            }
            m = s.adjoints(a);
        }
        join_lanes(m, per, totals, carry, in);
        if (some) {
            T z[SEG];
            s.slopes(a, t0, in, z);
            if (a.d_r) put(s.x, a.d_r + n * L + t0, 0, hi);
            if (a.d_v) {
                put(s.y, a.d_v + n * (L + 1) + t0, 0, hi);
                if (t0 + hi == L) {
#pragma unroll
                    for (int k = 1; k <= SEG; ++k)
                        if (k == hi) a.d_v[n * (L + 1) + L] = s.y[k];
                }
            }
            if (a.d_fin) put(z, a.d_fin + n * L + t0, 0, hi);
        }
    }
}

// ------------------------------------------------------------------------------- host side

template <typename T> Args<T> args_of(const swarp_gae_t *a)
{
    Args<T> k;
    k.steps = a->steps;
    k.columns = a->columns;
    k.group = a->group;
    k.gamma = (T)a->gamma;
    k.carry = (T)(a->gamma * a->lam) + T(0);  // (no -0)
    k.carries = k.carry;
    for (int i = 1; i < SEG; ++i) k.carries = product(k.carries, k.carry);
    k.r = (const T *)a->rewards;
    k.v = (const T *)a->values;
    k.fin = (const T *)a->final_values;
    k.has_fin = a->final_values != nullptr;
    k.term = a->terminated;
    k.trunc = a->truncated;
    k.adv = (T *)a->advantages;
    k.ret = (T *)a->returns;
    k.g_adv = (const T *)a->adj_advantages;
    k.g_ret = (const T *)a->adj_returns;
    k.d_r = (T *)a->adj_rewards;
    k.d_v = (T *)a->adj_values;
    k.d_fin = (T *)a->adj_final_values;
    return k;
}

int check(const swarp_gae_t *a)
{
    swarp::set_error("");
    if (!a) return fail("arguments must be set");
    if (a->dtype != SWARP_F32 && a->dtype != SWARP_F64) return fail("dtype must be SWARP_F32 or SWARP_F64");
    if (a->steps < 0 || a->columns < 0 || a->group < 1 || a->columns % a->group)
        return fail("bad sizes");
    if (a->columns > (int64_t)1 << 30) return fail("at most 2^30 columns");
    return 0;
}

// Waves of a workgroup of 64 columns: as many stretches as there are, while the columns alone
// leave the card's 256 compute units short of 16 waves each.
int waves_of(int64_t steps, int64_t columns)
{
    const int64_t groups = (columns + 63) / 64, stretches = (steps + SEG - 1) / SEG;
    int waves = 1;
    while (waves < MOST_WAVES && waves < stretches && groups * waves < 256 * 16) waves *= 2;
    return waves;
}
// Threads of a column whose steps lie next to each other.
int threads_of(int64_t steps)
{
    int per = 1;
    while (per < ROWS_BLOCK && (int64_t)per * SEG < steps) per *= 2;
    return per;
}

template <typename T> void run(const swarp_gae_t *a, bool back, hipStream_t st)
{
    const Args<T> k = args_of<T>(a);
    if (a->rows) {
        const int per = threads_of(a->steps);
        const dim3 g((unsigned)((a->columns * per + ROWS_BLOCK - 1) / ROWS_BLOCK)), b(ROWS_BLOCK);
        if (back) hipLaunchKernelGGL((k_gae_bwd_rows<T>), g, b, 0, st, k, per);
        else hipLaunchKernelGGL((k_gae_fwd_rows<T>), g, b, 0, st, k, per);
    } else {
        const dim3 g((unsigned)((a->columns + 63) / 64)), b(64 * waves_of(a->steps, a->columns));
        if (back) hipLaunchKernelGGL((k_gae_bwd_time<T>), g, b, 0, st, k);
        else hipLaunchKernelGGL((k_gae_fwd_time<T>), g, b, 0, st, k);
    }
}

}  // namespace

extern "C" {

int swarp_gae_fwd(const swarp_gae_t *a, void *stream)
{
    if (check(a)) return -1;
    if (a->steps == 0 || a->columns == 0) return 0;
    if (!a->rewards || !a->values || !a->advantages || !a->returns)
        return fail("pointer arguments must be set");
    if (a->dtype == SWARP_F32) run<float>(a, false, (hipStream_t)stream);
    else run<double>(a, false, (hipStream_t)stream);
    return launched();
}

int swarp_gae_bwd(const swarp_gae_t *a, void *stream)
{
    if (check(a)) return -1;
    if (a->columns == 0) return 0;
    if (a->adj_final_values && !a->final_values)
        return fail("adj_final_values without final_values");
    if (a->dtype == SWARP_F32) run<float>(a, true, (hipStream_t)stream);
    else run<double>(a, true, (hipStream_t)stream);
    return launched();
}

}  // extern "C"
