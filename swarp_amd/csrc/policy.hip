// policy.hip -- the clipped policy loss with KL and entropy terms, and its gradient
// (swarp_categorical_loss, swarp_gaussian_loss).
//
// Per decision, with lp the log-probability of its action and e = q - lp:
//   l = -min(rho A, clamp(rho) A) + kl_coef (exp(e) - 1 - e) - entropy_coef H
//   g = dl/dlp = -(rho A where the unclipped branch is the smaller) - kl_coef (exp(e) - 1)
// Categorical: p = softmax(x), dl/dx_j = g (1[j = a] - p_j) + entropy_coef p_j (log p_j + H).
// Gaussian: z = (a - mu) / sigma, dl/dmu = g z / sigma, dl/dls = g (z^2 - 1) - entropy_coef.
//
// A call is the mask's count, where there is a mask (its sums are needed before any gradient can
// be written), the rows' kernel (two where rows are split), and one workgroup that joins the
// sums.  Every sum has a fixed order.  The backward of a call whose gradients were left by the
// forward is a launch of the rows' kernel that reads the upstream gradient and ends.
#include <math.h>

#include "learn.hpp"

namespace {

using namespace learn;

constexpr int BLOCK = 256;
constexpr int MOST_BLOCKS = 2048;   // of a loss kernel: each leaves one row of sums
constexpr int COUNTERS = 256;       // blocks that count the mask
constexpr int MOST_DIMS = 64;       // of a Gaussian head
constexpr int FEW_ROWS = 256;       // fewer rows than compute units: long ones are split
constexpr double HALF_LOG_2PI = 0.91893853320467274178;

template <typename A> struct Row {  // what every decision has, and the loss's constants
    int64_t rows;
    A lo, hi, klc, entc;
    const A *old, *adv, *ref;
    const uint8_t *mask;
    A *logp;
    double *sums;        // [grid][4]: loss, entropy, kl, clipped
    double *std_sums;    // [grid][width]
    const int32_t *counts;  // [n_counts] of the mask
    int n_counts, sum, skip_unit;
    const A *scale;
};

// Decisions that count, at least 1: the same in every thread of the block.
template <typename A> __device__ double counted(const Row<A> &r)
{
    if (!r.mask) return r.rows > 1 ? (double)r.rows : 1.0;
    __shared__ double count;
    if (threadIdx.x < 64) {
        int64_t c = 0;
        for (int i = threadIdx.x; i < r.n_counts; i += 64) c += r.counts[i];
        c = wave_sum(c);
        if (threadIdx.x == 0) count = c > 1 ? (double)c : 1.0;
    }
    __syncthreads();
    return count;
}
// Weight of a decision in the gradient.
template <typename A> __device__ A weight_of(const Row<A> &r) { return r.sum ? A(1) : (A)(1.0 / counted(r)); }

template <typename A> struct Terms {
    A loss, ent, kl, clipped;
};

// exp and log of the accumulation types.  float: the hardware's base-2 functions, whose error is
// an ulp of the result; arguments are differences of a few units, which the product with log2(e)
// rounds by half an ulp more.
constexpr float LOG2E = 1.44269504088896340736f;
constexpr double LN_2 = 0.69314718055994530942;
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// expm1(e) - e, without the cancellation of small e (below 1/2 the series to e^9 / 9! in float, to
// e^15 / 15! in double: the next term is below a tenth of the last digit) and without inf - inf
// where the action taken has no probability left (beside e^80, e is nothing).
template <typename A> __device__ __forceinline__ A kl_of(A e)
{
    if (e > A(80)) return exp_of(e);
    A s = A(1) / A(362880);
    if constexpr (sizeof(A) == 8) {
        s = A(1) / A(1307674368000);
        s = s * e + A(1) / A(87178291200);
        s = s * e + A(1) / A(6227020800);
        s = s * e + A(1) / A(479001600);
        s = s * e + A(1) / A(39916800);
        s = s * e + A(1) / A(3628800);
        s = s * e + A(1) / A(362880);
    }
    s = s * e + A(1) / A(40320);
    s = s * e + A(1) / A(5040);
    s = s * e + A(1) / A(720);
    s = s * e + A(1) / A(120);
    s = s * e + A(1) / A(24);
    s = s * e + A(1) / A(6);
    s = s * e + A(0.5);
    const bool small = e < A(0.5) && e > A(-0.5);
    return small ? s * e * e : (sizeof(A) == 4 ? exp_of(e) - A(1) - e : (A)(expm1((double)e) - (double)e));
}

// One decision's terms added to `t`; returns g.  lp may be wider than A: its differences to the
// old and the reference log-probability are then rounded once.
template <typename A, typename L>
__device__ __forceinline__ A decide(const Row<A> &r, int64_t i, L lp, A H, Terms<A> &t)
{
    const A old = r.old[i], adv = r.adv[i];
    const A rho = exp_of((A)(lp - (L)old));
    const A bounded = rho < r.lo ? r.lo : (rho > r.hi ? r.hi : rho);
    const A first = rho * adv, second = bounded * adv;
    const bool clipped = second < first;
    const A e = (A)((L)(r.ref ? r.ref[i] : old) - lp);
    const A kl = kl_of(e);
    A l = clipped ? -second : -first;
    A g = clipped ? A(0) : -first;
    if (r.klc != A(0)) {
        l += r.klc * kl;
        // (exp(e) - 1; a reference that forbids the action makes kl infinite, this -1)
        g -= r.klc * (e < A(-80) ? A(-1) : kl + e);
    }
    if (r.entc != A(0)) l -= r.entc * H;
    t.loss += l;
    t.ent += H;
    t.kl += kl;
    t.clipped += clipped ? A(1) : A(0);
    return g;
}

// The block's sums of its threads' terms to row blockIdx.x of `sums`.
template <int THREADS, typename A> __device__ void leave_sums(const Terms<A> &t, double *sums)
{
    __shared__ double red[THREADS / 64][4];
    const double v[4] = {(double)t.loss, (double)t.ent, (double)t.kl, (double)t.clipped};
    for (int k = 0; k < 4; ++k) {
        const double s = wave_sum(v[k]);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][k] = s;
    }
    __syncthreads();
    if (threadIdx.x < 4) {
        double s = 0;
        for (int w = 0; w < THREADS / 64; ++w) s += red[w][threadIdx.x];
        sums[4 * (int64_t)blockIdx.x + threadIdx.x] = s;
    }
}

__global__ __launch_bounds__(BLOCK) void k_count(int64_t rows, const uint8_t *mask, int32_t *counts)
{
    __shared__ int32_t red[BLOCK / 64];
    int32_t c = 0;
    for (int64_t i = (int64_t)blockIdx.x * BLOCK + threadIdx.x; i < rows; i += (int64_t)gridDim.x * BLOCK)
        c += mask[i] != 0;
    c = wave_sum(c);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < BLOCK / 64; ++w) c += red[w];
        counts[blockIdx.x] = c;
    }
}

// ------------------------------------------------------------------------ categorical head
//
// A row of logits is read once, held in registers as it came (of its own type) while its maximum,
// its sums and its gradient are formed, and the gradient is written once.  Work is in base 2: with
// m the maximum, z = (x - m) log2(e), s = sum 2^z, q = sum 2^z z:
//   log2 p = z - log2 s;  H = (log2 s - q / s) ln 2;  dl/dx = 2^z (c1 z + c2) + g [j = a],
//   c1 = entropy_coef ln 2 / s,  c2 = (entropy_coef (H - ln s) - g) / s.
// The difference comes first: logits at the type's lowest value neither overflow nor differ from
// each other.  z is held above a number that 2^z makes 0, in the products alone: 0 times -inf is
// no NaN, and a NaN logit still is one through 2^z.

struct Logits {
    int64_t inner, outer_stride, inner_stride;
    int width, actions32, flat;
    int splits, part;    // of a row that goes to several workgroups: parts, elements of one
    const void *x, *actions;
    void *d;
    void *parts;         // [rows][splits][3]: max, sum, q of a part
};

// VEC neighbouring elements, 16 bytes; rows start at any element.
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Span {
    T e[N];
};

// The same where they lie on 16 bytes (in LDS).
template <typename T, int N> struct __align__(16) Line {
    Span<T, N> s;
};

template <typename A> struct Base2;
template <> struct Base2<float> {
    static __device__ __forceinline__ float z(float x, float m) { return (x - m) * LOG2E; }
    static __device__ __forceinline__ float exp(float z) { return __builtin_amdgcn_exp2f(z); }
    static __device__ __forceinline__ float log(float s) { return __builtin_amdgcn_logf(s); }
    static __device__ __forceinline__ float floor(float z) { return fmaxf(z, -2000.0f); }
};
template <> struct Base2<double> {
    static constexpr double L = 1.44269504088896340736;
    static __device__ __forceinline__ double z(double x, double m) { return (x - m) * L; }
    static __device__ __forceinline__ double exp(double z) { return exp2(z); }
    static __device__ __forceinline__ double log(double s) { return log2(s); }
    static __device__ __forceinline__ double floor(double z) { return fmax(z, -2000.0); }
};

__device__ __forceinline__ int64_t start_of(const Logits &g, int64_t i)
{
    if (g.flat) return i * g.inner_stride;
    const uint64_t o = (uint64_t)i / (uint64_t)g.inner;
    return (int64_t)o * g.outer_stride + (i - (int64_t)o * g.inner) * g.inner_stride;
}
__device__ __forceinline__ int64_t action_of(const Logits &g, int64_t i)
{
    return g.actions32 ? (int64_t)((const int32_t *)g.actions)[i] : ((const int64_t *)g.actions)[i];
}

// What the gradient of a row needs; `at`: where its action lies, below 0 if nowhere (its terms are
// NaN then, and so are c2 and the row).
template <typename A> struct Slope {
    A m, c1, c2, gw;
    int64_t at;
};

// The row's terms from its sums; `lp` is its log-probability.
template <typename A>
__device__ __forceinline__ Slope<A> slope_of(const Row<A> &r, const Logits &g, int64_t i, A m, A s, A q,
                                             A xa, int64_t at, A w, Terms<A> &t, A &lp)
{
    typedef Base2<A> B;
    const bool in = at >= 0 && at < g.width;
    const A ls = B::log(s), inv = A(1) / s;
    const A H = (ls - q * inv) * A(LN_2);
    lp = in ? (xa - m) - ls * A(LN_2) : A(NAN);
    const A gw = decide(r, i, lp, in ? H : A(NAN), t) * w;
    const A ew = r.entc * w;
    return {m, ew * A(LN_2) * inv, (ew * (H - ls * A(LN_2)) - gw) * inv, gw, in ? at : -1};
}

// The larger of x and m; m where x is NaN.
template <typename A> __device__ __forceinline__ A max_of(A x, A m) { return x > m ? x : m; }
__device__ __forceinline__ float fma_of(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_of(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Elements of a 32-bit word (two words, for double) and back.
template <typename T> struct Words;
template <> struct Words<float> {
    static constexpr uint32_t LOW = 0xff800000u, LOW_HI = LOW;  // -inf
    static __device__ __forceinline__ float get(const uint32_t (&w)[4], int k) { return __int_as_float((int)w[k]); }
    static __device__ __forceinline__ void set(uint32_t (&w)[4], const float (&y)[4])
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = (uint32_t)__float_as_int(y[k]);
    }
};
template <> struct Words<double> {
    static constexpr uint32_t LOW = 0, LOW_HI = 0xfff00000u;
    static __device__ __forceinline__ double get(const uint32_t (&w)[4], int k)
    {
        return __longlong_as_double((long long)((uint64_t)w[2 * k + 1] << 32 | w[2 * k]));
    }
    static __device__ __forceinline__ void set(uint32_t (&w)[4], const double (&y)[2])
    {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint64_t b = (uint64_t)__double_as_longlong(y[k]);
            w[2 * k] = (uint32_t)b;
            w[2 * k + 1] = (uint32_t)(b >> 32);
        }
    }
};
template <> struct Words<bf16> {
    static constexpr uint32_t LOW = 0xff80ff80u, LOW_HI = LOW;
    static __device__ __forceinline__ float get(const uint32_t (&w)[4], int k)
    {
        return __int_as_float((int)(k & 1 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16));
    }
    static __device__ __forceinline__ void set(uint32_t (&w)[4], const float (&y)[8])
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __builtin_bit_cast(uint32_t, Span<bf16, 2>{{(bf16)y[2 * k], (bf16)y[2 * k + 1]}});
    }
};
template <> struct Words<f16> {
    static constexpr uint32_t LOW = 0xfc00fc00u, LOW_HI = LOW;
    static __device__ __forceinline__ float get(const uint32_t (&w)[4], int k)
    {
        return (float)__builtin_bit_cast(f16, (uint16_t)(w[k / 2] >> 16 * (k & 1)));
    }
    static __device__ __forceinline__ void set(uint32_t (&w)[4], const float (&y)[8])
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __builtin_bit_cast(uint32_t, Span<f16, 2>{{(f16)y[2 * k], (f16)y[2 * k + 1]}});
    }
};

// The largest of many elements, word by word.  16-bit ones by twos, as integers: the largest signed
// one is the answer if it is not negative; if all are negative, the smallest unsigned one is (the
// magnitudes are then in that order).
template <typename T> struct Most {
    typedef typename Acc<T>::type A;
    A m = -INFINITY;
    __device__ __forceinline__ void add(const uint32_t (&w)[4], int k)
    {
        if (k < (int)(16 / sizeof(T))) m = max_of(Words<T>::get(w, k), m);
    }
    __device__ __forceinline__ A value() const { return m; }
};
template <typename T> struct Most16 {
    typedef short I2 __attribute__((ext_vector_type(2)));
    typedef unsigned short U2 __attribute__((ext_vector_type(2)));
    I2 i = {-32768, -32768};
    U2 u = {65535, 65535};
    __device__ __forceinline__ void add(const uint32_t (&w)[4], int k)
    {
        i = __builtin_elementwise_max(i, __builtin_bit_cast(I2, w[k]));
        u = __builtin_elementwise_min(u, __builtin_bit_cast(U2, w[k]));
    }
    __device__ __forceinline__ float value() const
    {
        const short a = i.x > i.y ? i.x : i.y;
        const unsigned short b = u.x < u.y ? u.x : u.y;
        return (float)__builtin_bit_cast(T, (unsigned short)(a >= 0 ? (unsigned short)a : b));
    }
};
template <> struct Most<bf16> : Most16<bf16> {};
template <> struct Most<f16> : Most16<f16> {};

// LANES threads hold a row of at most LANES * E elements, E a multiple of VEC: thread `lane` the
// spans lane, lane + LANES, ..., as the words they came in (as elements they would take a register
// each).  The last, short span is read and written in pieces; its length is the same for every
// row, so only scalar branches choose them.
template <typename T, int LANES, int E> struct Held {
    typedef typename Acc<T>::type A;
    typedef Base2<A> B;
    static constexpr int VEC = 16 / sizeof(T), NV = E / VEC;
    // Few logits a thread: the compiler keeps what it has of one from one use to the next (as a
    // float, z, 2^z), which saves the second 2^z.  More would not fit the registers: there each use
    // starts from the words as they were loaded, which the compiler is not to see through, one
    // span after the other.  (200 M bfloat16 logits in rows of 1000, 32 a thread: kept 166 us, not
    // kept 188; float32 is the same to 2 %.)
    static constexpr bool KEEP = E <= (sizeof(T) == 2 ? 32 : 16);
    struct Raw {
        uint32_t w[4];
    };
    uint32_t v[NV][4];
    int spans;  // of the row

    // Whether any thread has a span i: the same for the whole workgroup, so that what a row leaves
    // empty costs nothing.
    __device__ __forceinline__ bool used(int i) const { return KEEP || i * LANES < spans; }

    __device__ __forceinline__ void fill(uint32_t lo, uint32_t hi)
    {
        spans = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i][0] = v[i][2] = lo;
            v[i][1] = v[i][3] = hi;
        }
    }
    __device__ __forceinline__ void take(int i, const Raw &y)
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[i][k] = y.w[k];
    }
    __device__ __forceinline__ Raw give(int i) const { return Raw{{v[i][0], v[i][1], v[i][2], v[i][3]}}; }

    template <int N> static __device__ __forceinline__ Raw piece(const T *x)
    {
        Span<T, VEC> d;
#pragma unroll
        for (int k = 0; k < VEC; ++k) d.e[k] = (T)(-INFINITY);
        const Span<T, N> y = *(const Span<T, N> *)x;
#pragma unroll
        for (int k = 0; k < N; ++k) d.e[k] = y.e[k];
        return __builtin_bit_cast(Raw, d);
    }
    template <int N> __device__ __forceinline__ void piece_out(int i, T *x) const
    {
        const Span<T, VEC> s = __builtin_bit_cast(Span<T, VEC>, give(i));
        Span<T, N> y;
#pragma unroll
        for (int k = 0; k < N; ++k) y.e[k] = s.e[k];
        *(Span<T, N> *)x = y;
    }

    // A thread without a span of its own reads the row's first, so that every load is in flight at
    // once and into its own registers.  The row has a whole span: all but a double's of one element
    // are wider (33 logits and up of the smaller types; parts are cut so).
    __device__ __forceinline__ void load(const T *x, int width, int lane)
    {
        // (the offsets are formed here, row by row, and not kept in registers from row to row)
        if constexpr (!KEEP) asm volatile("" : "+v"(lane));
        const int full = width / VEC, rem = width % VEC;
        spans = full + (rem != 0);
        Raw last = {{Words<T>::LOW, Words<T>::LOW_HI, Words<T>::LOW, Words<T>::LOW_HI}};
        if (rem && lane == full % LANES) {
            const T *const y = x + full * VEC;
            switch (rem) {
            case 1: last = piece<1>(y); break;
            case 2: if constexpr (VEC > 2) last = piece<2>(y); break;
            case 3: if constexpr (VEC > 2) last = piece<3>(y); break;
            case 4: if constexpr (VEC > 4) last = piece<4>(y); break;
            case 5: if constexpr (VEC > 4) last = piece<5>(y); break;
            case 6: if constexpr (VEC > 4) last = piece<6>(y); break;
            default: if constexpr (VEC > 4) last = piece<7>(y); break;
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t at = lane < full - i * LANES ? (uint32_t)(i * LANES + lane) * VEC : 0u;
            if (sizeof(T) < 8 || full > 0) take(i, __builtin_bit_cast(Raw, *(const Span<T, VEC> *)(x + at)));
            else take(i, last);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int left = full - i * LANES;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t low = k & 1 ? Words<T>::LOW_HI : Words<T>::LOW;
                v[i][k] = lane < left ? v[i][k] : (lane == left ? last.w[k] : low);
            }
        }
        forget();
    }
    __device__ __forceinline__ A most() const
    {
        // (a NaN may be passed over or come out: the sums hold it either way)
        Most<T> m;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!used(i)) break;
#pragma unroll
            for (int k = 0; k < 4; ++k) m.add(v[i], k);
            in_turn();
        }
        return m.value();
    }
    __device__ __forceinline__ void sums(A m, A &s, A &q)
    {
        forget();
        s = q = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!used(i)) break;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const A z = B::z(Words<T>::get(v[i], k), m), e = B::exp(z);
                s += e;
                q = fma_of(e, B::floor(z), q);
            }
            in_turn();
        }
    }
    __device__ __forceinline__ void forget()
    {
        if constexpr (!KEEP) {
#pragma unroll
            for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(v[i][0]), "+v"(v[i][1]), "+v"(v[i][2]), "+v"(v[i][3]));
        }
    }
    static __device__ __forceinline__ void in_turn()
    {
        if constexpr (!KEEP) __builtin_amdgcn_sched_barrier(0);
    }
    // The gradient row to d.
    __device__ __forceinline__ void slope(const Slope<A> &c, T *d, int width, int lane)
    {
        const int full = width / VEC, rem = width % VEC;
        forget();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!used(i)) break;
            A y[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const A z = B::z(Words<T>::get(v[i], k), c.m);
                y[k] = B::exp(z) * fma_of(c.c1, B::floor(z), c.c2);
            }
            if (c.at >= 0 && (int)c.at / VEC - i * LANES == lane) {
                const int at = (int)c.at % VEC;
#pragma unroll
                for (int k = 0; k < VEC; ++k) y[k] += k == at ? c.gw : A(0);
            }
            Words<T>::set(v[i], y);
            put(d, lane, i, full, rem);
            in_turn();
        }
    }
    __device__ __forceinline__ void zero(T *d, int width, int lane)
    {
        const int full = width / VEC, rem = width % VEC;
        fill(0, 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) put(d, lane, i, full, rem);
    }
    __device__ __forceinline__ void put(T *d, int lane, int i, int full, int rem) const
    {
        T *const y = d + i * LANES * VEC + (uint32_t)(lane * VEC);
        const int left = full - i * LANES;
        if (lane < left) *(Span<T, VEC> *)y = __builtin_bit_cast(Span<T, VEC>, give(i));
        if (rem && full / LANES == i && lane == left) {
            switch (rem) {
            case 1: piece_out<1>(i, y); break;
            case 2: if constexpr (VEC > 2) piece_out<2>(i, y); break;
            case 3: if constexpr (VEC > 2) piece_out<3>(i, y); break;
            case 4: if constexpr (VEC > 4) piece_out<4>(i, y); break;
            case 5: if constexpr (VEC > 4) piece_out<5>(i, y); break;
            case 6: if constexpr (VEC > 4) piece_out<6>(i, y); break;
            default: if constexpr (VEC > 4) piece_out<7>(i, y); break;
            }
        }
    }
};

// Sums and maxima over LANES neighbouring threads of a wave.
template <int LANES, typename A> __device__ __forceinline__ A lanes_sum(A v)
{
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
template <int LANES, typename A> __device__ __forceinline__ A lanes_max(A v)
{
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
        const A y = __shfl_xor(v, d, 64);
        v = y > v ? y : v;
    }
    return v;
}

template <typename A> __device__ __forceinline__ void add(Terms<A> &t, const Terms<A> &x)
{
    t.loss += x.loss;
    t.ent += x.ent;
    t.kl += x.kl;
    t.clipped += x.clipped;
}

// The upstream gradient, and whether there is nothing to do.
template <typename A> __device__ __forceinline__ bool upstream(const Row<A> &r, A &g)
{
    g = r.scale ? *r.scale : A(1);
    return r.scale && r.skip_unit && g == A(1);
}

// Rows of 33 to 2048 elements (a double's: of any number up to that): LANES threads of a wave a row.
// What bounds it: memory from rows of 250 on (800 MB of bfloat16 logits and gradients in 156 to
// 189 us, of float32 in 152 to 169); below, what each row costs beside its logits (rows of 50:
// 282 and 247 us).  16-bit rows are held to four waves a SIMD: 133 registers instead of 128 cost
// rows of 1000 16 us.  (Rows of 32 and 64 lanes pay 16 bytes of scratch a thread for that.)
template <typename T, int LANES, int E>
__global__ __launch_bounds__(BLOCK, sizeof(T) == 2 ? 4 : 1) void k_cat_lanes(const Row<typename Acc<T>::type> r, const Logits g)
{
    typedef typename Acc<T>::type A;
    A up1;
    if (upstream(r, up1)) return;
    const A w = weight_of(r) * up1;
    const int lane = threadIdx.x % LANES;
    constexpr int ROWS = BLOCK / LANES;
    Terms<A> t = {};
    for (int64_t i0 = (int64_t)blockIdx.x * ROWS; i0 < r.rows; i0 += (int64_t)gridDim.x * ROWS) {
        // (a wave's last rows may be past the end: its threads stay for the sums over lanes)
        const int64_t i = i0 + threadIdx.x / LANES < r.rows ? i0 + threadIdx.x / LANES : r.rows - 1;
        const bool mine = i0 + threadIdx.x / LANES < r.rows;
        const bool on = mine && (!r.mask || r.mask[i]);
        const T *const x = (const T *)g.x + start_of(g, i);
        const int64_t at = action_of(g, i);
        const bool in = at >= 0 && at < g.width;
        Held<T, LANES, E> h;
        if (on) h.load(x, g.width, lane);
        else h.fill(0, 0);
        const A xa = up(x[in ? at : 0]);
        const A m = lanes_max<LANES>(h.most());
        A s, q, lp;
        h.sums(m, s, q);
        s = lanes_sum<LANES>(s);
        q = lanes_sum<LANES>(q);
        if (!mine) continue;
        Terms<A> x1 = {};
        const Slope<A> c = slope_of(r, g, i, m, s, q, xa, at, w, x1, lp);
        if (lane == 0) {
            if (on) add(t, x1);
            if (r.logp) r.logp[i] = on ? lp : A(0);
        }
        if (!g.d) continue;
        T *const d = (T *)g.d + i * g.width;
        if (on) h.slope(c, d, g.width, lane);
        else h.zero(d, g.width, lane);
    }
    if (r.sums) leave_sums<BLOCK>(t, r.sums);
}

// Sum or maximum over a workgroup; `red` is used again only after another barrier.
template <int THREADS, typename A> __device__ __forceinline__ A block_max(A v, A *red)
{
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lanes_max<THREADS / 64>(red[threadIdx.x % (THREADS / 64)]);
    return v;
}
template <int THREADS, typename A> __device__ __forceinline__ void block_sums(A &s, A &q, A (*red)[2])
{
    s = wave_sum(s);
    q = wave_sum(q);
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6][0] = s;
        red[threadIdx.x >> 6][1] = q;
    }
    __syncthreads();
    s = lanes_sum<THREADS / 64>(red[threadIdx.x % (THREADS / 64)][0]);
    q = lanes_sum<THREADS / 64>(red[threadIdx.x % (THREADS / 64)][1]);
}

// Longer rows, up to THREADS * E elements: a workgroup a row.  Where a thread holds 256 bytes of
// logits the registers are limited to four waves a SIMD, so that two workgroups of 512 share a
// compute unit and one loads while the other computes: 8184 rows of 50001 bfloat16 logits in 412 us
// (1.64 GB, which a copy moves in 346; the vector units are busy 0.54 of the time, which the
// two overlap in part); as 1024 threads of 64 logits each, one workgroup a unit, 547 us.
template <typename T, int THREADS, int E>
__global__ __launch_bounds__(THREADS, sizeof(T) < 8 && E * sizeof(T) >= 256 ? 4 : 1) void k_cat_block(const Row<typename Acc<T>::type> r, const Logits g)
{
    typedef typename Acc<T>::type A;
    __shared__ A red_m[THREADS / 64], red_s[THREADS / 64][2];
    A up1;
    if (upstream(r, up1)) return;
    const A w = weight_of(r) * up1;
    const int lane = threadIdx.x;
    Terms<A> t = {};
    for (int64_t i = blockIdx.x; i < r.rows; i += gridDim.x) {
        T *const d = g.d ? (T *)g.d + i * g.width : nullptr;
        Held<T, THREADS, E> h;
        if (r.mask && !r.mask[i]) {
            if (r.logp && lane == 0) r.logp[i] = A(0);
            if (d) h.zero(d, g.width, lane);
            continue;
        }
        const T *const x = (const T *)g.x + start_of(g, i);
        const int64_t at = action_of(g, i);
        const bool in = at >= 0 && at < g.width;
        h.load(x, g.width, lane);
        const A xa = up(x[in ? at : 0]);
        // (each buffer's next use lies behind the other's barrier)
        const A m = block_max<THREADS>(h.most(), red_m);
        A s, q, lp;
        h.sums(m, s, q);
        block_sums<THREADS>(s, q, red_s);
        Terms<A> x1 = {};
        const Slope<A> c = slope_of(r, g, i, m, s, q, xa, at, w, x1, lp);
        if (lane == 0) {
            add(t, x1);
            if (r.logp) r.logp[i] = lp;
        }
        if (d) h.slope(c, d, g.width, lane);
    }
    if (r.sums) leave_sums<THREADS>(t, r.sums);
}

// Rows too long for a workgroup's registers, or too few of them to fill the card: parts of up to
// PART elements, a workgroup a part; first each part's maximum and sums, then every part of a row
// joins them and writes its share of the gradient (its second reading comes from the caches).
// What bounds it: memory, read twice: 100 M float32 logits in rows of 120000 take 101 us and, with
// the gradient, 174.  96 rows of 131072 (a workgroup a row would leave 160 of the 256 compute units
// idle) take 12 and 26 us.
constexpr int PART = 8192;

template <typename T>
__global__ __launch_bounds__(BLOCK) void k_cat_parts(const Row<typename Acc<T>::type> r, const Logits g)
{
    typedef typename Acc<T>::type A;
    __shared__ A red_m[BLOCK / 64], red_s[BLOCK / 64][2];
    A up1;
    if (upstream(r, up1)) return;
    const int64_t units = r.rows * g.splits;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t i = u / g.splits;
        const int part = (int)(u - i * g.splits), j = part * g.part;
        if (r.mask && !r.mask[i]) continue;
        const int n = g.width - j < g.part ? g.width - j : g.part;
        Held<T, BLOCK, PART / BLOCK> h;
        const T *const x = (const T *)g.x + start_of(g, i);
        h.load(x + j, n, threadIdx.x);
        const A m = block_max<BLOCK>(h.most(), red_m);
        A s, q;
        h.sums(m == A(-INFINITY) ? A(0) : m, s, q);  // (nothing open here: sums of 0)
        block_sums<BLOCK>(s, q, red_s);
        if (threadIdx.x == 0) {
            A *const p = (A *)g.parts + 3 * u;
            p[0] = m;
            p[1] = s;
            p[2] = q;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(BLOCK) void k_cat_join(const Row<typename Acc<T>::type> r, const Logits g)
{
    typedef typename Acc<T>::type A;
    typedef Base2<A> B;
    A up1;
    if (upstream(r, up1)) return;
    const A w = weight_of(r) * up1;
    const int64_t per = g.d ? g.splits : 1, units = r.rows * per;
    Terms<A> t = {};
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t i = u / per;
        const int part = (int)(u - i * per), j = part * g.part;
        const int n = g.width - j < g.part ? g.width - j : g.part;
        T *const d = g.d ? (T *)g.d + i * g.width + j : nullptr;
        Held<T, BLOCK, PART / BLOCK> h;
        if (r.mask && !r.mask[i]) {
            if (part == 0 && r.logp && threadIdx.x == 0) r.logp[i] = A(0);
            if (d) h.zero(d, n, threadIdx.x);
            continue;
        }
        const T *const x = (const T *)g.x + start_of(g, i);
        if (d) h.load(x + j, n, threadIdx.x);
        const int64_t at = action_of(g, i);
        const bool in = at >= 0 && at < g.width;
        const A xa = up(x[in ? at : 0]);
        const A *const p = (const A *)g.parts + 3 * i * g.splits;
        A m = -INFINITY, s = 0, q = 0;
        for (int k = 0; k < g.splits; ++k) m = p[3 * k] > m ? p[3 * k] : m;
        for (int k = 0; k < g.splits; ++k) {
            const A dm = B::z(p[3 * k], m), f = B::exp(dm);
            s += f * p[3 * k + 1];
            q += f * (p[3 * k + 2] + B::floor(dm) * p[3 * k + 1]);
        }
        Terms<A> x1 = {};
        A lp;
        Slope<A> c = slope_of(r, g, i, m, s, q, xa, at, w, x1, lp);
        if (part == 0 && threadIdx.x == 0) {
            add(t, x1);
            if (r.logp) r.logp[i] = lp;
        }
        if (!d) continue;
        if (in) c.at = at >= j && at < j + n ? at - j : PART;  // (PART: in another part)
        h.slope(c, d, n, threadIdx.x);
    }
    if (r.sums) leave_sums<BLOCK>(t, r.sums);
}

// A wave's LDS instructions are executed in their order: between its writes and the reads of other
// lanes only the compiler is to be held.
__device__ __forceinline__ void wave_lds()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Rows of N - 3 to N <= 32 elements, N a multiple of 4 (so that only the last three ask whether they
// are there): a thread a row.  A wave's rows lie next to each other in
// memory (where the caller's strides say so) and pass through LDS both ways, so that memory sees
// whole lines; a row's place there has an odd length, which spreads the threads over the banks.
// A wave has 64 rows of its own and waits for no other (with the workgroup's 256 rows between
// barriers 4.1 M rows of 25 bfloat16 logits took 139 us, now 130).
// What bounds it: those are 491 MB, which a copy moves in 104 us; the vector units are busy half the
// time, the rest is the chain load, LDS, row, LDS, store with four waves a SIMD.  Keeping 2^z or
// forming it again measured the same, fetching the next rows ahead took more registers than it gave.
template <typename T, int N>
__global__ __launch_bounds__(BLOCK) void k_cat_rows(const Row<typename Acc<T>::type> r, const Logits g)
{
    typedef typename Acc<T>::type A;
    typedef Base2<A> B;
    constexpr int VEC = 16 / sizeof(T);
    __align__(16) __shared__ T tiles[BLOCK * (N + 1)];
    A up1;
    if (upstream(r, up1)) return;
    const A w = weight_of(r) * up1;
    const int V = g.width, S = V | 1, tid = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T *const tile = tiles + wave * (64 * (N + 1));
    const bool packed = g.flat && g.inner_stride == V;
    Terms<A> t = {};
    for (int64_t i0 = (int64_t)blockIdx.x * BLOCK + wave * 64; i0 < r.rows; i0 += (int64_t)gridDim.x * BLOCK) {
        const int rows = r.rows - i0 < 64 ? (int)(r.rows - i0) : 64, n = rows * V;
        const int64_t i = i0 + tid;
        const bool mine = tid < rows;
        T *const own = tile + tid * S;
        if (packed) {
            const T *const x = (const T *)g.x + i0 * V;
            for (int e = tid * VEC; e < n; e += 64 * VEC) {
                if (e + VEC <= n) {
                    const Span<T, VEC> y = *(const Span<T, VEC> *)(x + e);
                    if (S == V) {
                        ((Line<T, VEC> *)(tile + e))->s = y;
                    } else {
                        int row = e / V, col = e - row * V;
#pragma unroll
                        for (int k = 0; k < VEC; ++k) {
                            tile[row * S + col] = y.e[k];
                            if (++col == V) col = 0, ++row;
                        }
                    }
                } else {
                    for (int k = e; k < n; ++k) tile[k / V * S + k % V] = x[k];
                }
            }
        } else if (mine) {
            const T *const x = (const T *)g.x + start_of(g, i);
            for (int k = 0; k < V; ++k) own[k] = x[k];
        }
        wave_lds();
        const bool on = mine && (!r.mask || r.mask[i]);
        if (on) {
            const int64_t at = action_of(g, i);
            const bool in = at >= 0 && at < V;
            A z[N], m = -INFINITY, s = 0, q = 0, lp;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                // (a place past the row is another's, and read in vain)
                z[k] = up(own[k]);
                if (k > N - 4) z[k] = k < V ? z[k] : A(-INFINITY);
                m = max_of(z[k], m);
            }
            const A xa = up(own[in ? at : 0]);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                z[k] = B::z(z[k], m);
                const A e = B::exp(z[k]);
                s += e;
                q = fma_of(e, B::floor(z[k]), q);
            }
            const Slope<A> c = slope_of(r, g, i, m, s, q, xa, at, w, t, lp);
            if (r.logp) r.logp[i] = lp;
            if (g.d) {
#pragma unroll
                for (int k = 0; k < N; ++k)
                    if (k <= N - 4 || k < V) own[k] = (T)(B::exp(z[k]) * fma_of(c.c1, B::floor(z[k]), c.c2));
                const A za = B::z(xa, m);
                if (in) own[at] = (T)(B::exp(za) * fma_of(c.c1, B::floor(za), c.c2) + c.gw);
            }
        } else if (mine) {
            if (r.logp) r.logp[i] = A(0);
            for (int k = 0; k < V; ++k) own[k] = (T)0.0f;
        }
        wave_lds();
        if (!g.d) continue;
        T *const d = (T *)g.d + i0 * V;
        for (int e = tid * VEC; e < n; e += 64 * VEC) {
            if (e + VEC <= n) {
                Span<T, VEC> y;
                if (S == V) {
                    y = ((const Line<T, VEC> *)(tile + e))->s;
                } else {
                    int row = e / V, col = e - row * V;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        y.e[k] = tile[row * S + col];
                        if (++col == V) col = 0, ++row;
                    }
                }
                *(Span<T, VEC> *)(d + e) = y;
            } else {
                for (int k = e; k < n; ++k) d[k] = tile[k / V * S + k % V];
            }
        }
        wave_lds();
    }
    if (r.sums) leave_sums<BLOCK>(t, r.sums);
}

// ------------------------------------------------------------------------- Gaussian head
//
// z, its products and the gradient are in the head's accumulation type; log-probabilities are
// summed in double, which costs nothing beside the memory and leaves the ratio to the old
// policy, a small difference of sums of up to 64 terms, its last digits.

struct Normal {
    int width, shared_std;
    const void *mean, *log_std, *actions;
    void *d_mean, *d_log_std;
};

// The block's sums of the shared deviations' gradient, D of them a thread, to its row of std_sums.
template <int D, typename A> __device__ void leave_std(const A (&v)[D], double *out)
{
    __shared__ double red[BLOCK / 64][D];
#pragma unroll
    for (int k = 0; k < D; ++k) {
        const double s = wave_sum((double)v[k]);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][k] = s;
    }
    __syncthreads();
    if (threadIdx.x < D) {
        double s = 0;
        for (int w = 0; w < BLOCK / 64; ++w) s += red[w][threadIdx.x];
        out[(int64_t)blockIdx.x * D + threadIdx.x] = s;
    }
}

// Up to four dimensions: a thread a decision.  What bounds it: memory; 8.2 M decisions of two
// dimensions in 50 us (295 MB: 5.9 TB/s, part of it from the last cache).
template <typename T, int D, bool SHARED>
__global__ __launch_bounds__(BLOCK) void k_gauss_rows(const Row<typename Acc<T>::type> r, const Normal g)
{
    typedef typename Acc<T>::type A;
    A up1;
    if (upstream(r, up1)) return;
    const A w = weight_of(r) * up1;
    const Span<T, D> *mean = (const Span<T, D> *)g.mean, *ls = (const Span<T, D> *)g.log_std;
    const Span<A, D> *act = (const Span<A, D> *)g.actions;
    Span<T, D> *dm = (Span<T, D> *)g.d_mean, *dl = (Span<T, D> *)g.d_log_std;
    Terms<A> t = {};
    A std_sum[D] = {};
    Span<T, D> l0;
    if (SHARED) l0 = ls[0];
    for (int64_t i = (int64_t)blockIdx.x * BLOCK + threadIdx.x; i < r.rows; i += (int64_t)gridDim.x * BLOCK) {
        const bool on = !r.mask || r.mask[i];
        Span<T, D> om, ol;
        if (!on) {
#pragma unroll
            for (int k = 0; k < D; ++k) om.e[k] = (T)0.0f;
            ol = om;
            if (r.logp) r.logp[i] = A(0);
        } else {
            const Span<T, D> mu = mean[i], lv = SHARED ? l0 : ls[i];
            const Span<A, D> a = act[i];
            A z[D], inv[D], H = 0;
            double lp = 0;
#pragma unroll
            for (int k = 0; k < D; ++k) {
                const A l = up(lv.e[k]);
                inv[k] = exp_of(-l);
                z[k] = (a.e[k] - up(mu.e[k])) * inv[k];
                lp += -0.5 * (double)(z[k] * z[k]) - (double)l - HALF_LOG_2PI;
                H += l + A(HALF_LOG_2PI + 0.5);
            }
            const A gl = decide(r, i, lp, H, t) * w;
            if (r.logp) r.logp[i] = (A)lp;
#pragma unroll
            for (int k = 0; k < D; ++k) {
                om.e[k] = (T)(gl * z[k] * inv[k]);
                const A y = gl * (z[k] * z[k] - A(1)) - r.entc * w;
                if (SHARED) std_sum[k] += y;
                else ol.e[k] = (T)y;
            }
        }
        if (dm) dm[i] = om;
        if (!SHARED && dl) dl[i] = ol;
    }
    if (r.sums) leave_sums<BLOCK>(t, r.sums);
    if (SHARED && r.std_sums) leave_std<D>(std_sum, r.std_sums);
}

// More dimensions: LANES threads a decision, a thread a dimension.
template <typename T, int LANES>
__global__ __launch_bounds__(BLOCK) void k_gauss_lanes(const Row<typename Acc<T>::type> r, const Normal g)
{
    typedef typename Acc<T>::type A;
    __shared__ double red[BLOCK / LANES][LANES];
    A up1;
    if (upstream(r, up1)) return;
    const A w = weight_of(r) * up1;
    constexpr int ROWS = BLOCK / LANES;
    const int D = g.width, k = threadIdx.x % LANES, row = threadIdx.x / LANES;
    const bool dim = k < D;
    const T *mean = (const T *)g.mean, *ls = (const T *)g.log_std;
    const A *act = (const A *)g.actions;
    T *dm = (T *)g.d_mean, *dl = (T *)g.d_log_std;
    Terms<A> t = {};
    A std_sum = 0;
    const A l0 = g.shared_std && dim ? up(ls[k]) : A(0);
    for (int64_t i0 = (int64_t)blockIdx.x * ROWS; i0 < r.rows; i0 += (int64_t)gridDim.x * ROWS) {
        const int64_t i = i0 + row, j = i * D + k;
        const bool mine = i < r.rows, on = mine && (!r.mask || r.mask[i]);
        A z = 0, inv = 0, h = 0;
        double lp = 0;
        if (on && dim) {
            const A l = g.shared_std ? l0 : up(ls[j]);
            inv = exp_of(-l);
            z = (act[j] - up(mean[j])) * inv;
            lp = -0.5 * (double)(z * z) - (double)l - HALF_LOG_2PI;
            h = l + A(HALF_LOG_2PI + 0.5);
        }
        lp = lanes_sum<LANES>(lp);
        h = lanes_sum<LANES>(h);
        if (!mine) continue;
        A om = 0, ol = 0;
        if (on) {
            Terms<A> x1 = {};
            const A gl = decide(r, i, lp, h, x1) * w;
            if (k == 0) add(t, x1);
            om = gl * z * inv;
            ol = gl * (z * z - A(1)) - r.entc * w;
            if (dim) std_sum += ol;
        }
        if (k == 0 && r.logp) r.logp[i] = on ? (A)lp : A(0);
        if (dim && dm) dm[j] = (T)om;
        if (dim && dl && !g.shared_std) dl[j] = (T)ol;
    }
    if (r.sums) leave_sums<BLOCK>(t, r.sums);
    if (!r.std_sums) return;
    red[row][k] = (double)std_sum;
    __syncthreads();
    if (threadIdx.x < D) {
        double s = 0;
        for (int q = 0; q < ROWS; ++q) s += red[q][threadIdx.x];
        r.std_sums[(int64_t)blockIdx.x * D + threadIdx.x] = s;
    }
}

// One workgroup joins what the others left: sums of the columns of v [blocks][W], W <= 64, in
// threads below W.  `red`: FINISH doubles.
constexpr int FINISH = 1024;
__device__ __forceinline__ double columns(const double *v, int blocks, int W, double *red)
{
    const int groups = FINISH / W, g = threadIdx.x / W, c = threadIdx.x - g * W;
    double s = 0;
    if (g < groups)
        for (int b = g; b < blocks; b += groups) s += v[(int64_t)b * W + c];
    __syncthreads();
    red[threadIdx.x] = s;
    __syncthreads();
    for (int n = groups; n > 1;) {
        const int h = (n + 1) / 2;
        if (g < n - h) red[threadIdx.x] += red[threadIdx.x + h * W];
        __syncthreads();
        n = h;
    }
    return red[threadIdx.x];
}

template <typename T>
__global__ __launch_bounds__(FINISH) void k_finish(const Row<typename Acc<T>::type> r, int blocks, int D,
                                                   typename Acc<T>::type *loss,
                                                   typename Acc<T>::type *stats, T *d_log_std)
{
    typedef typename Acc<T>::type A;
    __shared__ double red[FINISH];
    if (r.scale && r.skip_unit && *r.scale == A(1)) return;
    if (stats) {
        const double n = counted(r), s = columns(r.sums, blocks, 4, red);
        if (threadIdx.x == 0) *loss = (A)(r.sum ? s : s / n);
        else if (threadIdx.x < 4) stats[threadIdx.x - 1] = (A)(s / n);
    }
    if (d_log_std) {
        const double s = columns(r.std_sums, blocks, D, red);
        if (threadIdx.x < D) d_log_std[threadIdx.x] = (T)(A)s;
    }
}

// ------------------------------------------------------------------------------ host side

uint64_t sums_bytes() { return (uint64_t)MOST_BLOCKS * 4 * sizeof(double); }
uint64_t counts_bytes() { return (uint64_t)COUNTERS * sizeof(int32_t); }
// Elements of a part: the largest multiple of `vec` up to PART that leaves none shorter than vec.
int part_of(int width, int vec)
{
    int n = PART;
    while (width % n && width % n < vec) n -= vec;
    return n;
}

int check(const swarp_policy_t *a)
{
    swarp::set_error("");
    if (!a) return fail("arguments must be set");
    if (a->dtype < SWARP_F32 || a->dtype > SWARP_F16) return fail("unknown dtype");
    if (a->rows < 0 || a->width < 1) return fail("bad sizes");
    if (!a->loss != !a->stats) return fail("loss and stats are set together");
    if (!a->work || a->work_bytes < swarp_policy_work_bytes(a->rows, a->width))
        return fail("work must be set, swarp_policy_work_bytes() long");
    if ((uintptr_t)a->work & 15u) return fail("work must be 16-byte aligned");
    if (a->rows == 0) return 0;
    if (!a->head || !a->actions || !a->old_logp || !a->advantages)
        return fail("pointer arguments must be set");
    return 0;
}

template <typename T> Row<typename Acc<T>::type> row_of(const swarp_policy_t *a)
{
    typedef typename Acc<T>::type A;
    Row<A> r;
    r.rows = a->rows;
    r.lo = (A)(1.0 - a->clip_low);
    r.hi = (A)(1.0 + a->clip_high);
    r.klc = (A)a->kl_coef;
    r.entc = (A)a->entropy_coef;
    r.old = (const A *)a->old_logp;
    r.adv = (const A *)a->advantages;
    r.ref = (const A *)a->ref_logp;
    r.mask = a->mask;
    r.logp = (A *)a->logp;
    r.sums = a->stats ? (double *)a->work : nullptr;
    r.counts = (const int32_t *)((char *)a->work + sums_bytes());
    r.std_sums = nullptr;
    r.n_counts = 0;
    r.sum = a->sum;
    r.skip_unit = a->skip_unit;
    r.scale = (const A *)a->scale;
    return r;
}

template <typename A> void count(const swarp_policy_t *a, Row<A> &r, hipStream_t st)
{
    if (!a->mask) return;
    const int64_t want = (a->rows + 8 * BLOCK - 1) / (8 * BLOCK);
    r.n_counts = (int)(want < 1 ? 1 : want > COUNTERS ? COUNTERS : want);
    if (a->counted) return;
    hipLaunchKernelGGL(k_count, dim3(r.n_counts), dim3(BLOCK), 0, st, a->rows, a->mask,
                       (int32_t *)r.counts);
}

int blocks_for(int64_t units) { return (int)(units < 1 ? 1 : units > MOST_BLOCKS ? MOST_BLOCKS : units); }

template <typename T, int LANES, int E>
int cat_lanes(const Row<typename Acc<T>::type> &r, const Logits &g, hipStream_t st)
{
    const int blocks = blocks_for((r.rows + BLOCK / LANES - 1) / (BLOCK / LANES));
    hipLaunchKernelGGL((k_cat_lanes<T, LANES, E>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    return blocks;
}
template <typename T, int THREADS, int E>
int cat_block(const Row<typename Acc<T>::type> &r, const Logits &g, hipStream_t st)
{
    const int blocks = blocks_for(r.rows);
    hipLaunchKernelGGL((k_cat_block<T, THREADS, E>), dim3(blocks), dim3(THREADS), 0, st, r, g);
    return blocks;
}
template <typename T, int N>
int cat_rows(const Row<typename Acc<T>::type> &r, const Logits &g, hipStream_t st)
{
    const int blocks = blocks_for((r.rows + BLOCK - 1) / BLOCK);
    hipLaunchKernelGGL((k_cat_rows<T, N>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    return blocks;
}
template <typename T> int cat_parts(const Row<typename Acc<T>::type> &r, Logits g, void *parts, hipStream_t st)
{
    g.parts = parts;
    g.part = part_of(g.width, 16 / sizeof(T));
    g.splits = (g.width - 1) / g.part + 1;
    const int blocks = blocks_for(r.rows * g.splits);
    hipLaunchKernelGGL((k_cat_parts<T>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    hipLaunchKernelGGL((k_cat_join<T>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    return blocks;
}

template <typename T> void categorical(const swarp_policy_t *a, hipStream_t st)
{
    Row<typename Acc<T>::type> r = row_of<T>(a);
    count(a, r, st);
    const int V = a->width;
    Logits g = {a->inner, a->outer_stride, a->inner_stride, V, a->actions32, a->inner >= a->rows, 1, PART,
                a->head, a->actions, a->d_head, nullptr};
    void *const parts = (char *)a->work + sums_bytes() + counts_bytes() + MOST_BLOCKS * sizeof(double) * MOST_DIMS;
    int blocks = 0;
    // A thread's share of a short row.  What a decision costs beside its logits is paid by every
    // lane of its row, so 16-bit logits, of which a line holds twice as many, go 32 to a thread:
    // 200 M bfloat16 ones in rows of 250 take 189 us, 16 to a thread 237; 100 M float32 ones 178 and
    // 169.
    constexpr int E = sizeof(T) == 2 ? 32 : 16;
    if constexpr (sizeof(T) < 8) {
        switch ((V + 3) / 4) {
        case 1: blocks = cat_rows<T, 4>(r, g, st); break;
        case 2: blocks = cat_rows<T, 8>(r, g, st); break;
        case 3: blocks = cat_rows<T, 12>(r, g, st); break;
        case 4: blocks = cat_rows<T, 16>(r, g, st); break;
        case 5: blocks = cat_rows<T, 20>(r, g, st); break;
        case 6: blocks = cat_rows<T, 24>(r, g, st); break;
        case 7: blocks = cat_rows<T, 28>(r, g, st); break;
        case 8: blocks = cat_rows<T, 32>(r, g, st); break;
        }
    }
    if (blocks) {
    } else if (V <= 64) blocks = cat_lanes<T, 64 / E, E>(r, g, st);
    else if (V <= 128) blocks = cat_lanes<T, 128 / E, E>(r, g, st);
    else if (V <= 256) blocks = cat_lanes<T, 256 / E, E>(r, g, st);
    else if (V <= 512) blocks = cat_lanes<T, 512 / E, E>(r, g, st);
    else if (V <= 1024) blocks = cat_lanes<T, 1024 / E, E>(r, g, st);
    else if (V <= 2048) blocks = cat_lanes<T, 64, 32>(r, g, st);
    else if (V <= 4096) blocks = cat_block<T, 4096 / E, E>(r, g, st);
    else if (V <= 8192) blocks = cat_block<T, 256, 32>(r, g, st);
    else if (r.rows < FEW_ROWS || V > 65536 || sizeof(T) == 8) blocks = cat_parts<T>(r, g, parts, st);
    else if constexpr (sizeof(T) < 8) {
        if (V <= 16384) blocks = cat_block<T, 256, 64>(r, g, st);
        else if (V <= 32768) blocks = cat_block<T, 512, 64>(r, g, st);
        else if constexpr (sizeof(T) == 2) blocks = cat_block<T, 512, 128>(r, g, st);
        else blocks = cat_block<T, 1024, 64>(r, g, st);
    }
    if (a->stats)
        hipLaunchKernelGGL((k_finish<T>), dim3(1), dim3(FINISH), 0, st, r, blocks, 0,
                           (typename Acc<T>::type *)a->loss, (typename Acc<T>::type *)a->stats,
                           (T *)nullptr);
}

template <typename T, int D> int gauss_rows(const Row<typename Acc<T>::type> &r, const Normal &g, hipStream_t st)
{
    const int blocks = blocks_for((r.rows + BLOCK - 1) / BLOCK);
    if (g.shared_std)
        hipLaunchKernelGGL((k_gauss_rows<T, D, true>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    else
        hipLaunchKernelGGL((k_gauss_rows<T, D, false>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    return blocks;
}
template <typename T, int LANES>
int gauss_lanes(const Row<typename Acc<T>::type> &r, const Normal &g, hipStream_t st)
{
    const int blocks = blocks_for((r.rows + BLOCK / LANES - 1) / (BLOCK / LANES));
    hipLaunchKernelGGL((k_gauss_lanes<T, LANES>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    return blocks;
}

template <typename T> void gaussian(const swarp_policy_t *a, hipStream_t st)
{
    Row<typename Acc<T>::type> r = row_of<T>(a);
    count(a, r, st);
    const bool shared = a->shared_std && a->d_log_std;
    if (shared) r.std_sums = (double *)((char *)a->work + sums_bytes() + counts_bytes());
    const Normal g = {a->width, a->shared_std, a->head, a->log_std, a->actions, a->d_head,
                      a->d_log_std};
    int blocks;
    switch (a->width) {
    case 1: blocks = gauss_rows<T, 1>(r, g, st); break;
    case 2: blocks = gauss_rows<T, 2>(r, g, st); break;
    case 3: blocks = gauss_rows<T, 3>(r, g, st); break;
    case 4: blocks = gauss_rows<T, 4>(r, g, st); break;
    default:
        blocks = a->width <= 8    ? gauss_lanes<T, 8>(r, g, st)
                 : a->width <= 16 ? gauss_lanes<T, 16>(r, g, st)
                 : a->width <= 32 ? gauss_lanes<T, 32>(r, g, st)
                                  : gauss_lanes<T, 64>(r, g, st);
    }
    if (a->stats || shared)
        hipLaunchKernelGGL((k_finish<T>), dim3(1), dim3(FINISH), 0, st, r, blocks, a->width,
                           (typename Acc<T>::type *)a->loss, (typename Acc<T>::type *)a->stats,
                           shared ? (T *)a->d_log_std : nullptr);
}

// No decision: a loss of zero, as an empty sum.
template <typename T> void nothing(const swarp_policy_t *a, hipStream_t st)
{
    const Row<typename Acc<T>::type> r = row_of<T>(a);
    hipLaunchKernelGGL((k_finish<T>), dim3(1), dim3(FINISH), 0, st, r, 0, a->width,
                       (typename Acc<T>::type *)a->loss, (typename Acc<T>::type *)a->stats,
                       a->shared_std ? (T *)a->d_log_std : (T *)nullptr);
}

}  // namespace

#define FOR_DTYPE(F, a, st)                      \
    switch ((a)->dtype) {                        \
    case SWARP_F32: F<float>(a, st); break;      \
    case SWARP_F64: F<double>(a, st); break;     \
    case SWARP_BF16: F<bf16>(a, st); break;      \
    default: F<f16>(a, st); break;               \
    }

extern "C" {

uint64_t swarp_policy_work_bytes(int64_t rows, int32_t width)
{
    uint64_t n = sums_bytes() + counts_bytes() + MOST_BLOCKS * sizeof(double) * MOST_DIMS;
    if (width > PART && rows > 0) {  // whichever type the call has
        const int part = part_of(width, 2), p4 = part_of(width, 4), p8 = part_of(width, 8);
        const int least = part < p4 ? (part < p8 ? part : p8) : (p4 < p8 ? p4 : p8);
        n += (uint64_t)rows * ((width - 1) / least + 1) * 3 * sizeof(double);
    }
    return n;
}

int swarp_categorical_loss(const swarp_policy_t *a, void *stream)
{
    if (check(a)) return -1;
    hipStream_t st = (hipStream_t)stream;
    if (a->rows == 0) {
        FOR_DTYPE(nothing, a, st)
        return launched();
    }
    if (a->inner < 1) return fail("inner must be >= 1");
    FOR_DTYPE(categorical, a, st)
    return launched();
}

int swarp_gaussian_loss(const swarp_policy_t *a, void *stream)
{
    if (check(a)) return -1;
    if (a->width > MOST_DIMS) return fail("a Gaussian head has at most 64 dimensions");
    hipStream_t st = (hipStream_t)stream;
    if (a->rows == 0) {
        FOR_DTYPE(nothing, a, st)
        return launched();
    }
    if (!a->log_std) return fail("pointer arguments must be set");
    FOR_DTYPE(gaussian, a, st)
    return launched();
}

static int backward(const swarp_policy_t *a, int32_t skip_unit, const void *scale, swarp_policy_t &b)
{
    swarp::set_error("");
    if (!a || !scale) return fail("arguments must be set");
    b = *a;
    b.logp = b.loss = b.stats = nullptr;
    b.scale = scale;
    b.skip_unit = skip_unit;
    b.counted = 1;
    return 0;
}

int swarp_categorical_loss_bwd(const swarp_policy_t *a, int32_t skip_unit, const void *scale, void *stream)
{
    swarp_policy_t b;
    return backward(a, skip_unit, scale, b) ? -1 : swarp_categorical_loss(&b, stream);
}

int swarp_gaussian_loss_bwd(const swarp_policy_t *a, int32_t skip_unit, const void *scale, void *stream)
{
    swarp_policy_t b;
    return backward(a, skip_unit, scale, b) ? -1 : swarp_gaussian_loss(&b, stream);
}

}  // extern "C"
