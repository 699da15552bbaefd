// policy.hip -- the clipped policy loss with KL and entropy terms, and its gradient
// (swarp_categorical_loss, swarp_gaussian_loss).
//
// Per decision, with lp the log-probability of its action and e = q - lp:
//   l = -min(rho A, clamp(rho) A) + kl_coef (exp(e) - 1 - e) - entropy_coef H
//   g = dl/dlp = -(rho A where the unclipped branch is the smaller) - kl_coef (exp(e) - 1)
// Categorical: p = softmax(x), dl/dx_j = g (1[j = a] - p_j) + entropy_coef p_j (log p_j + H).
// Gaussian: z = (a - mu) / sigma, dl/dmu = g z / sigma, dl/dls = g (z^2 - 1) - entropy_coef.
#include <math.h>

#include "learn.hpp"

namespace {

using namespace learn;

constexpr int BLOCK = 256;
constexpr int MOST_BLOCKS = 2048;   // of a loss kernel: each leaves one row of sums
constexpr int COUNTERS = 256;       // blocks that count the mask
constexpr int MOST_DIMS = 64;       // of a Gaussian head
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

// Weight of a counted decision in the gradient: the same in every thread of the block.
template <typename A> __device__ A weight_of(const Row<A> &r)
{
    if (r.sum) return A(1);
    if (!r.mask) return A(1) / (A)r.rows;
    __shared__ double count;
    if (threadIdx.x < 64) {
        double c = 0;
        for (int i = threadIdx.x; i < r.n_counts; i += 64) c += r.counts[i];
        c = wave_sum(c);
        if (threadIdx.x == 0) count = c;
    }
    __syncthreads();
    return A(1) / (A)(count > 1 ? count : 1);
}

template <typename A> struct Terms {
    A loss, ent, kl, clipped;
};

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float expm1_of(float x) { return expm1f(x); }
__device__ __forceinline__ double expm1_of(double x) { return expm1(x); }
__device__ __forceinline__ float log_of(float x) { return logf(x); }
__device__ __forceinline__ double log_of(double x) { return log(x); }

// One decision's terms added to `t`; returns g.
template <typename A>
__device__ __forceinline__ A decide(const Row<A> &r, int64_t i, A lp, A H, Terms<A> &t)
{
    const A old = r.old[i], adv = r.adv[i];
    const A rho = exp_of(lp - old);
    const A bounded = rho < r.lo ? r.lo : (rho > r.hi ? r.hi : rho);
    const A first = rho * adv, second = bounded * adv;
    const bool clipped = second < first;
    const A e = (r.ref ? r.ref[i] : old) - lp;
    const A em = expm1_of(e), kl = em - e;
    A l = clipped ? -second : -first;
    A g = clipped ? A(0) : -first;
    if (r.klc != A(0)) {
        l += r.klc * kl;
        g -= r.klc * em;
    }
    if (r.entc != A(0)) l -= r.entc * H;
    t.loss += l;
    t.ent += H;
    t.kl += kl;
    t.clipped += clipped ? A(1) : A(0);
    return g;
}

// The block's sums of its threads' terms to row blockIdx.x of `sums`.
template <typename A> __device__ void leave_sums(const Terms<A> &t, double *sums)
{
    __shared__ double red[BLOCK / 64][4];
    const double v[4] = {(double)t.loss, (double)t.ent, (double)t.kl, (double)t.clipped};
    for (int k = 0; k < 4; ++k) {
        const double s = wave_sum(v[k]);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][k] = s;
    }
    __syncthreads();
    if (threadIdx.x < 4) {
        double s = 0;
        for (int w = 0; w < BLOCK / 64; ++w) s += red[w][threadIdx.x];
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

struct Logits {
    int64_t inner, outer_stride, inner_stride;
    int width, actions32;
    const void *x, *actions;
    void *d;
};

template <typename T>
__global__ __launch_bounds__(BLOCK) void k_categorical(const Row<typename Acc<T>::type> r, const Logits g)
{
    typedef typename Acc<T>::type A;
    A up1 = A(1);
    if (r.scale) {
        up1 = *r.scale;
        if (r.skip_unit && up1 == A(1)) return;
    }
    const A w = weight_of(r) * up1;
    const int lane = threadIdx.x & 63;
    const int64_t waves = (int64_t)gridDim.x * (BLOCK / 64);
    Terms<A> t = {};
    for (int64_t i = (int64_t)blockIdx.x * (BLOCK / 64) + (threadIdx.x >> 6); i < r.rows; i += waves) {
        const T *x = (const T *)g.x + (i / g.inner) * g.outer_stride + (i % g.inner) * g.inner_stride;
        T *d = g.d ? (T *)g.d + i * g.width : nullptr;
        if (r.mask && !r.mask[i]) {
            if (r.logp && lane == 0) r.logp[i] = A(0);
            if (d)
                for (int j = lane; j < g.width; j += 64) d[j] = (T)A(0);
            continue;
        }
        const int64_t at = g.actions32 ? (int64_t)((const int32_t *)g.actions)[i]
                                       : ((const int64_t *)g.actions)[i];
        A m = -INFINITY;
        for (int j = lane; j < g.width; j += 64) m = up(x[j]) > m ? up(x[j]) : m;
        m = wave_max(m);
        A s = 0, q = 0;
        for (int j = lane; j < g.width; j += 64) {
            A z = up(x[j]) - m;
            z = z < A(-1000) ? A(-1000) : z;  // (-inf: no term; NaN stays)
            const A e = exp_of(z);
            s += e;
            q += e * z;
        }
        s = wave_sum(s);
        q = wave_sum(q);
        const A ls = log_of(s), H = ls - q / s;
        const bool in = at >= 0 && at < g.width;
        const A lp = in ? (up(x[in ? at : 0]) - m) - ls : A(NAN);
        Terms<A> mine = {};
        const A gl = decide(r, i, lp, H + (in ? A(0) : A(NAN)), mine);
        if (lane == 0) {
            if (r.logp) r.logp[i] = lp;
            t.loss += mine.loss;
            t.ent += mine.ent;
            t.kl += mine.kl;
            t.clipped += mine.clipped;
        }
        if (!d) continue;
        const A gw = gl * w + (in ? A(0) : A(NAN)), ew = r.entc * w;
        for (int j = lane; j < g.width; j += 64) {
            A z = up(x[j]) - m;
            z = z < A(-1000) ? A(-1000) : z;
            const A p = exp_of(z) / s;
            A v = p * (ew * (z - ls + H) - gw);
            if (j == at) v += gw;
            d[j] = (T)v;
        }
    }
    if (r.sums) leave_sums(t, r.sums);
}

struct Normal {
    int width, shared_std;
    const void *mean, *log_std, *actions;
    void *d_mean, *d_log_std;
};

// One thread per decision.
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_gaussian(const Row<typename Acc<T>::type> r, const Normal g)
{
    typedef typename Acc<T>::type A;
    A up1 = A(1);
    if (r.scale) {
        up1 = *r.scale;
        if (r.skip_unit && up1 == A(1)) return;
    }
    const A w = weight_of(r) * up1;
    const int D = g.width;
    const T *mean = (const T *)g.mean, *ls = (const T *)g.log_std;
    const A *act = (const A *)g.actions;
    T *dm = (T *)g.d_mean, *dl = (T *)g.d_log_std;
    __shared__ double red[BLOCK / 64];
    Terms<A> t = {};
    for (int64_t i0 = (int64_t)blockIdx.x * BLOCK; i0 < r.rows; i0 += (int64_t)gridDim.x * BLOCK) {
        const int64_t i = i0 + threadIdx.x;
        const bool on = i < r.rows && (!r.mask || r.mask[i]);
        if (i >= r.rows) continue;
        if (!on) {
            if (r.logp) r.logp[i] = A(0);
            for (int d = 0; d < D; ++d) {
                if (dm) dm[i * D + d] = (T)A(0);
                if (dl && !g.shared_std) dl[i * D + d] = (T)A(0);
            }
            continue;
        }
        A lp = 0, H = 0;
        for (int d = 0; d < D; ++d) {
            const A l = up(ls[g.shared_std ? d : i * D + d]);
            const A z = (act[i * D + d] - up(mean[i * D + d])) * exp_of(-l);
            lp += A(-0.5) * z * z - l - A(HALF_LOG_2PI);
            H += l + A(HALF_LOG_2PI + 0.5);
        }
        const A gl = decide(r, i, lp, H, t) * w;
        if (r.logp) r.logp[i] = lp;
        for (int d = 0; d < D; ++d) {
            const A l = up(ls[g.shared_std ? d : i * D + d]), inv = exp_of(-l);
            const A z = (act[i * D + d] - up(mean[i * D + d])) * inv;
            if (dm) dm[i * D + d] = (T)(gl * z * inv);
            if (dl && !g.shared_std) dl[i * D + d] = (T)(gl * (z * z - A(1)) - r.entc * w);
        }
    }
    if (r.sums) leave_sums(t, r.sums);
    if (!r.std_sums) return;
    // the shared deviations' gradient, dimension by dimension
    for (int d = 0; d < D; ++d) {
        const A l = up(ls[d]), inv = exp_of(-l);
        double s = 0;
        for (int64_t i = (int64_t)blockIdx.x * BLOCK + threadIdx.x; i < r.rows;
             i += (int64_t)gridDim.x * BLOCK) {
            if (r.mask && !r.mask[i]) continue;
            A lp = 0;
            for (int k = 0; k < D; ++k) {
                const A lk = up(ls[k]);
                const A zk = (act[i * D + k] - up(mean[i * D + k])) * exp_of(-lk);
                lp += A(-0.5) * zk * zk - lk - A(HALF_LOG_2PI);
            }
            Terms<A> none = {};
            const A gl = decide(r, i, lp, A(0), none) * w;
            const A z = (act[i * D + d] - up(mean[i * D + d])) * inv;
            s += (double)(gl * (z * z - A(1)) - r.entc * w);
        }
        s = wave_sum(s);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int k = 1; k < BLOCK / 64; ++k) s += red[k];
            r.std_sums[(int64_t)blockIdx.x * D + d] = s;
        }
    }
}

// One block: the blocks' sums to the loss and the means, and to the shared deviations' gradient.
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_finish(const Row<typename Acc<T>::type> r, int blocks, int D,
                                                  typename Acc<T>::type *loss,
                                                  typename Acc<T>::type *stats, T *d_log_std)
{
    typedef typename Acc<T>::type A;
    if (r.scale && r.skip_unit && *r.scale == A(1)) return;
    __shared__ double red[BLOCK];
    __shared__ double n;
    if (threadIdx.x == 0) {
        double c = (double)r.rows;
        if (r.mask) {
            c = 0;
            for (int i = 0; i < r.n_counts; ++i) c += r.counts[i];
        }
        n = c > 1 ? c : 1;
    }
    if (stats) {
        const int k = threadIdx.x & 3;
        double s = 0;
        for (int b = threadIdx.x >> 2; b < blocks; b += BLOCK / 4) s += r.sums[4 * (int64_t)b + k];
        red[threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.x < 4) {
            for (int b = 1; b < BLOCK / 4; ++b) s += red[4 * b + k];
            if (k == 0) *loss = (A)(r.sum ? s : s / n);
            else stats[k - 1] = (A)(s / n);
        }
    }
    if (!d_log_std) return;
    for (int d = 0; d < D; ++d) {
        double s = 0;
        for (int b = threadIdx.x; b < blocks; b += BLOCK) s += r.std_sums[(int64_t)b * D + d];
        __syncthreads();
        red[threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int b = 1; b < BLOCK; ++b) s += red[b];
            d_log_std[d] = (T)(A)s;
        }
    }
}

// ------------------------------------------------------------------------------ host side

uint64_t sums_bytes() { return (uint64_t)MOST_BLOCKS * 4 * sizeof(double); }
uint64_t counts_bytes() { return (uint64_t)COUNTERS * sizeof(int32_t); }

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
    hipLaunchKernelGGL(k_count, dim3(r.n_counts), dim3(BLOCK), 0, st, a->rows, a->mask,
                       (int32_t *)r.counts);
}

int blocks_for(int64_t units) { return (int)(units < 1 ? 1 : units > MOST_BLOCKS ? MOST_BLOCKS : units); }

template <typename T> void categorical(const swarp_policy_t *a, hipStream_t st)
{
    Row<typename Acc<T>::type> r = row_of<T>(a);
    count(a, r, st);
    const int blocks = blocks_for((a->rows + BLOCK / 64 - 1) / (BLOCK / 64));
    const Logits g = {a->inner, a->outer_stride, a->inner_stride, a->width, a->actions32,
                      a->head, a->actions, a->d_head};
    hipLaunchKernelGGL((k_categorical<T>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    if (a->stats)
        hipLaunchKernelGGL((k_finish<T>), dim3(1), dim3(BLOCK), 0, st, r, blocks, 0,
                           (typename Acc<T>::type *)a->loss, (typename Acc<T>::type *)a->stats,
                           (T *)nullptr);
}

template <typename T> void gaussian(const swarp_policy_t *a, hipStream_t st)
{
    Row<typename Acc<T>::type> r = row_of<T>(a);
    count(a, r, st);
    const int blocks = blocks_for((a->rows + BLOCK - 1) / BLOCK);
    const bool shared = a->shared_std && a->d_log_std;
    if (shared) r.std_sums = (double *)((char *)a->work + sums_bytes() + counts_bytes());
    const Normal g = {a->width, a->shared_std, a->head, a->log_std, a->actions, a->d_head,
                      a->d_log_std};
    hipLaunchKernelGGL((k_gaussian<T>), dim3(blocks), dim3(BLOCK), 0, st, r, g);
    if (a->stats || shared)
        hipLaunchKernelGGL((k_finish<T>), dim3(1), dim3(BLOCK), 0, st, r, blocks, a->width,
                           (typename Acc<T>::type *)a->loss, (typename Acc<T>::type *)a->stats,
                           shared ? (T *)a->d_log_std : nullptr);
}

// No decision: a loss of zero, as an empty sum.
template <typename T> void nothing(const swarp_policy_t *a, hipStream_t st)
{
    const Row<typename Acc<T>::type> r = row_of<T>(a);
    hipLaunchKernelGGL((k_finish<T>), dim3(1), dim3(BLOCK), 0, st, r, 0, a->width,
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
    (void)rows;
    const uint64_t dims = width < MOST_DIMS ? (width < 1 ? 1 : width) : MOST_DIMS;
    return sums_bytes() + counts_bytes() + MOST_BLOCKS * dims * sizeof(double);
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

}  // extern "C"
