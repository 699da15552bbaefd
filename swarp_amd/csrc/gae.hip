// gae.hip -- generalised advantage estimation and its adjoint (swarp_gae_fwd / _bwd).
//
//   A_t = d_t + c_t A_{t+1},  d_t = r_t + gamma n_t - V_t,  c_t = 0 at an episode's end, else
//   gamma lam;  G_t = (gA_t + gR_t) + c_{t-1} G_{t-1} is the adjoint of d_t.
// One thread per column walks the steps.
#include "learn.hpp"

namespace {

using namespace learn;

// Element (t, n) of an array of L steps.
struct Place {
    int64_t step, col;
};

template <typename T> struct Args {
    int64_t steps, columns, group;
    int rows;
    T gamma, carry;  // gamma, gamma * lam
    const T *r, *v, *fin;
    const uint8_t *term, *trunc;
    T *adv, *ret;
    const T *g_adv, *g_ret;
    T *d_r, *d_v, *d_fin;
};

constexpr int BLOCK = 256;

template <typename T> __global__ __launch_bounds__(BLOCK) void k_gae_fwd(const Args<T> a)
{
    const int64_t n = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
    if (n >= a.columns) return;
    const int64_t L = a.steps, N = a.columns, f = n / a.group, F = N / a.group;
    T adv = 0;
    for (int64_t t = L - 1; t >= 0; --t) {
        const int64_t i = a.rows ? n * L + t : t * N + n;
        const int64_t j = a.rows ? n * (L + 1) + t : t * N + n, j1 = a.rows ? j + 1 : j + N;
        const int64_t k = a.rows ? f * L + t : t * F + f;
        const bool te = a.term && a.term[k], tr = a.trunc && a.trunc[k];
        T next = 0;
        if (!te) next = tr && a.fin ? a.fin[i] : a.v[j1];
        const T v = a.v[j];
        const T d = a.r[i] + a.gamma * next - v;
        adv = te || tr ? d : d + a.carry * adv;
        a.adv[i] = adv;
        a.ret[i] = adv + v;
    }
}

template <typename T> __global__ __launch_bounds__(BLOCK) void k_gae_bwd(const Args<T> a)
{
    const int64_t n = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
    if (n >= a.columns) return;
    const int64_t L = a.steps, N = a.columns, f = n / a.group, F = N / a.group;
    T G = 0, into = 0;  // the adjoint of the step before, and what it sends to V_t
    bool ends = true;
    for (int64_t t = 0; t <= L; ++t) {
        const int64_t i = a.rows ? n * L + t : t * N + n;
        const int64_t j = a.rows ? n * (L + 1) + t : t * N + n;
        if (t == L) {
            if (a.d_v) a.d_v[j] = into;
            break;
        }
        const int64_t k = a.rows ? f * L + t : t * F + f;
        const bool te = a.term && a.term[k], tr = a.trunc && a.trunc[k];
        const T gr = a.g_ret ? a.g_ret[i] : T(0);
        const T g = (a.g_adv ? a.g_adv[i] : T(0)) + gr;
        G = ends ? g : g + a.carry * G;
        ends = te || tr;
        if (a.d_r) a.d_r[i] = G;
        if (a.d_v) a.d_v[j] = gr - G + into;
        if (a.d_fin) a.d_fin[i] = tr && !te ? a.gamma * G : T(0);
        into = te || (tr && a.fin) ? T(0) : a.gamma * G;
    }
}

template <typename T> Args<T> args_of(const swarp_gae_t *a)
{
    Args<T> k;
    k.steps = a->steps;
    k.columns = a->columns;
    k.group = a->group;
    k.rows = a->rows;
    k.gamma = (T)a->gamma;
    k.carry = (T)(a->gamma * a->lam);
    k.r = (const T *)a->rewards;
    k.v = (const T *)a->values;
    k.fin = (const T *)a->final_values;
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
    if (a->columns >= (int64_t)BLOCK << 31) return fail("too many columns");
    return 0;
}

template <typename T> void fwd(const swarp_gae_t *a, hipStream_t st)
{
    hipLaunchKernelGGL((k_gae_fwd<T>), dim3((unsigned)((a->columns + BLOCK - 1) / BLOCK)),
                       dim3(BLOCK), 0, st, args_of<T>(a));
}

template <typename T> void bwd(const swarp_gae_t *a, hipStream_t st)
{
    hipLaunchKernelGGL((k_gae_bwd<T>), dim3((unsigned)((a->columns + BLOCK - 1) / BLOCK)),
                       dim3(BLOCK), 0, st, args_of<T>(a));
}

}  // namespace

extern "C" {

int swarp_gae_fwd(const swarp_gae_t *a, void *stream)
{
    if (check(a)) return -1;
    if (a->steps == 0 || a->columns == 0) return 0;
    if (!a->rewards || !a->values || !a->advantages || !a->returns)
        return fail("pointer arguments must be set");
    if (a->dtype == SWARP_F32) fwd<float>(a, (hipStream_t)stream);
    else fwd<double>(a, (hipStream_t)stream);
    return launched();
}

int swarp_gae_bwd(const swarp_gae_t *a, void *stream)
{
    if (check(a)) return -1;
    if (a->columns == 0) return 0;
    if (a->adj_final_values && !a->final_values)
        return fail("adj_final_values without final_values");
    if (a->dtype == SWARP_F32) bwd<float>(a, (hipStream_t)stream);
    else bwd<double>(a, (hipStream_t)stream);
    return launched();
}

}  // extern "C"
