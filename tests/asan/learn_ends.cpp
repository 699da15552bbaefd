// The kernels of the policy update on the host under the sanitizers, at the ends of the number
// range: one case a run, named by the argument.  All outputs start as NaN, and a comparison that
// meets one fails, so an element that is never written shows.
#include <math.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <random>
#include <string>
#include <vector>

#include "learn.hpp"

// device functions of the GPU build that the host build has by other names
inline float __builtin_amdgcn_exp2f(float x) { return exp2f(x); }
inline float __builtin_amdgcn_logf(float x) { return log2f(x); }
inline void __builtin_amdgcn_sched_barrier(int) {}
struct alignas(16) float4 {
    float x, y, z, w;
};
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }

namespace g {
#include "gae.hip"
}
namespace p {
#include "policy.hip"
}
namespace o {
#include "adamw.hip"
}

namespace swarp {
std::string message;
int set_error(const char *m)
{
    message = m;
    return m[0] ? -1 : 0;
}
}  // namespace swarp

namespace {

template <typename T> struct Code;
template <> struct Code<float> { static constexpr int value = SWARP_F32; };
template <> struct Code<double> { static constexpr int value = SWARP_F64; };
template <> struct Code<learn::bf16> { static constexpr int value = SWARP_BF16; };
template <> struct Code<learn::f16> { static constexpr int value = SWARP_F16; };

// 1 and a line where got is not within tol of want; infinities have to be the same, and a NaN
// meets only a NaN that is wanted.
int differs(const char *what, double got, double want, double tol)
{
    const bool same = isnan(want) ? isnan(got) : isinf(want) ? got == want : fabs(got - want) <= tol;
    if (!same) printf("%s: %.17g, not %.17g (within %g)\n", what, got, want, tol);
    return !same;
}

// A policy loss over `n` decisions and its gradients for an upstream gradient of 1.
template <typename T> struct Loss {
    typedef typename learn::Acc<T>::type A;
    int n, width;
    bool gauss, shared;
    std::vector<T> head, std, d_head, d_std;
    std::vector<A> old, adv, ref, logp, loss, stats, taken;
    std::vector<int64_t> actions;
    std::vector<uint8_t> mask;
    std::vector<double> work;
    swarp_policy_t a = {};

    Loss(int n, int width, bool gauss = false, bool shared = false)
        : n(n), width(width), gauss(gauss), shared(shared), head((size_t)n * width, (T)0.0f),
          std(!gauss ? 0 : shared ? width : (size_t)n * width, (T)0.0f),
          d_head((size_t)n * width, (T)NAN), d_std(std.size(), (T)NAN), old(n, A(-1)), adv(n, A(1)),
          logp(n, A(NAN)), loss(1, A(NAN)), stats(3, A(NAN)), taken(gauss ? (size_t)n * width : 0, A(0)),
          actions(n, 0), work(swarp_policy_work_bytes(n, width) / 8, NAN)
    {
        a.dtype = Code<T>::value;
        a.width = width;
        a.shared_std = shared;
        a.rows = n;
        a.inner = n;
        a.inner_stride = width;
        a.clip_low = 0.2;
        a.clip_high = 0.3;
    }
    int run()
    {
        a.head = head.data();
        a.log_std = gauss ? std.data() : nullptr;
        a.actions = gauss ? (const void *)taken.data() : (const void *)actions.data();
        a.old_logp = old.data();
        a.advantages = adv.data();
        a.ref_logp = ref.empty() ? nullptr : ref.data();
        a.mask = mask.empty() ? nullptr : mask.data();
        a.logp = logp.data();
        a.loss = loss.data();
        a.stats = stats.data();
        a.d_head = d_head.data();
        a.d_log_std = gauss ? d_std.data() : nullptr;
        a.work = work.data();
        a.work_bytes = work.size() * 8;
        const int rc = gauss ? swarp_gaussian_loss(&a, nullptr) : swarp_categorical_loss(&a, nullptr);
        if (rc) printf("refused: %s\n", swarp::message.c_str());
        return rc != 0;
    }
};

// A reference that forbids the action taken: the loss is infinite, its slope along the
// log-probability g = -rho A + kl_coef (as exp(e) is 0), and the gradients are that times the
// head's.  Uniform logits, a unit Gaussian at its mean: rho = 1 with the old log-probability.
template <typename T> int forbidden(double tol)
{
    const double klc = 0.25;
    int bad = 0;
    for (int V : {3, 40, 4100}) {
        Loss<T> c(4, V);
        c.a.kl_coef = klc;
        c.ref.assign(4, (typename Loss<T>::A)(-log(V)));
        c.old = c.ref;
        c.ref[1] = -INFINITY;
        c.actions = {0, V - 1, 1, 0};
        bad += c.run();
        bad += differs("loss", c.loss[0], INFINITY, 0) + differs("kl", c.stats[1], INFINITY, 0);
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < V; ++j) {
                const double gi = i == 1 ? -1 + klc : -1;
                bad += differs("d_logits", (double)c.d_head[(size_t)i * V + j],
                               gi * ((j == c.actions[i]) - 1.0 / V) / 4, tol);
            }
    }
    for (int D : {2, 6})
        for (int shared = 0; shared < 2; ++shared) {
            Loss<T> c(3, D, true, shared);
            c.a.kl_coef = klc;
            c.taken.assign(c.taken.size(), 1);  // z = 1: dl/dmu = g, dl/dls = 0
            c.ref.assign(3, (typename Loss<T>::A)(D * (-0.5 - 0.5 * log(2 * M_PI))));
            c.old = c.ref;
            c.ref[2] = -INFINITY;
            bad += c.run();
            bad += differs("loss", c.loss[0], INFINITY, 0);
            for (size_t k = 0; k < c.d_head.size(); ++k)
                bad += differs("d_mean", (double)c.d_head[k], (k / D == 2 ? -1 + klc : -1) / 3, tol);
            for (size_t k = 0; k < c.d_std.size(); ++k) bad += differs("d_log_std", (double)c.d_std[k], 0, tol);
        }
    return bad;
}

// The KL term of a decision whose log-probability is exactly 0 (its only action), for reference
// log-probabilities e of all sizes: e^2 / 2 + e^3 / 6 + ..., to a few roundings of itself.
template <typename T> int kl(double least, double most, double tol)
{
    int bad = 0;
    for (double size = least; size <= most; size *= 20)
        for (double e : {size, -size}) {
            Loss<T> c(1, 1);
            c.a.kl_coef = 1;
            c.adv[0] = 0;
            c.ref.assign(1, (typename Loss<T>::A)e);
            long double want = 0, term = 1, x = c.ref[0];
            for (int k = 1; k < 60; ++k) {
                term *= x / k;
                if (k > 1) want += term;
            }
            bad += c.run() + differs("kl", c.stats[1], (double)want, tol * (double)want);
        }
    return bad;
}

// What is not finite reaches back (the adjoint: on) to the next end of an episode and no further,
// wherever the stretches of the scan lie, with lam = 0 and with factors whose product underflows.
template <typename T> int cut(int rows, double lam, T seed)
{
    const int L = 300, N = 2;
    const double carry = (double)(T)(0.5 * lam);
    std::vector<T> r((size_t)L * N, T(0)), v((size_t)(L + 1) * N, T(0)), adv(r.size(), T(NAN)), ret(adv), d_r(adv),
        d_v(v.size(), T(NAN)), up(r.size(), T(1));
    std::vector<uint8_t> te(r.size(), 0);
    auto at = [&](int t, int n) { return rows ? (size_t)n * L + t : (size_t)t * N + n; };
    for (size_t i = 0; i < r.size(); ++i) r[i] = T(0.25) * T(i % 7);
    r[at(290, 0)] = r[at(150, 1)] = seed;
    up[at(3, 0)] = up[at(200, 1)] = seed;
    te[at(9, 0)] = te[at(277, 0)] = te[at(100, 1)] = te[at(201, 1)] = 1;
    swarp_gae_t a = {};
    a.dtype = Code<T>::value;
    a.rows = rows;
    a.steps = L;
    a.columns = N;
    a.group = 1;
    a.gamma = 0.5;
    a.lam = lam;
    a.rewards = r.data();
    a.values = v.data();
    a.terminated = te.data();
    a.advantages = adv.data();
    a.returns = ret.data();
    a.adj_advantages = up.data();
    a.adj_rewards = d_r.data();
    a.adj_values = d_v.data();
    if (swarp_gae_fwd(&a, nullptr) || swarp_gae_bwd(&a, nullptr)) return printf("refused\n"), 1;
    int bad = 0;
    const double tol = 16 * (sizeof(T) == 4 ? 0x1p-24 : 0x1p-53) * 4;  // of values up to 4
    for (int n = 0; n < N; ++n) {
        double A = 0, G = 0;
        for (int t = L - 1; t >= 0; --t) {
            A = te[at(t, n)] ? (double)r[at(t, n)] : (double)r[at(t, n)] + carry * A;
            bad += differs("advantage", adv[at(t, n)], A, tol) + differs("return", ret[at(t, n)], A, tol);
        }
        for (int t = 0; t < L; ++t) {
            G = t == 0 || te[at(t - 1, n)] ? (double)up[at(t, n)] : (double)up[at(t, n)] + carry * G;
            bad += differs("d_rewards", d_r[at(t, n)], G, tol);
        }
    }
    return bad;
}

// Every gradient element against plain loops, the forward's and those of a backward with an
// upstream gradient of -2: remainders of spans, -inf logits, masked decisions that hold NaN.
std::mt19937 rng(5);
double uni() { return std::uniform_real_distribution<double>(0, 1)(rng); }
double nrm() { return std::normal_distribution<double>(0, 1)(rng); }

template <typename T> int gradients(int n, int width, bool gauss, bool shared, double tol)
{
    typedef typename learn::Acc<T>::type A;
    const double klc = 0.1, entc = 0.05;
    Loss<T> c(n, width, gauss, shared);
    c.a.kl_coef = klc;
    c.a.entropy_coef = entc;
    c.ref.resize(n);
    c.mask.resize(n);
    double count = 0;
    for (T &x : c.head) x = (T)(float)nrm();
    for (T &x : c.std) x = (T)(float)(0.2 * nrm());
    for (A &x : c.taken) x = (A)nrm();
    for (int i = 0; i < n; ++i) {
        c.mask[i] = i == 0 || uni() < 0.7;
        count += c.mask[i];
        c.actions[i] = c.mask[i] ? (int64_t)(uni() * width) : -100;
        c.adv[i] = c.mask[i] ? (A)nrm() : (A)NAN;
        for (int j = 0; j < width && !gauss; ++j)
            if (!c.mask[i]) c.head[(size_t)i * width + j] = (T)NAN;
            else if (j != c.actions[i] && uni() < 0.2) c.head[(size_t)i * width + j] = (T)-INFINITY;
    }
    std::vector<double> want(c.head.size(), 0.0), wants(c.std.size(), 0.0);
    double top = 0, tops = 0;
    for (int i = 0; i < n; ++i) {
        if (!c.mask[i]) continue;
        const T *row = &c.head[(size_t)i * width];
        double lp = 0, m = -INFINITY, s = 0, H = 0;
        for (int j = 0; j < width && !gauss; ++j) m = fmax(m, (double)row[j]);
        for (int j = 0; j < width && !gauss; ++j) s += exp((double)row[j] - m);
        for (int j = 0; j < width; ++j) {
            if (gauss) {
                const double l = (double)c.std[shared ? j : (size_t)i * width + j], z = ((double)c.taken[(size_t)i * width + j] - (double)row[j]) * exp(-l);
                lp += -0.5 * z * z - l - 0.5 * log(2 * M_PI);
            } else {
                const double l = (double)row[j] - m - log(s);
                if (exp(l) > 0) H -= exp(l) * l;
                if (j == c.actions[i]) lp = l;
            }
        }
        // (ratios away from the clip's bounds)
        c.old[i] = (A)(lp - (i % 3 == 0 ? 0.05 : i % 3 == 1 ? 0.5 : -0.5));
        c.ref[i] = (A)(lp + 0.3 * nrm());
        const double rho = exp(lp - (double)c.old[i]), b = fmin(fmax(rho, 0.8), 1.3), adv = c.adv[i];
        const double g = ((b * adv < rho * adv ? 0 : -rho * adv) - klc * expm1((double)c.ref[i] - lp)) / count;
        for (int j = 0; j < width; ++j) {
            double &y = want[(size_t)i * width + j];
            if (gauss) {
                const size_t k = shared ? j : (size_t)i * width + j;
                const double l = (double)c.std[k], z = ((double)c.taken[(size_t)i * width + j] - (double)row[j]) * exp(-l);
                y = g * z * exp(-l);
                wants[k] += g * (z * z - 1) - entc / count;
            } else {
                const double l = (double)row[j] - m - log(s), pj = exp(l);
                y = g * ((j == c.actions[i]) - pj) + (pj > 0 ? entc * pj * (l + H) / count : 0);
            }
            top = fmax(top, fabs(y));
        }
    }
    for (double y : wants) tops = fmax(tops, fabs(y));
    char what[64];
    snprintf(what, sizeof what, "%s %d: %d x %d shared %d", gauss ? "gauss" : "cat", Code<T>::value, n, width, shared);
    int bad = c.run();
    for (int pass = 0; pass < 2; ++pass) {
        const double up = pass ? -2 : 1;
        for (size_t k = 0; k < want.size(); ++k) bad += differs(what, (double)c.d_head[k], up * want[k], tol * 2 * top);
        for (size_t k = 0; k < wants.size(); ++k) bad += differs(what, (double)c.d_std[k], up * wants[k], tol * 2 * tops);
        std::fill(c.d_head.begin(), c.d_head.end(), (T)NAN);
        std::fill(c.d_std.begin(), c.d_std.end(), (T)NAN);
        A scale = A(-2);
        if (!pass) bad += gauss ? swarp_gaussian_loss_bwd(&c.a, pass, &scale, nullptr) : swarp_categorical_loss_bwd(&c.a, pass, &scale, nullptr);
    }
    return bad;
}

}  // namespace

int main(int argc, char **argv)
{
    const std::string what = argc > 1 ? argv[1] : "";
    int bad = -1;
    // a few roundings of terms of size 1: 16 of the type's
    if (what == "forbidden") bad = forbidden<float>(0x1p-20) + forbidden<double>(0x1p-48) + forbidden<learn::f16>(0x1p-9);
    // 16 roundings; above 1/2 the difference from e loses a digit in four, and float's exp two more
    if (what == "kl") bad = kl<float>(1e-15, 0.5, 0x1p-20) + kl<double>(1e-17, 3.0, 0x1p-49);
    if (what == "cut") {
        bad = 0;
        for (int rows = 0; rows < 2; ++rows)
            for (double lam : {0.0, -0.0, 0.04, 1e-7, 0.9})
                for (double seed : {(double)NAN, (double)INFINITY, -(double)INFINITY})
                    bad += cut<float>(rows, lam, (float)seed) + cut<double>(rows, lam, seed);
    }
    if (what == "gradients") {
        bad = 0;
        // float: log-probabilities of up to 12 to a few roundings, which the ratio takes whole;
        // 16-bit heads: half a step of the type and that
        for (int V : {3, 9, 33, 100, 2049, 8200}) bad += gradients<float>(7, V, false, false, 6e-6);
        for (int V : {5, 40, 129, 4100}) bad += gradients<learn::bf16>(5, V, false, false, 5e-3);
        bad += gradients<learn::f16>(5, 37, false, false, 1e-3) + gradients<double>(5, 30, false, false, 1e-14 * 8);
        for (int shared = 0; shared < 2; ++shared) {
            bad += gradients<float>(70, 2, true, shared, 6e-6) + gradients<float>(21, 5, true, shared, 1.2e-5);
            bad += gradients<learn::bf16>(33, 3, true, shared, 5e-3) + gradients<learn::f16>(19, 9, true, shared, 1e-3);
            bad += gradients<double>(11, 17, true, shared, 1e-14 * 8);
        }
    }
    printf("%s: %d wrong\n", what.c_str(), bad);
    return bad != 0;
}
