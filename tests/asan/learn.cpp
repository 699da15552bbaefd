// The kernels and entry points of the policy update (gae.hip, policy.hip, adamw.hip) on the host
// under the sanitizers: buffers of exactly the extents the ABI documents, odd sizes, both layouts,
// strided logits, masked decisions that hold NaN and actions out of range.  Results against plain
// loops in double; the 8-bit moments, which are integer work, bit for bit.
#include <math.h>
#include <stdio.h>
#include <string.h>

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

std::mt19937 rng(11);
double uni() { return std::uniform_real_distribution<double>(0, 1)(rng); }
double nrm() { return std::normal_distribution<double>(0, 1)(rng); }

// A heap block of exactly n elements.
template <typename T> struct Buf {
    T *p;
    size_t n;
    explicit Buf(size_t k, int shift = 0) : base((char *)malloc((k + shift) * sizeof(T) + (k + shift == 0))), n(k)
    {
        p = (T *)base + shift;
    }
    ~Buf() { free(base); }
    T &operator[](size_t i) { return p[i]; }
    char *base;
};

int bad(const char *what, double err, double tol)
{
    if (err <= tol) return 0;
    printf("%s: error %g above %g\n", what, err, tol);
    return 1;
}

double off(double x, double y, double scale)
{
    if (isnan(x) || isnan(y)) return isnan(x) && isnan(y) ? 0 : 1e30;
    if (isinf(x) || isinf(y)) return x == y ? 0 : 1e30;
    return fabs(x - y) / (fabs(y) + scale);
}

template <typename T> int check_gae(int T_, int N, int group, int rows, bool flags, bool fin, double tol)
{
    const size_t L = T_, F = N / group;
    Buf<T> r(L * N), v((L + 1) * N), f(L * N), adv(L * N), ret(L * N), ga(L * N), gr(L * N), dr(L * N),
        dv((L + 1) * N), df(L * N);
    Buf<uint8_t> te(L * F), tr(L * F);
    for (size_t i = 0; i < L * N; ++i) r[i] = (T)nrm(), f[i] = (T)nrm(), ga[i] = (T)nrm(), gr[i] = (T)nrm();
    for (size_t i = 0; i < (L + 1) * N; ++i) v[i] = (T)nrm();
    for (size_t i = 0; i < L * F; ++i) te[i] = uni() < 0.1, tr[i] = uni() < 0.1;
    swarp_gae_t a = {};
    a.dtype = sizeof(T) == 4 ? SWARP_F32 : SWARP_F64;
    a.rows = rows;
    a.steps = L;
    a.columns = N;
    a.group = group;
    a.gamma = 0.9;
    a.lam = 0.8;
    a.rewards = r.p;
    a.values = v.p;
    if (flags) a.terminated = te.p, a.truncated = tr.p;
    if (fin) a.final_values = f.p;
    a.advantages = adv.p;
    a.returns = ret.p;
    a.adj_advantages = ga.p;
    a.adj_returns = gr.p;
    a.adj_rewards = dr.p;
    a.adj_values = dv.p;
    if (fin) a.adj_final_values = df.p;
    if (swarp_gae_fwd(&a, nullptr) || swarp_gae_bwd(&a, nullptr)) return printf("gae refused\n"), 1;
    double err = 0;
    for (int n = 0; n < N; ++n) {
        auto at = [&](int t) { return rows ? (size_t)n * L + t : (size_t)t * N + n; };
        auto av = [&](int t) { return rows ? (size_t)n * (L + 1) + t : (size_t)t * N + n; };
        auto af = [&](int t) { return rows ? (size_t)(n / group) * L + t : (size_t)t * F + n / group; };
        double A = 0;
        std::vector<double> wv(L + 1, 0.0), G(L);
        for (int t = T_ - 1; t >= 0; --t) {
            const bool e = flags && te[af(t)], c = flags && tr[af(t)];
            const double nx = e ? 0 : c && fin ? (double)f[at(t)] : (double)v[av(t + 1)];
            A = (double)r[at(t)] + 0.9 * nx - (double)v[av(t)] + (e || c ? 0 : 0.9 * 0.8 * A);
            err = fmax(err, off(adv[at(t)], A, 1));
            err = fmax(err, off(ret[at(t)], A + (double)v[av(t)], 1));
        }
        double S = 0;
        bool ends = true;
        for (int t = 0; t < T_; ++t) {
            const bool e = flags && te[af(t)], c = flags && tr[af(t)];
            S = (double)ga[at(t)] + (double)gr[at(t)] + (ends ? 0 : 0.9 * 0.8 * S);
            ends = e || c;
            wv[t] += (double)gr[at(t)] - S;
            if (!e && !(c && fin)) wv[t + 1] += 0.9 * S;
            err = fmax(err, off(dr[at(t)], S, 1));
            if (fin) err = fmax(err, off(df[at(t)], c && !e ? 0.9 * S : 0, 1));
        }
        for (int t = 0; t <= T_; ++t) err = fmax(err, off(dv[av(t)], wv[t], 1));
    }
    char what[96];
    snprintf(what, sizeof what, "gae %d x %d group %d rows %d flags %d fin %d", T_, N, group, rows, flags, fin);
    return bad(what, err, tol);
}

struct Decision {
    double loss, kl, clip, g;
};
Decision decide(double lp, double H, double old, double adv, double q, double klc, double entc)
{
    const double rho = exp(lp - old), b = fmin(fmax(rho, 0.8), 1.3);
    const bool c = b * adv < rho * adv;
    const double e = q - lp;
    Decision d;
    d.clip = c;
    d.kl = expm1(e) - e;
    d.loss = -(c ? b : rho) * adv + klc * d.kl - entc * H;
    d.g = (c ? 0 : -rho * adv) - klc * expm1(e);
    return d;
}

template <typename T> int code();
template <> int code<float>() { return SWARP_F32; }
template <> int code<double>() { return SWARP_F64; }
template <> int code<learn::bf16>() { return SWARP_BF16; }
template <> int code<learn::f16>() { return SWARP_F16; }

template <typename T> int check_cat(int outer, int inner, int V, int pad, bool masked, bool ref, bool ban, int shift, double tol, double gtol)
{
    typedef typename learn::Acc<T>::type A;
    const int64_t n = (int64_t)outer * inner;
    const int64_t os = (int64_t)(inner + 1) * (V + pad), is = V + pad;
    // rows of V + pad elements, inner of them and one more; the last row ends the block
    Buf<T> x((size_t)((outer - 1) * os + (inner - 1) * is + V), shift), d((size_t)n * V, shift), d2((size_t)n * V);
    for (size_t i = 0; i < x.n; ++i) x[i] = (T)(float)(nrm() * 2);
    Buf<int64_t> act(n);
    Buf<A> old(n), adv(n), q(n), logp(n), loss(1), stats(3), scale(1);
    Buf<uint8_t> mask(n);
    double count = 0;
    for (int64_t i = 0; i < n; ++i) {
        mask[i] = !masked || uni() < 0.7;
        count += mask[i];
        act[i] = mask[i] ? (int64_t)(uni() * V) : -100;
        old[i] = (A)(-1.5 + 0.2 * nrm()), q[i] = (A)(-1.5 + 0.2 * nrm());
        adv[i] = mask[i] ? (A)nrm() : (A)NAN;
        T *row = x.p + (i / inner) * os + (i % inner) * is;
        if (ban)
            for (int j = 0; j < V; ++j)
                if (j != act[i] && uni() < 0.3) row[j] = (T)(-INFINITY);
    }
    const double w = 1 / fmax(1, count);
    const uint64_t wb = swarp_policy_work_bytes(n, V);
    Buf<double> work(wb / 8);
    swarp_policy_t a = {};
    a.dtype = code<T>();
    a.width = V;
    a.rows = n;
    a.inner = inner;
    a.outer_stride = os;
    a.inner_stride = is;
    a.clip_low = 0.2;
    a.clip_high = 0.3;
    a.kl_coef = ref ? 0.1 : 0;
    a.entropy_coef = 0.05;
    a.head = x.p;
    a.actions = act.p;
    a.old_logp = old.p;
    a.advantages = adv.p;
    a.ref_logp = ref ? q.p : nullptr;
    a.mask = masked ? mask.p : nullptr;
    a.logp = logp.p;
    a.loss = loss.p;
    a.stats = stats.p;
    a.d_head = d.p;
    a.work = work.p;
    a.work_bytes = wb;
    if (swarp_categorical_loss(&a, nullptr)) return printf("cat refused: %s\n", swarp::message.c_str()), 1;
    // the backward with an upstream gradient of -2 into another buffer
    a.d_head = d2.p;
    scale[0] = (A)-2;
    if (swarp_categorical_loss_bwd(&a, 1, scale.p, nullptr)) return printf("cat refused: %s\n", swarp::message.c_str()), 1;
    double L = 0, E = 0, K = 0, C = 0, err = 0, gerr = 0, top = 0;
    std::vector<double> want((size_t)n * V, 0.0);
    for (int64_t i = 0; i < n; ++i) {
        if (!mask[i]) {
            err = fmax(err, off(logp[i], 0, 1));
            continue;
        }
        const T *row = x.p + (i / inner) * os + (i % inner) * is;
        double m = -INFINITY, s = 0, H = 0;
        for (int j = 0; j < V; ++j) m = fmax(m, (double)row[j]);
        for (int j = 0; j < V; ++j) s += exp((double)row[j] - m);
        for (int j = 0; j < V; ++j) {
            const double lp = (double)row[j] - m - log(s);
            if (exp(lp) > 0) H -= exp(lp) * lp;
        }
        const double lp = (double)row[act[i]] - m - log(s);
        const Decision t = decide(lp, H, old[i], adv[i], ref ? q[i] : old[i], ref ? 0.1 : 0, 0.05);
        L += t.loss, E += H, K += t.kl, C += t.clip;
        err = fmax(err, off(logp[i], lp, 1));
        for (int j = 0; j < V; ++j) {
            const double l = (double)row[j] - m - log(s), pj = exp(l);
            double &y = want[(size_t)i * V + j];
            y = w * (t.g * ((j == act[i]) - pj) + (pj > 0 ? 0.05 * pj * (l + H) : 0));
            top = fmax(top, fabs(y));
        }
    }
    err = fmax(err, fmax(off(loss[0], L * w, 0.1), fmax(off(stats[0], E * w, 1), fmax(off(stats[1], K * w, 0.1), off(stats[2], C * w, 1)))));
    for (size_t k = 0; k < want.size(); ++k) {
        gerr = fmax(gerr, fabs((double)d[k] - want[k]) / (top + 1e-30));
        gerr = fmax(gerr, fabs((double)d2[k] + 2 * want[k]) / (2 * top + 1e-30));
    }
    char what[128];
    snprintf(what, sizeof what, "cat %d: %d x %d x %d pad %d mask %d ref %d ban %d shift %d", code<T>(), outer, inner, V, pad, masked, ref, ban, shift);
    return bad(what, err, tol) | bad(what, gerr, gtol);
}

template <typename T> int check_gauss(int n, int D, bool shared, bool masked, double tol, double gtol)
{
    typedef typename learn::Acc<T>::type A;
    Buf<T> mu((size_t)n * D), ls(shared ? D : (size_t)n * D), dm((size_t)n * D), dl(ls.n);
    Buf<A> act((size_t)n * D), old(n), adv(n), logp(n), loss(1), stats(3);
    Buf<uint8_t> mask(n);
    for (size_t i = 0; i < mu.n; ++i) mu[i] = (T)(float)nrm(), act[i] = (A)((double)mu[i] + 0.5 * nrm());
    for (size_t i = 0; i < ls.n; ++i) ls[i] = (T)(float)(-0.5 + 0.2 * nrm());
    double count = 0;
    for (int i = 0; i < n; ++i) {
        mask[i] = !masked || uni() < 0.7;
        count += mask[i];
        old[i] = (A)(-0.7 * D + 0.2 * nrm()), adv[i] = mask[i] ? (A)nrm() : (A)NAN;
    }
    const double w = 1 / fmax(1, count);
    const uint64_t wb = swarp_policy_work_bytes(n, D);
    Buf<double> work(wb / 8);
    swarp_policy_t a = {};
    a.dtype = code<T>();
    a.width = D;
    a.rows = n;
    a.inner = 1;
    a.clip_low = 0.2;
    a.clip_high = 0.3;
    a.kl_coef = 0.1;
    a.entropy_coef = 0.05;
    a.shared_std = shared;
    a.head = mu.p;
    a.log_std = ls.p;
    a.actions = act.p;
    a.old_logp = old.p;
    a.advantages = adv.p;
    a.mask = masked ? mask.p : nullptr;
    a.logp = logp.p;
    a.loss = loss.p;
    a.stats = stats.p;
    a.d_head = dm.p;
    a.d_log_std = dl.p;
    a.work = work.p;
    a.work_bytes = wb;
    if (swarp_gaussian_loss(&a, nullptr)) return printf("gauss refused: %s\n", swarp::message.c_str()), 1;
    double L = 0, E = 0, err = 0, gerr = 0, top = 0, toph = 0;
    std::vector<double> wm((size_t)n * D, 0.0), wl(ls.n, 0.0);
    for (int i = 0; i < n; ++i) {
        if (!mask[i]) continue;
        double lp = 0, H = 0;
        for (int d = 0; d < D; ++d) {
            const double l = (double)ls[shared ? d : (size_t)i * D + d], z = ((double)act[(size_t)i * D + d] - (double)mu[(size_t)i * D + d]) * exp(-l);
            lp += -0.5 * z * z - l - 0.5 * log(2 * M_PI);
            H += l + 0.5 * log(2 * M_PI * M_E);
        }
        const Decision t = decide(lp, H, old[i], adv[i], old[i], 0.1, 0.05);
        L += t.loss, E += H;
        err = fmax(err, off(logp[i], lp, 1));
        for (int d = 0; d < D; ++d) {
            const size_t k = shared ? d : (size_t)i * D + d;
            const double l = (double)ls[k], z = ((double)act[(size_t)i * D + d] - (double)mu[(size_t)i * D + d]) * exp(-l);
            wm[(size_t)i * D + d] = w * t.g * z * exp(-l);
            wl[k] += w * (t.g * (z * z - 1) - 0.05);
        }
    }
    err = fmax(err, fmax(off(loss[0], L * w, 0.1), off(stats[0], E * w, 1)));
    for (double y : wm) top = fmax(top, fabs(y));
    for (double y : wl) toph = fmax(toph, fabs(y));
    for (size_t k = 0; k < wm.size(); ++k) gerr = fmax(gerr, fabs((double)dm[k] - wm[k]) / (top + 1e-30));
    for (size_t k = 0; k < wl.size(); ++k) gerr = fmax(gerr, fabs((double)dl[k] - wl[k]) / (toph + 1e-30));
    char what[96];
    snprintf(what, sizeof what, "gauss %d: %d x %d shared %d mask %d", code<T>(), n, D, shared, masked);
    return bad(what, err, tol) | bad(what, gerr, gtol);
}

template <typename P, typename G> int check_adamw(std::vector<int> sizes, int bits, bool master, int shift, double tol)
{
    size_t len = 0;
    std::vector<size_t> at;
    for (int n : sizes) at.push_back(len), len += (n + 255) / 256 * 256;
    Buf<float> m(len), v(len), mm(len), um(len), uv(len), ns(2);
    Buf<uint8_t> m8(len), v8(len), mb(len / 256), vb(len / 256);
    Buf<double> work(SWARP_NORM_WORK / 8);
    std::vector<Buf<P> *> ps;
    std::vector<Buf<G> *> gs;
    std::vector<swarp_tensor_t> tab;
    memset(m.p, 0, len * 4);
    memset(v.p, 0, len * 4);
    memset(m8.p, 0, len);
    memset(v8.p, 0, len);
    memset(mb.p, 0, len / 256);
    memset(vb.p, 0, len / 256);
    memset(mm.p, 0, len * 4);
    double sq = 0;
    for (size_t k = 0; k < sizes.size(); ++k) {
        ps.push_back(new Buf<P>(sizes[k], shift));
        gs.push_back(new Buf<G>(sizes[k], shift));
        for (int i = 0; i < sizes[k]; ++i) {
            (*ps[k])[i] = (P)(float)nrm();
            (*gs[k])[i] = (G)(float)nrm();
            sq += (double)(*gs[k])[i] * (double)(*gs[k])[i];
            if (master) mm[at[k] + i] = (float)(*ps[k])[i];
        }
        tab.push_back({ps[k]->p, gs[k]->p, sizes[k], (int64_t)at[k], code<P>(), code<G>()});
    }
    std::vector<std::vector<double>> w, ms, vs;
    for (size_t k = 0; k < sizes.size(); ++k) {
        w.push_back({});
        for (int i = 0; i < sizes[k]; ++i) w[k].push_back((double)(*ps[k])[i]);
        ms.push_back(std::vector<double>(sizes[k], 0.0));
        vs.push_back(std::vector<double>(sizes[k], 0.0));
    }
    int fails = 0;
    if (swarp_grad_norm(tab.data(), (int)tab.size(), 1.0, ns.p, work.p, nullptr)) return printf("norm refused\n"), 1;
    fails += bad("norm", off(ns[0], sqrt(sq), 0), 1e-5);
    for (int t = 1; t <= 2; ++t) {
        swarp_adamw_t a = {};
        a.bits = bits;
        a.seed = 7 + t;
        a.step = t;
        a.state_len = len;
        a.lr = 0.01;
        a.beta1 = 0.9;
        a.beta2 = 0.99;
        a.eps = 1e-8;
        a.weight_decay = 0.1;
        a.exp_avg = bits == 8 ? (void *)m8.p : (void *)m.p;
        a.exp_avg_sq = bits == 8 ? (void *)v8.p : (void *)v.p;
        a.avg_base = mb.p;
        a.sq_base = vb.p;
        a.master = master ? mm.p : nullptr;
        a.grad_scale = ns.p + 1;
        if (swarp_adamw(&a, tab.data(), (int)tab.size(), nullptr)) return printf("adamw refused: %s\n", swarp::message.c_str()), 1;
        if (bits == 8 && swarp_adamw_unpack(&a, um.p, uv.p, nullptr)) return printf("unpack refused\n"), 1;
        double err = 0, merr = 0;
        for (size_t k = 0; k < sizes.size(); ++k)
            for (int i = 0; i < sizes[k]; ++i) {
                const double g = (double)(*gs[k])[i] * ns[1];
                double &M = ms[k][i], &V = vs[k][i];
                M = 0.9 * M + 0.1 * g;
                V = 0.99 * V + 0.01 * g * g;
                w[k][i] = w[k][i] * (1 - 0.01 * 0.1) - 0.01 * (M / (1 - pow(0.9, t))) / (sqrt(V / (1 - pow(0.99, t))) + 1e-8);
                err = fmax(err, off((double)(*ps[k])[i], w[k][i], 1));
                const size_t j = at[k] + i;
                if (bits == 8) {
                    // within a code's step of the exact moment; the next step starts from the code
                    merr = fmax(merr, fmax(off(um[j], M, 1e-3), off(uv[j], V, 1e-6)) - 0.13);
                    M = um[j], V = uv[j];
                } else {
                    merr = fmax(merr, fmax(off(m[j], M, 1e-3), off(v[j], V, 1e-6)));
                }
                if (!master) w[k][i] = (double)(*ps[k])[i];
            }
        char what[96];
        snprintf(what, sizeof what, "adamw %d/%d bits %d master %d step %d", code<P>(), code<G>(), bits, master, t);
        fails += bad(what, err, tol) | bad(what, merr, 1e-5);
    }
    for (auto *b : ps) delete b;
    for (auto *b : gs) delete b;
    return fails;
}

}  // namespace

int main()
{
    int fails = 0;
    for (int rows = 0; rows < 2; ++rows)
        for (int fin = 0; fin < 2; ++fin) {
            for (int t : {1, 2, 7, 16, 17, 63, 130, 300})
                fails += check_gae<float>(t, 15, 3, rows, true, fin, 2e-5);
            fails += check_gae<double>(67, 130, 1, rows, true, fin, 1e-12);
            fails += check_gae<float>(5, 4, 4, rows, false, fin, 2e-5);
            fails += check_gae<float>(1100, 3, 1, rows, true, fin, 2e-5);
        }
    for (int V : {1, 2, 3, 5, 8, 9, 25, 31, 32, 33, 64, 65, 100, 127, 128, 200, 513, 1030})
        fails += check_cat<float>(3, 5, V, 0, V % 2, V % 3 == 0, V > 2 && V % 2, 0, 2e-6, 3e-6);
    for (int V : {1, 3, 9, 16, 25, 40, 64, 67, 129, 257, 1000, 2049})
        fails += check_cat<learn::bf16>(2, 7, V, V % 2, V % 3 == 0, true, V > 2, 1, 2e-6, 6e-3);
    for (int V : {3, 33, 600}) fails += check_cat<learn::f16>(2, 3, V, 3, true, true, true, 0, 2e-6, 2e-3);
    for (int V : {2, 30, 300}) fails += check_cat<double>(2, 3, V, 1, true, true, true, 0, 1e-13, 1e-13);
    for (int V : {1, 3}) fails += check_cat<double>(1, 3, V, 0, false, true, false, 0, 1e-13, 1e-13);
    for (int V : {8193, 8195}) fails += check_cat<double>(1, 1, V, 0, false, true, true, 0, 1e-12, 1e-12);
    for (int V : {4100, 8200, 20001}) {
        fails += check_cat<float>(1, 2, V, 1, false, true, true, 1, 3e-6, 3e-6);
        fails += check_cat<learn::bf16>(1, 2, V, 0, true, false, false, 0, 3e-6, 6e-3);
    }
    fails += check_cat<float>(1, 700, 9, 0, true, true, true, 0, 2e-6, 3e-6);
    for (int D : {1, 2, 3, 4, 5, 7, 8, 9, 17, 33, 64})
        for (int shared = 0; shared < 2; ++shared) {
            fails += check_gauss<float>(D < 5 ? 300 : 37, D, shared, D % 2, 5e-6, 1e-5);
            fails += check_gauss<learn::bf16>(29, D, shared, D % 3 == 0, 5e-6, 8e-3);
            fails += check_gauss<double>(19, D, shared, true, 1e-13, 1e-13);
        }
    const std::vector<int> sizes = {1, 0, 255, 256, 257, 4096, 5003, 3};
    for (int shift = 0; shift < 2; ++shift) {
        fails += check_adamw<float, float>(sizes, 32, false, shift, 2e-6);
        fails += check_adamw<float, float>(sizes, 8, false, shift, 2e-6);
        fails += check_adamw<learn::bf16, learn::bf16>(sizes, 32, false, shift, 8e-3);
        fails += check_adamw<learn::bf16, learn::bf16>(sizes, 8, false, shift, 8e-3);
        fails += check_adamw<learn::bf16, float>(sizes, 8, true, shift, 5e-3);
        fails += check_adamw<learn::f16, learn::f16>(sizes, 32, true, shift, 1e-3);
    }
    fails += check_adamw<float, float>(std::vector<int>(70, 5), 32, false, 0, 2e-6);
    printf("%d case(s) failed\n", fails);
    return fails != 0;
}
