"""The policy update on the GPU -- gae, the policy losses, AdamW -- against their definitions in
float64, at the sizes and masks where they can go wrong, their gradients against the formula's and
against differences, and their refusals."""

import copy
import math

import pytest
import torch

from swarp_amd import (AdamW, AdamWState, adamw_state, adamw_step, categorical_policy_loss, gae,
                       gaussian_policy_loss, grad_norm)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# largest relative error of one rounding to nearest: 24, 53, 8 and 11 bits of significand
EPS = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.bfloat16: 2.0 ** -8,
       torch.float16: 2.0 ** -11}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# -------------------------------------------------------------------------------------- gae


def gae_ref(r, v, te, tr, fin, gamma, lam):
    """The definition, time first, step by step."""
    T = r.shape[0]
    a, out = torch.zeros_like(v[0]), [None] * T
    for t in reversed(range(T)):
        nxt = v[t + 1] if fin is None else torch.where(tr[t], fin[t], v[t + 1])
        d = r[t] + gamma * torch.where(te[t], torch.zeros_like(nxt), nxt) - v[t]
        a = d + torch.where(te[t] | tr[t], torch.zeros_like(a), gamma * lam * a)
        out[t] = a
    adv = torch.stack(out)
    return adv, adv + v[:-1]


def gae_case(T, E, A, dtype, seed):
    g = gen(seed)

    def rn(*s):
        return torch.randn(*s, generator=g, device=DEV, dtype=torch.float64).to(dtype)
    te = torch.rand(T, E, generator=g, device=DEV) < 0.1
    tr = torch.rand(T, E, generator=g, device=DEV) < 0.1
    return rn(T, E, A), rn(T + 1, E, A), te, tr, rn(T, E, A), rn(T, E, A), rn(T, E, A)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("final", [False, True])
@pytest.mark.parametrize("T,E,A", [(1, 3, 2), (2, 1, 1), (7, 5, 4), (8, 70, 1), (9, 3, 3), (64, 2, 5),
                                   (129, 13, 1), (513, 2, 2), (2049, 1, 3), (40, 400, 16)])
def test_gae_and_its_adjoint(T, E, A, final, last, dtype):
    r, v, te, tr, fin, ga, gr = gae_case(T, E, A, dtype, 3 * T + E)
    fin = fin if final else None
    x = [t.double().requires_grad_(True) for t in ([r, v] + ([fin] if final else []))]
    f = (te[..., None].expand(T, E, A), tr[..., None].expand(T, E, A))
    want = gae_ref(x[0], x[1], *f, x[2] if final else None, 0.97, 0.9)
    gwant = torch.autograd.grad(want, x, (ga.double(), gr.double()))

    def lay(t):
        return t.movedim(0, -1).contiguous() if last else t
    y = [lay(t).requires_grad_(True) for t in ([r, v] + ([fin] if final else []))]
    got = gae(y[0], y[1], lay(te), lay(tr), y[2] if final else None, gamma=0.97, lam=0.9,
              time_dim=-1 if last else 0)
    ggot = torch.autograd.grad(got, y, (lay(ga), lay(gr)))
    # sums of at most 1 / (1 - 0.873) terms' weight, each a few operations: 64 roundings of the
    # largest magnitude
    for a, b in zip((*got, *ggot), (*want, *gwant)):
        b = lay(b.detach())
        tol = 64 * EPS[dtype] * float(b.abs().max())
        assert float((a.detach().double() - b).abs().max()) <= tol
    with torch.no_grad():
        plain = gae(y[0], y[1], lay(te), lay(tr), y[2] if final else None, gamma=0.97, lam=0.9,
                    time_dim=-1 if last else 0)
    assert torch.equal(plain.advantages, got.advantages) and torch.equal(plain.returns, got.returns)


def test_gae_against_differences():
    r, v, te, tr, fin, _, _ = gae_case(11, 2, 2, torch.float64, 5)
    r, v, fin = (t.requires_grad_(True) for t in (r, v, fin))
    assert torch.autograd.gradcheck(lambda *x: gae(x[0], x[1], te, tr, x[2]), (r, v, fin))
    assert torch.autograd.gradcheck(
        lambda a, b: gae(a, b, time_dim=-1).returns,
        (torch.randn(3, 20, device=DEV, dtype=torch.float64, requires_grad=True),
         torch.randn(3, 21, device=DEV, dtype=torch.float64, requires_grad=True)))


@pytest.mark.parametrize("last", [False, True])
def test_gae_reads_no_value_across_an_end(last):
    """Values that no step reads may be NaN; nothing carries over an end, not even infinities."""
    T, N = 700, 3
    r = torch.ones(T, N, device=DEV)
    v = torch.zeros(T + 1, N, device=DEV)
    te = torch.zeros(T, N, dtype=torch.bool, device=DEV)
    te[350] = True
    v[351:] = math.nan
    if last:
        r, v, te = (t.T.contiguous() for t in (r, v, te))
    adv = gae(r, v, te, time_dim=-1 if last else 0).advantages
    adv = adv.T if last else adv
    assert torch.isfinite(adv[:351]).all() and torch.isnan(adv[351:]).all()
    assert float(adv[350, 0]) == 1.0


def test_gae_shapes():
    z = gae(torch.zeros(0, 4, device=DEV), torch.ones(1, 4, device=DEV))
    assert z.advantages.shape == (0, 4)
    v = torch.ones(1, 4, device=DEV, requires_grad=True)
    gae(torch.zeros(0, 4, device=DEV), v).returns.sum().backward()
    assert torch.equal(v.grad, torch.zeros_like(v))
    assert gae(torch.zeros(5, 0, device=DEV), torch.zeros(6, 0, device=DEV)).returns.shape == (5, 0)
    one = gae(torch.ones(3, device=DEV), torch.zeros(4, device=DEV), gamma=1.0, lam=1.0)
    assert torch.equal(one.advantages, torch.tensor([3.0, 2.0, 1.0], device=DEV))
    # a view of every second column is taken as it reads
    r, v = torch.randn(9, 8, device=DEV), torch.randn(10, 8, device=DEV)
    assert torch.equal(gae(r[:, ::2], v[:, ::2]).returns,
                       gae(r[:, ::2].contiguous(), v[:, ::2].contiguous()).returns)


def test_gae_refuses():
    r, v = torch.zeros(4, 3, device=DEV), torch.zeros(5, 3, device=DEV)
    f = torch.zeros(4, 3, dtype=torch.bool, device=DEV)
    with pytest.raises(ValueError, match="values"):
        gae(r, v[:4])
    with pytest.raises(TypeError, match="float32 or float64"):
        gae(r.half(), v.half())
    with pytest.raises(TypeError, match="values"):
        gae(r, v.double())
    with pytest.raises(TypeError, match="terminated"):
        gae(r, v, f.float())
    with pytest.raises(ValueError, match="terminated"):
        gae(r, v, f[:3])
    with pytest.raises(ValueError, match="same shape"):
        gae(r, v, f, f[:, 0])
    with pytest.raises(ValueError, match="gamma"):
        gae(r, v, gamma=1.5)
    with pytest.raises(ValueError, match="time_dim"):
        gae(torch.zeros(2, 3, 4, device=DEV), torch.zeros(2, 4, 4, device=DEV), time_dim=1)
    with pytest.raises(ValueError, match="is on"):
        gae(r, v.cpu())


# ------------------------------------------------------------------------------ policy losses

CLIP = (0.2, 0.3)


def loss_ref(logp, entropy, old, adv, ref, mask, kl_c, ent_c, total):
    on = torch.ones_like(old, dtype=torch.bool) if mask is None else mask
    logp, entropy, old, adv = logp[on], entropy[on], old.double()[on], adv.double()[on]
    e = (old if ref is None else ref.double()[on]) - logp
    ratio = torch.exp(logp - old)
    first, second = ratio * adv, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * adv
    low = torch.where(second < first, second.detach() * 0 + second, first)
    kl = torch.special.expm1(e) - e
    n = 1 if total else max(1, int(on.sum()))
    loss = (-low + kl_c * kl - ent_c * entropy).sum() / n
    n = max(1, int(on.sum()))
    return loss, entropy.sum() / n, kl.sum() / n, (second < first).double().sum() / n


def rows_of(n, g, logp, mask, ref, dtype):
    """Inputs of n decisions, their ratios kept away from the clip bounds."""
    d = torch.randn(n, generator=g, device=DEV, dtype=torch.float64) * 0.2
    for b in (math.log(1 - CLIP[0]), math.log(1 + CLIP[1])):
        d = torch.where((d - b).abs() < 1e-2, d + 0.05, d)
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    old = (logp - d).to(wide)
    adv = torch.randn(n, generator=g, device=DEV, dtype=wide)
    q = (logp + 0.3 * torch.randn(n, generator=g, device=DEV, dtype=torch.float64)).to(wide)
    m = None
    if mask:
        m = torch.rand(n, generator=g, device=DEV) < 0.7
        adv = torch.where(m, adv, math.nan)
    return old, adv, (q if ref else None), m


def close(name, got, want, tol):
    err = float((got.detach().double() - want).abs().max()) if got.numel() else 0.0
    assert err <= tol, f"{name}: {err:.3e} > {tol:.3e}"


def check_loss(op, heads, actions, old, adv, ref, mask, logp, entropy, heads64, span, reduction,
               kl_c, ent_c):
    """One call and its gradient against float64.  `span`: the largest |logp| and the like."""
    dtype = heads[0].dtype
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    want = loss_ref(logp.reshape(-1), entropy.reshape(-1), old.reshape(-1), adv.reshape(-1),
                    None if ref is None else ref.reshape(-1),
                    None if mask is None else mask.reshape(-1), kl_c, ent_c, reduction == "sum")
    up = 512.0 if dtype == torch.float16 else 1.0
    gwant = torch.autograd.grad(want[0] * up, heads64, allow_unused=True)
    x = [h.detach().requires_grad_(True) for h in heads]
    got = op(*x, actions, old, adv, ref, mask, clip=CLIP, kl_coef=kl_c, entropy_coef=ent_c,
             reduction=reduction)
    (got.loss * up if up != 1.0 else got.loss).backward()
    on = torch.ones_like(old, dtype=torch.bool) if mask is None else mask
    # a log-probability is a sum of a few terms up to `span`; a ratio's relative error is a
    # log-probability's absolute one
    lp_tol = 16 * EPS[wide] * (1 + span)
    close("logp", got.logp, torch.where(on, logp, 0.0), lp_tol)
    n = 1 if reduction == "mean" else max(1, int(on.sum()))
    size = 1 + float(torch.where(on, adv, 0.0).abs().max()) * 3 + abs(ent_c) * float(entropy.abs().max())
    close("loss", got.loss, want[0].detach(), lp_tol * size * n)
    close("entropy", got.entropy, want[1].detach(), lp_tol * 4)
    close("kl", got.kl, want[2].detach(), lp_tol * 4)
    close("clip_fraction", got.clip_fraction, want[3].detach(), 4 * EPS[wide])
    for h, w in zip(x, gwant):
        w = torch.zeros_like(h, dtype=torch.float64) if w is None else w
        top = float(w.abs().max())
        # the rounding to the head's type, and the terms' own error relative to the largest
        bound = EPS[dtype] * w.abs() * (0 if dtype == wide else 1.01) + 4 * lp_tol * top
        bound = bound + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert bool(((h.grad.double() - w).abs() <= bound + 1e-300).all()), (
            float(((h.grad.double() - w).abs() - bound).max()), top)
        assert not h.grad[~on].any() if h.shape[:on.dim()] == on.shape else True
    return got, x


WIDTHS = [1, 2, 3, 8, 9, 16, 25, 32, 33, 64, 65, 100, 128, 200, 256, 300, 512, 700, 1024, 1500, 2048,
          3001, 5000]


def cat_case(lead, V, dtype, seed, ban, spread=2.0):
    g = gen(seed)
    x = torch.randn(*lead, V, generator=g, device=DEV) * spread
    if ban and V > 1:
        x[..., 1:].masked_fill_(torch.rand(*lead, V - 1, generator=g, device=DEV) < 0.2, -math.inf)
    x = x.to(dtype)
    f = x.double()
    act = torch.argmax(f - torch.log(-torch.log(torch.rand(*lead, V, generator=g, device=DEV,
                                                           dtype=torch.float64))), -1)
    return g, x, act


def cat_ref(x, act):
    x64 = x.double().detach().requires_grad_(True)
    lsm = torch.log_softmax(x64, -1)
    lp = lsm.gather(-1, act.clamp(min=0, max=x.shape[-1] - 1)[..., None])[..., 0]
    ent = -(lsm.exp() * torch.where(torch.isinf(lsm), torch.zeros_like(lsm), lsm)).sum(-1)
    return x64, lp, ent


def run_cat(lead, V, dtype, seed, ban=False, mask=False, ref=False, reduction="mean", kl_c=None,
            ent_c=0.05, x=None, act32=False):
    g, made, act = cat_case(lead, V, dtype, seed, ban)
    if x is not None:
        x.copy_(made)
    x = made if x is None else x
    x64, lp, ent = cat_ref(x, act)
    old, adv, q, m = (None if t is None else t.view(lead) for t in
                      rows_of(math.prod(lead), g, lp.detach().reshape(-1), mask, ref, dtype))
    act = act if m is None else torch.where(m, act, -100)
    act = act.int() if act32 else act
    # (the reference's gradient is of the decisions that count: those of the others are zero)
    return check_loss(categorical_policy_loss, [x], act, old, adv, q, m, lp, ent, [x64],
                      float(torch.where(torch.isinf(x64), 0.0, x64).detach().abs().max()) + math.log(V),
                      reduction, (0.1 if ref else 0.0) if kl_c is None else kl_c, ent_c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("V", WIDTHS)
def test_categorical(V, dtype):
    run_cat((37,), V, dtype, V, ban=V % 3 == 1, mask=V % 2 == 1, ref=V % 5 == 0,
            reduction="sum" if V % 7 == 0 else "mean", act32=V % 4 == 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(257, 8193), (256, 16384), (260, 16391), (256, 32769),
                                    (256, 65535), (3, 8193), (2, 40001), (1, 131077), (2, 70001)])
def test_categorical_long_rows(rows, V, dtype):
    run_cat((rows,), V, dtype, V, ban=V % 2 == 1, mask=rows % 2 == 1, ref=True)


@pytest.mark.parametrize("rows,V", [(1, 5), (255, 9), (256, 9), (257, 25), (5000, 4), (3000, 40),
                                    (40000, 9)])
def test_categorical_many_rows(rows, V):
    run_cat((rows,), V, torch.float32, rows, ban=True, mask=True, ref=True)


@pytest.mark.parametrize("V", [7, 33, 600, 9001])
def test_categorical_reads_a_slice_where_it_lies(V):
    """logits[:, :-1] and other strides over the leading axes; odd offsets."""
    base = torch.zeros(3, 6, V, device=DEV, dtype=torch.bfloat16)
    run_cat((3, 5), V, torch.bfloat16, V, mask=True, ref=True, x=base[:, :-1])
    flat = torch.zeros(3 * 5 * (V + 3) + 1, device=DEV)
    view = flat[1:].view(3, 5, V + 3)[..., 2:V + 2]
    run_cat((3, 5), V, torch.float32, V + 1, ban=True, x=view)
    run_cat((5, 3), V, torch.float32, V + 2, x=torch.zeros(3, 5, V, device=DEV).transpose(0, 1))
    wide = torch.zeros(3, 5, 2 * V, device=DEV)[..., ::2]
    run_cat((3, 5), V, torch.float32, V + 3, x=wide)


@pytest.mark.parametrize("V", [9, 50, 3000, 20000])
def test_categorical_masks_of_the_lowest_value(V):
    """Logits at the type's lowest value weigh nothing beside others and are equal among
    themselves; a row of nothing else is uniform."""
    for dtype in (torch.float32, torch.bfloat16):
        low = torch.finfo(dtype).min
        x = torch.full((2, V), low, dtype=dtype, device=DEV)
        x[0, :2] = 1.0
        x.requires_grad_(True)
        z = torch.zeros(2, device=DEV)
        r = categorical_policy_loss(x, torch.tensor([1, V - 1], device=DEV), z - 1, z + 1,
                                    entropy_coef=0.1)
        r.loss.backward()
        want = torch.tensor([math.log(0.5), -math.log(V)], dtype=torch.float64)
        close("logp", r.logp.cpu(), want, 1e-5)
        assert abs(float(r.entropy) - (math.log(2) + math.log(V)) / 2) < 1e-5
        assert torch.isfinite(x.grad).all() and not x.grad[0, 2:].any()


@pytest.mark.parametrize("V", [9, 50, 3000, 20000])
def test_categorical_masked_rows_are_not_looked_at(V):
    x = torch.randn(4, V, device=DEV)
    x[1], x[2] = math.nan, -math.inf
    x.requires_grad_(True)
    mask = torch.tensor([True, False, False, True], device=DEV)
    act = torch.tensor([0, -100, 1 << 40, V - 1], device=DEV)
    nan = torch.tensor([0.0, math.nan, math.inf, 0.0], device=DEV)
    one = nan + 1
    r = categorical_policy_loss(x, act, nan - 2, one, nan - 2, mask, kl_coef=0.1, entropy_coef=0.1)
    r.loss.backward()
    assert all(bool(torch.isfinite(t).all()) for t in (r.loss, r.logp, r.entropy, r.kl, x.grad))
    assert not x.grad[1:3].any() and bool(x.grad[0].any()) and not r.logp[1:3].any()
    # nothing counts: a loss of zero, with zero gradients
    x.grad = None
    r = categorical_policy_loss(x, act, nan, one, None, mask & False, entropy_coef=0.1)
    r.loss.backward()
    assert float(r.loss) == 0.0 and float(r.entropy) == 0.0 and not x.grad.any()


@pytest.mark.parametrize("V", [9, 50, 3000, 20000])
def test_categorical_what_is_wrong_shows(V):
    """NaN or +inf logits, a row with no open action, an action that does not exist: NaN."""
    z = torch.zeros(2, device=DEV)
    for kind in ("nan", "inf", "none", "low", "high"):
        x = torch.randn(2, V, device=DEV)
        act = torch.tensor([0, 1], device=DEV)
        if kind == "nan":
            x[1, V - 1] = math.nan
        elif kind == "inf":
            x[1, V // 2] = math.inf
        elif kind == "none":
            x[1] = -math.inf
        else:
            act[1] = -1 if kind == "low" else V
        x.requires_grad_(True)
        r = categorical_policy_loss(x, act, z - 2, z + 1)
        r.loss.backward()
        assert math.isnan(float(r.loss)) and math.isnan(float(r.logp[1])), kind
        assert torch.isfinite(x.grad[0]).all() and torch.isnan(x.grad[1]).all(), kind
        assert torch.isfinite(r.logp[0])


@pytest.mark.parametrize("V", [9, 300, 9000])
def test_upstream_gradients_and_repeated_backward(V):
    """Any upstream gradient, a second backward over the same graph, and gradients that are the
    caller's to change."""
    g, x, act = cat_case((20,), V, torch.float32, 5, False)
    z = torch.zeros(20, device=DEV)
    x.requires_grad_(True)

    def loss():
        return categorical_policy_loss(x, act, z - 2, z + 1, entropy_coef=0.1).loss
    base, = torch.autograd.grad(loss(), x)
    for up in (1.0, -2.5, 0.0):
        got, = torch.autograd.grad(loss() * up, x)
        assert torch.allclose(got, base * up, rtol=1e-5, atol=1e-9)
    r = loss()
    a, = torch.autograd.grad(r, x, retain_graph=True)
    a.zero_()
    b, = torch.autograd.grad(r, x)
    assert torch.equal(b, base)
    c, = torch.autograd.grad(loss() + loss(), x)
    assert torch.allclose(c, 2 * base, rtol=1e-6)
    total = loss()
    total /= 4  # in place on the loss itself
    assert torch.allclose(torch.autograd.grad(total, x)[0], base / 4, rtol=1e-5, atol=1e-9)
    y = x.detach().clone().requires_grad_(True)
    z2 = y * 1.0
    r = categorical_policy_loss(z2, act, z - 2, z + 1).loss
    with torch.no_grad():
        z2.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        r.backward()


@pytest.mark.parametrize("V", [5, 40, 2100, 8200])
def test_categorical_against_differences(V):
    g, x, act = cat_case((2,), V, torch.float64, 9, False)
    x64, lp, _ = cat_ref(x, act)
    old, adv, q, _ = rows_of(2, g, lp.detach(), False, True, torch.float64)
    x.requires_grad_(True)

    def f(y):
        return categorical_policy_loss(y, act, old, adv, q, kl_coef=0.2, entropy_coef=0.3).loss
    assert torch.autograd.gradcheck(f, (x,), fast_mode=V > 100)


def gauss_case(lead, D, dtype, shared, seed, mask, ref):
    g = gen(seed)
    mu = torch.randn(*lead, D, generator=g, device=DEV).to(dtype)
    ls = (torch.randn(*(() if shared else lead), D, generator=g, device=DEV) * 0.3 - 0.5).to(dtype)
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    act = (mu.double() + ls.double().exp() * torch.randn(*lead, D, generator=g, device=DEV,
                                                         dtype=torch.float64)).to(wide)
    h = [t.double().clone().requires_grad_(True) for t in (mu, ls)]
    z = (act.double() - h[0]) * torch.exp(-h[1])
    lp = (-0.5 * z * z - h[1] - 0.5 * math.log(2 * math.pi)).sum(-1)
    ent = (h[1] + 0.5 * math.log(2 * math.pi * math.e)).sum(-1).expand(lp.shape)
    old, adv, q, m = (None if t is None else t.view(lead) for t in
                      rows_of(math.prod(lead), g, lp.detach().reshape(-1), mask, ref, dtype))
    if m is not None:
        mu[~m] = math.nan
    return mu, ls, act, old, adv, q, m, lp, ent, h


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 8, 9, 17, 33, 64])
def test_gaussian(D, shared, dtype):
    lead = (3, 70) if D % 2 else (301,)
    mu, ls, act, old, adv, q, m, lp, ent, h = gauss_case(lead, D, dtype, shared, D, D % 3 == 1,
                                                         D % 4 == 1)
    check_loss(gaussian_policy_loss, [mu, ls], act, old, adv, q, m, lp, ent, h,
               float(lp.detach().abs().max()) + D, "mean", 0.1, 0.02)


@pytest.mark.parametrize("D", [2, 6])
def test_gaussian_many_rows(D):
    mu, ls, act, old, adv, q, m, lp, ent, h = gauss_case((600_001,), D, torch.float32, True, 1, True,
                                                         True)
    check_loss(gaussian_policy_loss, [mu, ls], act, old, adv, q, m, lp, ent, h,
               float(lp.detach().abs().max()) + D, "mean", 0.1, 0.02)


def test_gaussian_against_differences_and_broadcast():
    for D, shared in ((2, True), (3, False), (7, True)):
        mu, ls, act, old, adv, q, _, *_ = gauss_case((5,), D, torch.float64, shared, 3, False, True)
        mu.requires_grad_(True)
        ls.requires_grad_(True)
        assert torch.autograd.gradcheck(
            lambda a, b: gaussian_policy_loss(a, b, act, old, adv, q, kl_coef=0.2,
                                              entropy_coef=0.1).loss, (mu, ls))
    # one deviation per agent, shared by the envs: the gradient is summed over what it spans
    mu, ls, act, old, adv, *_ = gauss_case((4, 3), 2, torch.float64, False, 4, False, False)
    per_agent = ls[0].detach().clone().requires_grad_(True)
    got, = torch.autograd.grad(gaussian_policy_loss(mu, per_agent, act, old, adv).loss, per_agent)
    full = per_agent.detach().expand(4, 3, 2).contiguous().requires_grad_(True)
    want, = torch.autograd.grad(gaussian_policy_loss(mu, full, act, old, adv).loss, full)
    assert torch.allclose(got, want.sum(0), rtol=1e-12)


def test_losses_without_decisions():
    x = torch.zeros(0, 5, device=DEV, requires_grad=True)
    e = torch.zeros(0, device=DEV)
    r = categorical_policy_loss(x, e.long(), e, e)
    r.loss.backward()
    assert float(r.loss) == 0.0 and x.grad.shape == (0, 5)
    ls = torch.zeros(2, device=DEV, requires_grad=True)
    gaussian_policy_loss(torch.zeros(0, 2, device=DEV), ls, torch.zeros(0, 2, device=DEV), e,
                         e).loss.backward()
    assert torch.equal(ls.grad, torch.zeros(2, device=DEV))


def test_losses_refuse():
    x, z = torch.zeros(4, 6, device=DEV), torch.zeros(4, device=DEV)
    a = torch.zeros(4, dtype=torch.int64, device=DEV)
    with pytest.raises(TypeError, match="actions"):
        categorical_policy_loss(x, z, z, z)
    with pytest.raises(ValueError, match="actions"):
        categorical_policy_loss(x, a[:3], z, z)
    with pytest.raises(TypeError, match="old_logp"):
        categorical_policy_loss(x, a, z.double(), z)
    with pytest.raises(ValueError, match="advantages requires grad"):
        categorical_policy_loss(x, a, z, z.clone().requires_grad_(True))
    with pytest.raises(TypeError, match="mask"):
        categorical_policy_loss(x, a, z, z, None, z)
    with pytest.raises(ValueError, match="clip"):
        categorical_policy_loss(x, a, z, z, clip=(1.5, 0.2))
    with pytest.raises(ValueError, match="reduction"):
        categorical_policy_loss(x, a, z, z, reduction="none")
    with pytest.raises(ValueError, match="finite"):
        categorical_policy_loss(x, a, z, z, kl_coef=math.nan)
    with pytest.raises(TypeError, match="logits"):
        categorical_policy_loss(x.long(), a, z, z)
    with pytest.raises(ValueError, match="64"):
        gaussian_policy_loss(torch.zeros(4, 65, device=DEV), z, torch.zeros(4, 65, device=DEV), z, z)
    with pytest.raises(TypeError, match="log_std"):
        gaussian_policy_loss(x, torch.zeros(6, device=DEV).half(), x, z, z)
    with pytest.raises(ValueError, match="broadcast"):
        gaussian_policy_loss(x, torch.zeros(5, device=DEV), x, z, z)
    with pytest.raises(ValueError, match="is on"):
        categorical_policy_loss(x, a.cpu(), z, z)


# -------------------------------------------------------------------------------------- AdamW

SIZES = [1, 3, 255, 256, 257, 4096, 5003, 0]


def adamw_case(dtype, gdtype, seed, sizes=SIZES, shift=0):
    g = gen(seed)

    def made(n, d, s):
        return (torch.randn(n + shift, generator=g, device=DEV) * s).to(d)[shift:]
    return [made(n, dtype, 0.1) for n in sizes], [made(n, gdtype, 0.01) for n in sizes]


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype,gdtype,master", [
    (torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, True),
    (torch.bfloat16, torch.float32, True), (torch.float16, torch.float16, True)])
def test_adamw_against_the_definition(dtype, gdtype, master, shift):
    """Five steps, odd sizes, tensors that start off a 16-byte boundary, a clipped norm."""
    params, _ = adamw_case(dtype, gdtype, 1, shift=shift)
    state = adamw_state(params, master=master)
    w = [p.double() for p in params]
    m, v = ([torch.zeros_like(x) for x in w] for _ in range(2))
    for t in range(1, 6):
        _, grads = adamw_case(dtype, gdtype, 10 + t, shift=shift)
        norm = adamw_step(params, grads, state, t, lr=1e-2, betas=(0.9, 0.95), eps=1e-6,
                          weight_decay=0.1, max_grad_norm=0.5)
        true = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        assert abs(float(norm) - true) <= 1e-6 * true
        for k, g in enumerate(grads):
            g = g.double() * min(1.0, 0.5 / (true + 1e-6))
            m[k] = 0.9 * m[k] + 0.1 * g
            v[k] = 0.95 * v[k] + 0.05 * g * g
            w[k] = w[k] * (1 - 1e-3) - 1e-2 * (m[k] / (1 - 0.9 ** t)) / (
                torch.sqrt(v[k] / (1 - 0.95 ** t)) + 1e-6)
    # each step rounds the parameter and an update of up to 1e-2 a few times
    for p, x in zip(params, w):
        tol = 5 * 8 * EPS[torch.float32] + EPS[dtype] * x.abs() * (dtype != torch.float32) * 1.01
        assert bool(((p.double() - x).abs() <= tol + 2.0 ** -25).all())
    gm, gv = state.moments()
    at = 0
    for x, y in zip(m, v):
        n = x.numel()
        close("m", gm[at:at + n], x, 40 * EPS[torch.float32] * 0.05)
        close("v", gv[at:at + n], y, 40 * EPS[torch.float32] * 0.003)
        end = at + -(-n // 256) * 256
        assert not gm[at + n:end].any() and not gv[at + n:end].any()
        at = end


def code_values(x, signed):
    """The floats a moment's neighbours in 8 bits are: (below, above) in magnitude, per group."""
    mag = x.abs().view(-1, 256)
    bits = mag.contiguous().view(torch.int32)
    reach = 15 if signed else 31
    e = (bits.amax(-1, keepdim=True) + 0xfffff >> 23) - reach
    low = e.clamp(min=0) << 3
    k = bits >> 20
    down = torch.where(k > low, k, low)
    as_float = (down << 20).view(torch.float32), ((down + 1) << 20).view(torch.float32)
    floor = torch.where(k > low, as_float[0], torch.zeros_like(mag))
    return floor.view(-1), as_float[1].view(-1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adamw_8_bit_moments_are_neighbours_of_the_exact(dtype):
    params, _ = adamw_case(dtype, dtype, 1)
    state = adamw_state(params, bits=8)
    for t in range(1, 5):
        _, grads = adamw_case(dtype, dtype, 10 + t)
        m0, v0 = (x.clone() for x in state.moments())
        before = [p.clone() for p in params]
        adamw_step(params, grads, state, t, lr=1e-2, betas=(0.9, 0.95), seed=t)
        m1, v1 = state.moments()
        at = 0
        for k, g in enumerate(grads):
            n, pad = g.numel(), -(-g.numel() // 256) * 256
            x = torch.zeros(2, pad, device=DEV)
            b = [torch.tensor(c, dtype=torch.float32) for c in (0.9, 1 - 0.9, 0.95, 1 - 0.95)]
            x[0, :n] = m0[at:at + n] * b[0].item() + g.float() * b[1].item()
            x[1, :n] = v0[at:at + n] * b[2].item() + g.float() * g.float() * b[3].item()
            for want, got, signed in ((x[0], m1, True), (x[1], v1, False)):
                if not n:
                    continue
                lo, hi = code_values(want, signed)
                y = got[at:at + pad]
                assert bool(((y.abs() >= lo) & (y.abs() <= hi)).all())
                assert bool((torch.sign(y) * torch.sign(want) >= 0).all())
            assert bool((m1[at + n:at + pad] == 0).all()) and bool((v1[at + n:at + pad] == 0).all())
            assert bool((v1[at:at + n][x[1, :n] > 0] > 0).all())
            # the update is of the moments before they are rounded
            upd = 1e-2 * (x[0, :n].double() / (1 - 0.9 ** t)) / (
                (x[1, :n].double() / (1 - 0.95 ** t)).sqrt() + 1e-8)
            want = before[k].double() * (1 - 1e-4) - upd
            step = 2 * EPS[dtype] * want.abs() if dtype == torch.bfloat16 else 0.0
            assert bool(((params[k].double() - want).abs() <= step + 8 * EPS[torch.float32]).all())
            at += pad


def test_adamw_rounding_at_random_keeps_the_mean():
    """A constant gradient for 300 steps: the mean second moment follows its exact course, which
    rounding to nearest would stop at once.  Its spread: a step's rounding has a deviation of at
    most half a code's step (v / 16), steps are independent, and beta2 forgets none of 300 --
    at most v / 16 sqrt(300) an element, over 65536 elements 0.0043 v; five of those."""
    n = 65536
    p, g = [torch.zeros(n, device=DEV)], [torch.full((n,), 0.5, device=DEV)]
    state = adamw_state(p, bits=8)
    for t in range(1, 301):
        adamw_step(p, g, state, t, lr=0.0, seed=977 * t)
    m, v = state.moments()
    exact = 0.25 * (1 - 0.999 ** 300)
    assert abs(float(v.double().mean()) - exact) <= 5 * 0.0043 * exact
    assert abs(float(m.double().mean()) - 0.5 * (1 - 0.9 ** 300)) <= 5 * 0.0043 * 0.5
    assert int(torch.unique(v).numel()) > 2


def test_adamw_bfloat16_without_a_master_moves_on_average():
    """Updates of a sixteenth of a step: nearest rounding would lose every one."""
    n = 65536
    p, g = [torch.ones(n, device=DEV, dtype=torch.bfloat16)], [torch.ones(n, device=DEV, dtype=torch.bfloat16)]
    state = adamw_state(p)
    for t in range(1, 17):
        adamw_step(p, g, state, t, lr=2.0 ** -12, weight_decay=0.0, seed=t)
    # 16 steps of 2^-12 down from 1, in units of 2^-8 (2^-9 below 1): deviation of the mean below
    # sqrt(16) 2^-9 / sqrt(n); five of those, and the updates' own rounding
    assert abs(float(p[0].double().mean()) - (1 - 16 * 2.0 ** -12)) <= 5 * 4 * 2.0 ** -9 / 256 + 1e-6


def test_adamw_skips_what_has_no_gradient_and_takes_many_tensors():
    p = [torch.ones(5, device=DEV) for _ in range(150)]
    g = [torch.ones(5, device=DEV) if k % 3 else None for k in range(150)]
    state = adamw_state(p)
    adamw_step(p, g, state, 1, lr=0.1, weight_decay=0.0)
    for k in range(150):
        assert float(p[k][0]) == (1.0 if k % 3 == 0 else pytest.approx(0.9, abs=1e-6))
    mixed = [torch.ones(300, device=DEV), torch.ones(300, device=DEV, dtype=torch.bfloat16)]
    state = adamw_state(mixed, master=True)
    adamw_step(mixed, [torch.ones_like(x) for x in mixed], state, 1, lr=0.1, weight_decay=0.0)
    assert float(mixed[0][7]) == pytest.approx(0.9, abs=1e-6)
    assert float(mixed[1][7]) == float(torch.tensor(0.9).bfloat16())


def test_adamw_non_finite_gradients_stay_visible():
    for bits in (32, 8):
        p, g = [torch.ones(600, device=DEV)], [torch.ones(600, device=DEV)]
        g[0][300] = math.nan
        g[0][10] = math.inf
        state = adamw_state(p, bits=bits)
        adamw_step(p, g, state, 1)
        m, v = state.moments()
        assert not torch.isfinite(p[0][[10, 300]]).any() and not torch.isfinite(m[[10, 300]]).any()
        assert torch.isfinite(p[0][[11, 299, 599]]).all() and torch.isfinite(m[512:600]).all()


def test_grad_norm():
    g = [torch.randn(n, generator=gen(n), device=DEV).to(d) for n in (1, 777, 300_001)
         for d in (torch.float32, torch.bfloat16, torch.float16)]
    true = math.sqrt(sum(float(x.double().square().sum()) for x in g))
    norm, scale = grad_norm(g, 2.0)
    assert abs(float(norm) - true) <= 1e-6 * true
    assert abs(float(scale) - 2.0 / (true + 1e-6)) <= 1e-6
    assert float(grad_norm(g)[1]) == 1.0
    again = grad_norm(g, 2.0)
    assert torch.equal(norm, again[0])
    assert float(grad_norm([torch.zeros(4, device=DEV), None])[0]) == 0.0


def test_adamw_optimizer_and_its_state():
    torch.manual_seed(0)
    x, y = torch.randn(256, 8, device=DEV), torch.randn(256, 1, device=DEV)

    def net():
        torch.manual_seed(1)
        return torch.nn.Sequential(torch.nn.Linear(8, 32), torch.nn.Tanh(),
                                   torch.nn.Linear(32, 1)).to(DEV)

    def go(model, opt, steps):
        for _ in range(steps):
            opt.zero_grad()
            ((model(x) - y) ** 2).mean().backward()
            opt.step()
    ours, theirs = net(), net()
    groups = [{"params": ours[0].parameters()}, {"params": ours[2].parameters(), "lr": 3e-3}]
    opt = AdamW(groups, lr=1e-2, weight_decay=0.05)
    ref = torch.optim.AdamW([{"params": theirs[0].parameters()},
                             {"params": theirs[2].parameters(), "lr": 3e-3}], lr=1e-2,
                            weight_decay=0.05, foreach=False)
    sched = torch.optim.lr_scheduler.StepLR(opt, 5, 0.5)
    sched_ref = torch.optim.lr_scheduler.StepLR(ref, 5, 0.5)
    for _ in range(3):
        go(ours, opt, 5)
        go(theirs, ref, 5)
        sched.step()
        sched_ref.step()
    for a, b in zip(ours.parameters(), theirs.parameters()):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-6)
    # a second optimizer goes on where the first left off, bit for bit, 8-bit moments too
    for bits in (32, 8):
        a, b = net(), net()
        one = AdamW(a.parameters(), bits=bits, max_grad_norm=0.1, seed=5)
        go(a, one, 3)
        b.load_state_dict(a.state_dict())
        two = AdamW(b.parameters(), bits=bits, max_grad_norm=0.1)
        two.load_state_dict(one.state_dict())
        go(a, one, 3)
        go(b, two, 3)
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    with pytest.raises(ValueError, match="bits"):
        AdamW(a.parameters(), bits=32).load_state_dict(one.state_dict())


def test_adamw_is_seen_by_autograd():
    w, idle = (torch.ones(300, device=DEV, requires_grad=True) for _ in range(2))
    loss = (w * w * idle).sum()
    before = idle._version
    adamw_step([w, idle], [torch.ones_like(w), None], adamw_state([w, idle]), 1)
    assert idle._version == before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_adamw_optimizer_is_copied_whole():
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    one = AdamW([p], bits=8, max_grad_norm=1.0, seed=3)
    p.grad = torch.linspace(-1, 1, 300, device=DEV)
    one.step()
    two = copy.deepcopy(one)
    q = two.param_groups[0]["params"][0]
    q.grad = p.grad.clone()
    one.step()
    two.step()
    assert q is not p and torch.equal(p, q)
    assert torch.equal(one.last_grad_norm, two.last_grad_norm)
    for a, b in zip(one._states[0][:4], two._states[0][:4]):
        assert torch.equal(a, b)


def test_adamw_refuses():
    p, g = [torch.zeros(4, device=DEV)], [torch.zeros(4, device=DEV)]
    s = adamw_state(p)
    with pytest.raises(ValueError, match="gradients"):
        adamw_step(p, [], s, 1)
    with pytest.raises(ValueError, match="step"):
        adamw_step(p, g, s, 0)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([p[0], p[0].view(2, 2)], [g[0], g[0].view(2, 2)], adamw_state(p + p), 1)
    with pytest.raises(ValueError, match="betas"):
        adamw_step(p, g, s, 1, betas=(1.0, 0.9))
    with pytest.raises(TypeError, match="parameter 0"):
        adamw_step([p[0].double()], [g[0].double()], s, 1)
    with pytest.raises(TypeError, match="gradient 0"):
        adamw_step(p, [g[0].bfloat16()], s, 1)
    with pytest.raises(ValueError, match="gradient 0"):
        adamw_step(p, [g[0][:3]], s, 1)
    with pytest.raises(ValueError, match="contiguous"):
        adamw_step([torch.zeros(4, 2, device=DEV)[:, 0]], g, s, 1)
    with pytest.raises(ValueError, match="elements"):
        adamw_step([torch.zeros(300, device=DEV)], [torch.zeros(300, device=DEV)], s, 1)
    with pytest.raises(ValueError, match="master"):
        adamw_step([p[0].half()], [g[0].half()], s, 1)
    with pytest.raises(ValueError, match="exp_avg_sq"):
        adamw_step(p, g, AdamWState(s.exp_avg, s.exp_avg_sq[:10]), 1)
    with pytest.raises(ValueError, match="not both"):
        adamw_step(p, g, s, 1, max_grad_norm=1.0, grad_scale=torch.ones((), device=DEV))
    with pytest.raises(ValueError, match="norm"):
        grad_norm(g, 0.0)
    with pytest.raises(ValueError, match="bits"):
        adamw_state(p, bits=16)


# ------------------------------------------------------------------- streams, graphs, together


def test_on_another_stream_and_in_a_graph():
    """The operators run where torch's current stream is; captured, their replays give what eager
    calls give, with eager work between the replays."""
    g, x, act = cat_case((300,), 50, torch.float32, 3, False)
    z = torch.randn(300, generator=g, device=DEV)
    mask = torch.rand(300, generator=g, device=DEV) < 0.5
    r, v = torch.randn(40, 300, generator=g, device=DEV), torch.randn(41, 300, generator=g, device=DEV)
    x.requires_grad_(True)

    def work():
        adv = gae(r, v).advantages[0].contiguous()
        loss = categorical_policy_loss(x, act, z - 3, adv, None, mask, entropy_coef=0.1).loss
        return adv, loss, torch.autograd.grad(loss, x)[0]
    want = [t.detach().clone() for t in work()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = work()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        work()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            out = work()
    torch.cuda.synchronize()
    for k in range(4):
        with torch.no_grad():
            x.add_(0.25 * (-1) ** k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, work()))
        torch.cuda.synchronize()


@pytest.mark.parametrize("head,bits", [("gaussian", 32), ("categorical", 8)])
def test_example_trains(head, bits):
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "train_navigation.py"
    spec = importlib.util.spec_from_file_location("train_navigation", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    said = []
    rewards = mod.train(head, bits, n_envs=256, n_agents=3, steps=16, iterations=11,
                        log=said.append)
    assert len(rewards) == 11 and all(math.isfinite(x) for x in rewards)
    first, last = (float(line.split("entropy ")[1].split()[0]) for line in said)
    assert last < first and "nan" not in "".join(said)  # the policy has made up its mind a little
