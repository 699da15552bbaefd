"""linear_cross_entropy on the GPU against the definition in float64.

Tolerances.  With u the type's half step (finfo.eps / 2) and every product and sum in float32:
a logit is a sum of D products (and a bias), off by at most (D + 2) 2^-24 of the sum of their
magnitudes, `dz`; an exponential of a difference of two logits, relative to a sum of V of them by a
tree, is then off by 2 dz + 32 2^-24 of itself at most (the hardware's exp2 and log2 and what leads to
them cost a few 2^-24 each, the argument's rounding 2^-24 times its magnitude, below 2^6 here).  A
gradient is a sum of such weights times h or W: its magnitudes' sum times that error, times u for
the weight's rounding to the type, and n 2^-24 for adding n terms; and u of itself, for the end."""

import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from swarp_amd import categorical_policy_loss, linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F24 = 2.0 ** -24


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def inputs(rows, D, V, dtype, seed, bias=True, mask=0.0, spread=2.0):
    g = gen(seed)
    h = torch.randn(rows, D, generator=g, device=DEV).to(dtype)
    w = (torch.randn(V, D, generator=g, device=DEV) * spread / math.sqrt(D)).to(dtype)
    b = (torch.randn(V, generator=g, device=DEV) * 0.5).to(dtype) if bias else None
    t = torch.randint(0, V, (rows,), generator=g, device=DEV)
    m = torch.rand(rows, generator=g, device=DEV) >= mask if mask else None
    return h, w, t, b, m


def half(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def reference(h, w, t, b, m, up=1.0, reduction="mean"):
    """Values in float64, and how far a right answer may be off: {name: (value, tolerance)}."""
    rows, D = h.shape
    V = w.shape[0]
    u = half(h.dtype)
    on = torch.ones(rows, dtype=torch.bool, device=DEV) if m is None else m
    hd = torch.where(on[:, None], h.double(), 0.0)
    wd = w.double()
    z = hd @ wd.t() + (0.0 if b is None else b.double())
    dz = (D + 2) * F24 * (hd.abs() @ wd.abs().t() + (0.0 if b is None else torch.nan_to_num(b.double(), neginf=0.0).abs())).amax(-1, keepdim=True)
    lse = torch.logsumexp(z, -1, keepdim=True)
    at = torch.where(on, t.long(), 0)[:, None]
    logp = torch.where(on, (z.gather(-1, at) - lse)[:, 0], 0.0)
    n = int(on.sum()) if reduction == "mean" else 1
    weight = on.double()[:, None] * up / max(n, 1)
    p = torch.exp(z - lse)
    one = torch.zeros_like(p).scatter_(-1, at, 1.0)
    G, err = (p - one) * weight, 2 * dz + 32 * F24
    err = err + F24 * torch.nan_to_num(z - lse, neginf=0.0).abs().amax(-1, keepdim=True)
    mag = (p + one) * weight.abs()
    dlogp = (2 * dz + 32 * F24)[:, 0] + 4 * F24 * logp.abs()
    out = {"logp": (logp, dlogp)}
    out["loss"] = (-logp.sum() / max(n, 1), (dlogp * on).sum() / max(n, 1) + 2 * F24 * logp.abs().sum() / max(n, 1))
    least = torch.finfo(h.dtype).tiny  # (below it a type has fewer digits)

    def tol(value, m_err, magnitude, terms, roundings):
        return m_err + magnitude * (roundings * u * 1.01 + terms * F24) + (u + 4 * F24) * value.abs() + least
    dh = G @ wd
    out["hidden"] = (dh, tol(dh, (mag * err) @ wd.abs(), mag @ wd.abs(), V, 1))
    dw = G.t() @ hd
    out["weight"] = (dw, tol(dw, (mag * err).t() @ hd.abs(), mag.t() @ hd.abs(), rows, 1))
    db = G.sum(0)
    out["bias"] = (db, tol(db, (mag * err).sum(0), mag.sum(0), rows, 1))
    return out


def close(got, want, what):
    value, tol = want
    assert got.shape == value.shape, what
    err = (got.double() - value).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err - tol).max())} above, error {float(err.max())}"


def run(h, w, t, b, m, up=1.0, reduction="mean"):
    leaves = [x.detach().clone().requires_grad_(True) for x in (h, w, b) if x is not None]
    r = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2] if b is not None else None, m, reduction=reduction)
    (r.loss * up).backward()
    got = {"loss": r.loss.detach(), "logp": r.logp, "hidden": leaves[0].grad, "weight": leaves[1].grad}
    if b is not None:
        got["bias"] = leaves[2].grad
    return got


SHAPES = [(1, 1, 1), (1, 16, 2), (3, 5, 7), (32, 64, 31), (33, 32, 256), (64, 100, 257), (257, 33, 300),
          (300, 64, 25), (2560, 64, 9), (1000, 7, 40), (129, 256, 1000), (520, 96, 4099), (16, 520, 9001),
          (4100, 40, 130), (96, 128, 20000), (300, 129, 33), (601, 200, 22), (2100, 520, 9), (77, 65, 64),
          (70, 1261, 65)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,V", SHAPES)
def test_against_float64(rows, D, V, dtype):
    for k, (bias, mask) in enumerate([(True, 0.0), (False, 0.3)]):
        h, w, t, b, m = inputs(rows, D, V, dtype, rows + V + k, bias, mask)
        up = 1024.0 if dtype == torch.float16 else 1.0
        if m is not None:
            h = torch.where(m[:, None], h, math.nan)
            t = torch.where(m, t, -100)
        want = reference(h, w, t, b, m, up)
        got = run(h, w, t, b, m, up)
        for name in got:
            close(got[name], want[name], f"{rows}x{D}x{V} {dtype} {name}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_logp_alone_sums_and_integers(dtype):
    h, w, t, b, m = inputs(333, 70, 1234, dtype, 5, True, 0.4)
    want = reference(h, w, t, b, m, reduction="sum")
    with torch.no_grad():
        r = linear_cross_entropy(h, w, t.int(), b, m, reduction="sum")
    close(r.loss, want["loss"], "loss")
    close(r.logp, want["logp"], "logp")
    assert not r.loss.requires_grad
    got = run(h, w, t.int(), b, m, 8.0 if dtype == torch.float16 else 1.0, "sum")
    want = reference(h, w, t, b, m, 8.0 if dtype == torch.float16 else 1.0, "sum")
    for name in got:
        close(got[name], want[name], name)


def test_logp_feeds_the_policy_loss():
    """A behaviour-cloned head's log-probabilities as the policy loss's old and reference ones."""
    h, w, t, b, _ = inputs(200, 32, 500, torch.bfloat16, 3)
    with torch.no_grad():
        ref = linear_cross_entropy(h, w, t, b).logp
    logits = (h.float() @ w.float().t() + b.float()).requires_grad_(True)
    pg = categorical_policy_loss(logits, t, ref, torch.ones_like(ref), ref, kl_coef=0.1)
    assert abs(float(pg.loss) + 1.0) < 1e-3 and float(pg.kl) < 1e-6 and float(pg.clip_fraction) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masked_decisions_are_not_looked_at(dtype):
    h, w, t, b, _ = inputs(700, 48, 600, dtype, 9)
    m = torch.zeros(700, dtype=torch.bool, device=DEV)
    m[5:80] = m[300:301] = m[699:] = True
    clean = run(h, w, t, b, m)
    h2 = torch.where(m[:, None], h, math.nan)
    h2[~m, 0] = math.inf
    t2 = torch.where(m, t, 1 << 40)
    dirty = run(h2, w, t2, b, m)
    for name in clean:
        assert torch.equal(clean[name], dirty[name]), name
    assert not clean["hidden"][~m].any() and not clean["logp"][~m].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [0, 5, 300])
def test_nothing_counts(rows, dtype):
    h, w, t, b, _ = inputs(rows, 24, 50, dtype, 1)
    for m in ([torch.zeros(rows, dtype=torch.bool, device=DEV)] + ([None] if rows == 0 else [])):
        got = run(h, w, t, b, m)
        for name in got:
            assert not got[name].any() and got[name].isfinite().all(), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_closed_actions_and_far_targets(dtype):
    """Biases of -inf; targets so unlikely that the exponentials start from elsewhere."""
    h, w, t, b, _ = inputs(100, 16, 90, dtype, 2)
    b[10:40] = -math.inf
    t = torch.where((t >= 10) & (t < 40), 3, t)
    want = reference(h, w, t, b, None, 64.0)
    got = run(h, w, t, b, None, 64.0)
    for name in ("logp", "loss", "hidden", "weight"):
        close(got[name], (torch.nan_to_num(want[name][0]), want[name][1]), name)
    assert not got["bias"][10:40].any()
    b = b.clone()
    b[3] = -400.0  # exp(-400) is nothing beside the others: a second pass
    want = reference(h, w, t, b, None, 64.0)
    got = run(h, w, t, b, None, 64.0)
    for name in ("logp", "loss", "hidden", "weight"):
        close(got[name], want[name], name)
    b[3] = -math.inf  # a target that is closed: no probability, and a gradient all the same
    got = run(h, w, t, b, None, 64.0)
    assert float(got["loss"]) == math.inf and bool((got["logp"][t == 3] == -math.inf).all())
    want = reference(h, w, t, b, None, 64.0)
    close(got["hidden"], want["hidden"], "hidden")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,V", [(3, 583, 3), (3, 64, 3), (400, 130, 2), (4000, 40, 100)])
def test_the_bias_gradient_is_summed_before_it_is_rounded(rows, D, V, dtype):
    """Its terms cancel: their rounding to the type would be most of it.  Only the logits' own error and
    the end's rounding are left, so the type's half step counts once, relative to the sum."""
    h, w, t, b, m = inputs(rows, D, V, dtype, rows + V)
    up = 1024.0 if dtype == torch.float16 else 1.0
    value, tol = reference(h, w, t, b, m, up)["bias"]
    p = torch.softmax(h.double() @ w.double().t() + b.double(), -1)
    mag = (p + torch.nn.functional.one_hot(t, V)).sum(0) * up / rows
    # (24 bits of an exponential are kept: 2^-17 of a half step, where the tolerance above has u)
    tol = tol - mag * (1.01 * half(dtype) - 2.0 ** -16)
    close(run(h, w, t, b, m, up)["bias"], (value, tol), "bias")


@pytest.mark.parametrize("rows,D,V", [(1, 64, 9), (200, 64, 25), (300, 30, 60), (70, 128, 31), (33, 9, 40), (4000, 64, 64)])
def test_gradients_of_narrow_bfloat16_heads_are_rounded_once(rows, D, V):
    """What a target's probability lacks of 1 and the others' go into the products with 16 bits: a 2^-16 of
    them where the tolerance of wide heads has a half step of the type."""
    h, w, t, b, m = inputs(rows, D, V, torch.bfloat16, rows + V, mask=0.2 if rows > 1 else 0.0)
    want, got = reference(h, w, t, b, m), run(h, w, t, b, m)
    on = torch.ones(rows, dtype=torch.bool, device=DEV) if m is None else m
    p = torch.softmax(h.double() @ w.double().t() + b.double(), -1)
    mag = (p + torch.nn.functional.one_hot(t, V)) * on[:, None] / int(on.sum())
    less = 1.01 * half(torch.bfloat16) - 2.0 ** -16
    for name, of in (("hidden", mag @ w.double().abs()), ("weight", mag.t() @ h.double().abs())):
        value, tol = want[name]
        close(got[name], (value, tol - less * of), name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D,V", [(40, 64, 25), (300, 64, 300), (20, 64, 300)])
def test_a_row_of_the_lowest_biases(rows, D, V, dtype):
    """Beside the type's lowest value a logit vanishes: every action is as likely as another."""
    h, w, t = inputs(rows, D, V, dtype, 21)[:3]
    b = torch.full((V,), torch.finfo(dtype).min, dtype=dtype, device=DEV)
    got = run(h, w, t, b, None)
    # (hardware's exp2 and log2 and the sum's tree: the 32 2^-24 of the others)
    assert float((got["logp"].double() + math.log(V)).abs().max()) <= (32 + 4 * math.log(V)) * F24
    G = (1.0 / V - torch.nn.functional.one_hot(t, V).double()) / rows
    mag, u = (1.0 / V + torch.nn.functional.one_hot(t, V).double()) / rows, half(dtype)

    def tol(m, value, terms):
        return m * (1.01 * u + (32 + terms) * F24) + (u + 4 * F24) * value.abs()
    hd, wd = h.double(), w.double()
    close(got["hidden"], (G @ wd, tol(mag @ wd.abs(), G @ wd, V)), "hidden")
    close(got["weight"], (G.t() @ hd, tol(mag.t() @ hd.abs(), G.t() @ hd, rows)), "weight")
    close(got["bias"], (G.sum(0), tol(mag.sum(0), G.sum(0), rows)), "bias")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("what", ["nan", "inf", "closed", "target", "below"])
def test_what_is_wrong_shows(what, dtype):
    h, w, t, b, _ = inputs(70, 16, 300, dtype, 4)
    if what == "nan":
        h[7, 3] = math.nan
    elif what == "inf":
        b[2] = math.inf
    elif what == "closed":
        b[:] = -math.inf
    else:
        t[7] = 300 if what == "target" else -1
    got = run(h, w, t, b, None)
    assert got["loss"].isnan() and got["logp"][7].isnan()
    assert got["hidden"][7].isnan().any() and got["weight"].isnan().any()
    with torch.no_grad():
        assert linear_cross_entropy(h, w, t, b).loss.isnan()
    if what in ("nan", "target", "below"):  # the other decisions are none the worse
        assert bool(got["logp"][torch.arange(70, device=DEV) != 7].isfinite().all())
        m = torch.ones(70, dtype=torch.bool, device=DEV)
        m[7] = False
        got = run(h, w, t, b, m)
        assert all(bool(x.isfinite().all()) for x in got.values())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,V", [(16, 300), (400, 300), (16, 25), (200, 20)])
def test_a_target_that_is_none_shows_beside_a_far_one(D, V, dtype):
    """A row whose target is e^-400 sends its neighbours through a second pass."""
    h, w, t, b, _ = inputs(70, D, V, dtype, 22)
    t = torch.where(t == 5, 6, t)
    t[3], t[7], b[5] = 5, V, -400.0
    got = run(h, w, t, b, None)
    assert got["loss"].isnan() and got["logp"][7].isnan()
    assert got["hidden"][7].isnan().all() and got["weight"].isnan().all() and got["bias"].isnan().all()
    rest = torch.arange(70, device=DEV) != 7
    assert got["logp"][rest].isfinite().all() and got["hidden"][rest].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,V", [(64, 1024, 1000), (20, 1024, 1000), (300, 1261, 60), (16500, 520, 40), (200, 64, 25)])
def test_confident_decisions(rows, D, V, dtype):
    """Where the target's probability is almost 1, 1 - p and log p are what the others leave, and no
    difference of two roundings of the target's logit.  q = 1 - p is off by the others' relative error, and by
    what adding terms to a sum near 1 loses: no more than they are, and 2^-24 an addition, of which a
    logit passes V / 32 + 64 at most; and by 8 2^-24 for quotient, logarithm and the like."""
    h, w, t, b, _ = inputs(rows, D, V, dtype, rows + V)
    scale = torch.linspace(6.0, 30.0, rows, device=DEV)[:, None] / w[t].float().square().sum(-1, keepdim=True)
    h = (w[t].float() * scale + 0.1 * h.float()).to(dtype)
    # (float16: neither beyond its largest, summed over the rows, nor below its smallest)
    up, u, kinds = (2.0 ** 14 * min(1.0, 256 / rows) if dtype == torch.float16 else 1.0), half(dtype), (h, w, t, b, None)
    hd, wd = h.double(), w.double()
    z = hd @ wd.t() + b.double()
    dz = (D + 2) * F24 * (hd.abs() @ wd.abs().t() + b.double().abs()).amax(-1, keepdim=True)
    lse = torch.logsumexp(z, -1, keepdim=True)
    one = torch.nn.functional.one_hot(t, V).double()
    p = torch.exp(z - lse) * (1 - one)  # of the others
    q = p.sum(-1, keepdim=True)
    assert float(q.median()) < 1e-4
    relative = 2 * dz + 32 * F24 + 2 * F24 * (z - lse).abs().amax(-1, keepdim=True)
    dq = q * relative + torch.minimum(q, torch.tensor((V / 32 + 64) * F24)) + 8 * F24
    logp = torch.log1p(-q)
    with torch.no_grad():
        alone = linear_cross_entropy(h, w, t, b, reduction="sum")
    got = run(*kinds, up, "sum")
    for y in (alone.logp, got["logp"]):
        assert bool((y <= 0).all()), float(y.max())
        close(y, (logp[:, 0], (2 * dq + 4 * F24 * logp.abs())[:, 0]), "logp")
    G, err = (p - one * q) * up, (p * relative + one * dq) * up
    mag = G.abs()
    least = 2.0 ** -39 * up if dtype == torch.float16 else 0.0  # (float16's smallest, over what G is kept times)
    rounding = 1.02 * u + V * F24
    dh, db = G @ wd, G.sum(0)
    tiny = torch.finfo(dtype).tiny
    close(got["hidden"], (dh, (err + mag * rounding + least) @ wd.abs() + (u + 4 * F24) * dh.abs() + tiny), "hidden")
    dw = G.t() @ hd
    close(got["weight"], (dw, (err + mag * (1.02 * u + rows * F24) + least).t() @ hd.abs() + (u + 4 * F24) * dw.abs() + tiny), "weight")
    # (24 bits of an exponential are kept: 2^-17 of half a step)
    close(got["bias"], (db, (err + mag * (2.0 ** -16 + rows * F24)).sum(0) + (u + 4 * F24) * db.abs() + tiny), "bias")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_over_leading_axes(dtype):
    g = gen(0)
    base = torch.randn(3, 21, 2, 40, generator=g, device=DEV).to(dtype)
    w = torch.randn(55, 40, generator=g, device=DEV).to(dtype) * 0.3
    for x in (base[:, :-1], base[:, :, 0], base.permute(2, 0, 1, 3), base[:, ::2, :, 3:30], base[0, 0, 0], base[..., ::2]):
        t = torch.randint(0, 55, x.shape[:-1], generator=g, device=DEV)
        W = w[:, :x.shape[-1]]
        a = x.detach().requires_grad_(True)
        c = x.detach().contiguous().requires_grad_(True)
        r, s = linear_cross_entropy(a, W, t), linear_cross_entropy(c, W.contiguous(), t)
        r.loss.backward()
        s.loss.backward()
        assert torch.equal(r.loss, s.loss) and torch.equal(r.logp, s.logp) and torch.equal(a.grad, c.grad)


def test_more_rows_than_a_piece_holds():
    """2^21 logits a row: 1 GiB holds 256 of 16 bits."""
    V = 1 << 21
    h, w, t, _, m = inputs(300, 4, V, torch.bfloat16, 8, False, 0.1, spread=1.0)
    got = run(h, w, t, None, m)
    # the definition, a few rows at a time (tolerances as above)
    on = m.nonzero()[:, 0]
    n, dw, mag, logp = len(on), torch.zeros(V, 4, dtype=torch.float64, device=DEV), torch.zeros(V, 4, dtype=torch.float64, device=DEV), []
    for part in on.split(50):
        z = h[part].double() @ w.double().t()
        p = torch.softmax(z, -1)
        logp.append(torch.log_softmax(z, -1).gather(-1, t[part][:, None])[:, 0])
        one = torch.zeros_like(p).scatter_(-1, t[part][:, None], 1.0)
        dw += (p - one).t() @ h[part].double() / n
        mag += (p + one).t() @ h[part].double().abs() / n
        dh = (p - one) @ w.double() / n
        dh_mag = (p + one) @ w.double().abs() / n
        close(got["hidden"][part], (dh, dh_mag * (2.0 ** -8 * 1.01 + 1e-5) + 2.0 ** -8 * dh.abs() + 1e-30), "hidden")
    logp = torch.cat(logp)
    close(got["logp"][on], (logp, torch.full_like(logp, 1e-5)), "logp")
    close(got["weight"], (dw, mag * (2 * 2.0 ** -8 * 1.01 + 1e-5) + 2.0 ** -8 * dw.abs() + 1e-30), "weight")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("far", [5, 600])
def test_one_piece_of_several_starts_from_elsewhere(dtype, far):
    """2^20 logits a row: 512 rows a piece of 16 bits, 256 of float32.  One row's target is e^-400."""
    V, rows = 1 << 20, 601
    h, w, t, b, _ = inputs(rows, 4, V, dtype, 9, spread=1.0)
    t = torch.where(t == 77, 78, t)
    t[far] = 77
    b[77] = -400.0
    got = run(h, w, t, b, None, reduction="sum")
    u = half(dtype)
    for part in (torch.arange(0, 30, device=DEV), torch.arange(590, rows, device=DEV)):
        z = h[part].double() @ w.double().t() + b.double()
        p = torch.softmax(z, -1)
        one = torch.nn.functional.one_hot(t[part], V).double()
        logp = torch.log_softmax(z, -1).gather(-1, t[part][:, None])[:, 0]
        # (32 of the sum and the hardware's functions, 6 + 4 of a logit below 2^6, as above; 2^-24 of 400)
        assert float((got["logp"][part] - logp).abs().max()) < 1e-4
        dh, mag = (p - one) @ w.double(), (p + one) @ w.double().abs()
        close(got["hidden"][part], (dh, mag * (1.01 * u + 1e-5) + (u + 4 * F24) * dh.abs() + 1e-30), "hidden")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,V", [(300, 64, 25), (20, 64, 300), (300, 200, 22), (260, 40, 300)])
def test_graphs_of_every_shape(rows, D, V, dtype):
    """Two graphs at once, each replayed three times with eager calls between."""
    def one(seed):
        h, w, t, b, m = inputs(rows, D, V, dtype, seed, True, 0.3)
        x = [y.detach().clone().requires_grad_(True) for y in (h, w, b)]
        run(h, w, t, b, m)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = linear_cross_entropy(x[0], x[1], t, x[2], m)
            grads = torch.autograd.grad(r.loss, x)
        return graph, x, t, m, r, grads
    made = [one(60), one(61)]
    for seed in (1, 2, 3):
        new = []
        for n, (graph, x, t, m, r, grads) in enumerate(made):
            h2, _, t2, _, m2 = inputs(rows, D, V, dtype, 70 + 2 * seed + n, True, 0.25 * seed)
            with torch.no_grad():
                x[0].copy_(h2)
                t.copy_(t2)
                m.copy_(m2)
            new.append((h2, t2, m2))
        for graph, *_ in made:
            graph.replay()
        for (graph, x, t, m, r, grads), (h2, t2, m2) in zip(made, new):
            want = run(h2, x[1].detach(), t2, x[2].detach(), m2)
            assert torch.equal(r.loss, want["loss"]) and torch.equal(r.logp, want["logp"])
            assert all(torch.equal(y, want[k]) for y, k in zip(grads, ("hidden", "weight", "bias")))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,V", [(300, 64, 25), (300, 64, 300)])
def test_a_backward_captured_without_its_forward(rows, D, V, dtype):
    """Every replay leaves what an eager backward does, whatever became of the gradients in between."""
    h, w, t, b, m = inputs(rows, D, V, dtype, 62, True, 0.3)
    side = torch.cuda.Stream()
    for up in (1.0, 2.0):
        want = run(h, w, t, b, m, up)
        x = [y.clone().requires_grad_(True) for y in (h, w, b)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            loss = linear_cross_entropy(x[0], x[1], t, x[2], m).loss
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            grads = torch.autograd.grad(loss * up, x, retain_graph=True)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(y, want[k]) for y, k in zip(grads, ("hidden", "weight", "bias")))
            for y in grads:
                y.zero_()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,V", [(300, 64, 25), (300, 64, 300)])
def test_a_forward_and_its_backward_in_two_graphs(rows, D, V, dtype):
    """The second graph is replayed twice for a replay of the first."""
    for up in (1.0, 2.0):
        h, w, t, b, m = inputs(rows, D, V, dtype, 64, True, 0.3)
        x = [y.clone().requires_grad_(True) for y in (h, w, b)]
        run(h, w, t, b, m)
        torch.cuda.synchronize()
        one, two, side = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(one, stream=side):
            loss = linear_cross_entropy(x[0], x[1], t, x[2], m).loss
        with torch.cuda.graph(two, stream=side):
            grads = torch.autograd.grad(loss * up, x, retain_graph=True)
        for seed in (65, 66, 67):
            h, _, t2, _, m2 = inputs(rows, D, V, dtype, seed, True, 0.3)
            with torch.no_grad():
                x[0].copy_(h)
                t.copy_(t2)
                m.copy_(m2)
            one.replay()
            want = run(h, w, t2, b, m2, up)
            for _ in range(2):
                two.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(y, want[k]) for y, k in zip(grads, ("hidden", "weight", "bias")))
                for y in grads:
                    y.zero_()


@pytest.mark.parametrize("rows,D,V", [((1 << 24) + 33, 128, 9), ((1 << 21) + 33, 1032, 20)])
def test_offsets_beyond_32_bits(rows, D, V):
    """2^31 + elements of the hidden states; their last rows."""
    g = gen(13)
    h = torch.empty(rows, D, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    w = torch.randn(V, D, generator=g, device=DEV).to(torch.bfloat16) / 16
    t = torch.randint(0, V, (rows,), generator=g, device=DEV)
    assert h.numel() > 1 << 31
    got = run(h, w, t, None, None, reduction="sum")
    part = slice(rows - 70, rows)
    want = reference(h[part], w, t[part], None, None, reduction="sum")
    close(got["logp"][part], want["logp"], "logp")
    close(got["hidden"][part], want["hidden"], "hidden")


def test_only_what_is_wanted():
    h, w, t, b, _ = inputs(90, 33, 70, torch.bfloat16, 6)
    full = run(h, w, t, b, None)
    for want in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)):
        x = [y.detach().clone().requires_grad_(bool(n)) for y, n in zip((h, w, b), want)]
        linear_cross_entropy(x[0], x[1], t, x[2]).loss.backward()
        for y, n, name in zip(x, want, ("hidden", "weight", "bias")):
            assert (y.grad is None) == (not n)
            assert not n or torch.equal(y.grad, full[name]), (want, name)


def test_repeats_bit_for_bit_and_twice_backward():
    h, w, t, b, m = inputs(777, 80, 900, torch.bfloat16, 7, True, 0.2)
    a, c = run(h, w, t, b, m), run(h, w, t, b, m)
    assert all(torch.equal(a[k], c[k]) for k in a)
    x = h.detach().clone().requires_grad_(True)
    loss = linear_cross_entropy(x, w, t, b, m).loss
    g1, = torch.autograd.grad(loss, x, retain_graph=True)
    g2, = torch.autograd.grad(loss * 2.0, x)
    assert torch.equal(g1, a["hidden"]) and torch.equal(g2, 2 * g1)


def test_checkpoint_and_packed_tensors():
    h, w, t, b, m = inputs(64, 32, 100, torch.bfloat16, 11, True, 0.3)
    plain = run(h, w, t, b, m)

    def f(x, y, z):
        return linear_cross_entropy(x * 1.0, y, t, z, m).loss
    for hooks in (lambda: torch.autograd.graph.save_on_cpu(),
                  lambda: torch.autograd.graph.saved_tensors_hooks(lambda x: x.clone(), lambda x: x.clone())):
        leaves = [x.detach().clone().requires_grad_(True) for x in (h, w, b)]
        with hooks():
            loss = f(*leaves)
        loss.backward()
        for x, k in zip(leaves, ("hidden", "weight", "bias")):
            assert torch.equal(x.grad, plain[k])
    leaves = [x.detach().clone().requires_grad_(True) for x in (h, w, b)]
    checkpoint(f, *leaves, use_reentrant=False).backward()
    for x, k in zip(leaves, ("hidden", "weight", "bias")):
        assert torch.equal(x.grad, plain[k])


def test_on_another_stream_and_in_a_graph():
    h, w, t, b, m = inputs(500, 64, 700, torch.bfloat16, 12, True, 0.3)
    plain = run(h, w, t, b, m)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(h, w, t, b, m)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[k], plain[k]) for k in plain)
    x = [y.detach().clone().requires_grad_(True) for y in (h, w, b)]

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = linear_cross_entropy(x[0], x[1], t, x[2], m)
        grads = torch.autograd.grad(r.loss, x)
    for seed in (1, 2, 3):
        h2, _, t2, _, m2 = inputs(500, 64, 700, torch.bfloat16, 50 + seed, True, 0.1 * seed)
        with torch.no_grad():
            x[0].copy_(h2)
            t.copy_(t2)
            m.copy_(m2)
        graph.replay()
        torch.cuda.synchronize()
        want = run(h2, w, t2, b, m2)
        assert torch.equal(r.loss, want["loss"]) and torch.equal(r.logp, want["logp"])
        assert all(torch.equal(y, want[k]) for y, k in zip(grads, ("hidden", "weight", "bias")))


def test_gradients_against_differences():
    h, w, t, b, m = inputs(12, 6, 9, torch.float32, 13, True, 0.2)
    got = run(h, w, t, b, m)

    def f(h, w, b):
        z = h.double() @ w.double().t() + b.double()
        lp = torch.log_softmax(z, -1).gather(-1, t[:, None])[:, 0]
        return -lp[m].mean()
    g = gen(14)
    for k, name in enumerate(("hidden", "weight", "bias")):
        x = [h.double(), w.double(), b.double()]
        d = torch.randn(x[k].shape, generator=g, device=DEV, dtype=torch.float64)
        hi, lo = list(x), list(x)
        hi[k], lo[k] = x[k] + 1e-5 * d, x[k] - 1e-5 * d
        want = float((f(*hi) - f(*lo)) / 2e-5)
        # (the difference: 1e-10 of third derivatives, and 1e-16 / 1e-5 of rounding)
        assert abs(float((got[name].double() * d).sum()) - want) < 1e-5 * (1 + float(d.abs().sum()) * 1e-1)


def test_refusals():
    h, w, t, b, m = inputs(6, 4, 5, torch.float32, 1, True, 0.5)
    ok = dict(hidden=h, weight=w, targets=t, bias=b, mask=m)

    def call(**kw):
        return linear_cross_entropy(**{**ok, **kw})
    for error, word, kw in [
            (TypeError, "hidden must be", dict(hidden=h.double(), weight=w.double(), bias=b.double())),
            (TypeError, "weight must be", dict(weight=w.bfloat16())),
            (TypeError, "bias must be", dict(bias=b.half())),
            (TypeError, "targets must be", dict(targets=t.float())),
            (TypeError, "mask must be", dict(mask=m.int())),
            (ValueError, "weight must be", dict(weight=w[:, :3])),
            (ValueError, "weight must be", dict(weight=w[0])),
            (ValueError, "weight must be", dict(weight=w[:0])),
            (ValueError, "bias must be", dict(bias=b[:3])),
            (ValueError, "targets must be", dict(targets=t[:3])),
            (ValueError, "mask must be", dict(mask=m[:3])),
            (ValueError, "hidden must be", dict(hidden=h[:, :0], weight=w[:, :0])),
            (ValueError, "reduction", dict(reduction="none")),
            (ValueError, "is on", dict(weight=w.cpu())),
            (ValueError, "is on", dict(targets=t.cpu()))]:
        with pytest.raises(error, match=word):
            call(**kw)
    with pytest.raises(RuntimeError, match="HIP device"):
        call(hidden=h.cpu())
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(h, h)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(hidden=dual)
    x = h.clone().requires_grad_(True)
    one = torch.ones((), device=DEV, requires_grad=True)
    g, = torch.autograd.grad(call(hidden=x).loss, x, one, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    z = torch.complex(h, -h).conj()  # a negated view reads as it reads
    assert torch.equal(call(hidden=z.imag).loss, call(hidden=h).loss)


def test_under_compile_the_graph_breaks():
    h, w, t, b, m = inputs(16, 8, 9, torch.float32, 2, True, 0.3)
    f = torch.compile(lambda x: linear_cross_entropy(x * 1.0, w, t, b, m).loss * 2, backend="eager")
    assert torch.equal(f(h), linear_cross_entropy(h, w, t, b, m).loss * 2)
