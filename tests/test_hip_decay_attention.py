"""decay_attention and decay_attention_step on the GPU against the recurrence in float64.

Tolerances.  An output or a gradient is a sum of products of a decay, three inputs and a scale.
Everything is float32: each product and each addition on its way costs 2^-24 of the magnitudes that
meet there.  A term passes a score's sum (dk or dv additions), a chunk's (32), one multiplication and
one addition a chunk in the state (T / 32 of each), and a handful of factors (a decay's exponent is off
by 2^-24 of up to 33 steps' worth, below 33 here): in all at most (dk + dv + T / 16 + 150) 2^-24 of the sum
of all terms' magnitudes.  bfloat16 products are of two terms that leave 2^-16 of what they stand
for; the result is rounded to its type, half a step."""

import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from swarp_amd import decay_attention, decay_attention_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def inputs(T, batch, H, dk, dv, dtype, seed, starts=0.0, flags=None):
    g = gen(seed)
    q, k = (torch.randn(T, *batch, H, dk, generator=g, device=DEV).to(dtype) for _ in range(2))
    v = torch.randn(T, *batch, H, dv, generator=g, device=DEV).to(dtype)
    ld = -torch.rand(H, generator=g, device=DEV) * 0.3
    state = torch.randn(*batch, H, dk, dv, generator=g, device=DEV)
    s = torch.rand(T, *(batch if flags is None else flags), generator=g, device=DEV) < starts if starts else None
    return q, k, v, ld, state, s


def recurrence(q, k, v, ld, state, starts, scale=None):
    """The definition, step by step, in the inputs' type."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    S = torch.zeros(*q.shape[1:], v.shape[-1], dtype=q.dtype, device=DEV) if state is None else state
    decay, out = torch.exp(ld)[:, None, None], []
    for t in range(q.shape[0]):
        S = S * decay
        if starts is not None:
            f = starts[t].view(*starts.shape[1:], *([1] * (S.dim() - starts.dim() + 1)))
            S = torch.where(f, torch.zeros_like(S), S)
        S = S + k[t][..., :, None] * v[t][..., None, :]
        out.append((q[t][..., :, None] * S).sum(-2) * scale)
    return (torch.stack(out) if out else q.new_zeros(v.shape)), S


def both(q, k, v, ld, state, starts, g_out, g_state, scale=None):
    """Results and gradients in float64, and the sums of their terms' magnitudes."""
    res = []
    for f in (lambda x: x.double(), lambda x: x.double().abs()):
        x = [f(t).requires_grad_(True) for t in (q, k, v)] + ([f(state).requires_grad_(True)] if state is not None else [])
        o, S = recurrence(*x[:3], ld.double(), x[3] if state is not None else None, starts, scale if scale is None or f(torch.tensor(-1.0)) < 0 else abs(scale))
        d = torch.autograd.grad((o, S), x, (f(g_out), f(g_state)), allow_unused=True)
        d = [torch.zeros_like(y) if g is None else g for y, g in zip(x, d)]
        res.append([o.detach(), S.detach(), *d])
    return list(zip(*res))


def check(got, want, T, dk, dv, dtype, what):
    names = ("out", "state", "q", "k", "v", "state0")
    u = torch.finfo(dtype).eps / 2
    for name, y, (value, mag) in zip(names, got, want):
        own = u if name not in ("state", "state0") else 0.0
        tol = mag * ((dk + dv + T / 16 + 150) * 2.0 ** -24 + (2.0 ** -15 if dtype == torch.bfloat16 and name in ("out", "q", "k", "v") else 0.0))
        tol = tol + own * value.abs() + (torch.finfo(dtype).tiny if own else 0.0)
        assert y.shape == value.shape, (what, name)
        err = (y.double() - value).abs()
        assert bool((err <= tol).all()), f"{what} {name}: {float((err - tol).max())} above, error {float(err.max())}"


def run(q, k, v, ld, state, starts, g_out, g_state, scale=None):
    x = [t.detach().requires_grad_(True) for t in (q, k, v)] + ([state.detach().requires_grad_(True)] if state is not None else [])
    r = decay_attention(*x[:3], ld, x[3] if state is not None else None, starts, scale=scale)
    return [r.out.detach(), r.state.detach(), *torch.autograd.grad((r.out, r.state), x, (g_out, g_state))]


SHAPES = [(1, (3,), 2, 5, 7), (2, (1,), 1, 1, 1), (31, (2, 3), 2, 32, 32), (32, (5,), 3, 16, 33), (33, (4,), 1, 64, 64),
          (65, (2,), 2, 40, 72), (100, (3,), 2, 128, 128), (64, (2,), 3, 31, 100), (130, (1,), 1, 127, 3),
          (257, (2, 2), 2, 64, 32), (1000, (1,), 1, 48, 65), (32, (7,), 3, 32, 32), (17, (3, 3), 1, 24, 9), (32, (41,), 5, 8, 32),
          (8, (1,), 1, 32, 16), (40, (70,), 4, 32, 24), (96, (13,), 6, 11, 30),
          (40, (3,), 2, 9, 15), (33, (2,), 1, 13, 122), (70, (3,), 2, 58, 23), (1, (5,), 3, 33, 6), (34, (2,), 2, 8, 127), (20, (9,), 2, 30, 29)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,batch,H,dk,dv", SHAPES)
def test_against_float64(T, batch, H, dk, dv, dtype):
    for n, (starts, with_state) in enumerate([(0.0, True), (0.08, True), (0.3, False)]):
        q, k, v, ld, state, s = inputs(T, batch, H, dk, dv, dtype, T + dk + n, starts)
        state = state if with_state else None
        g = gen(n)
        g_out = torch.randn(v.shape, generator=g, device=DEV).to(dtype)
        g_state = torch.randn(*batch, H, dk, dv, generator=g, device=DEV)
        want = both(q, k, v, ld, state, s, g_out, g_state)
        check(run(q, k, v, ld, state, s, g_out, g_state), want, T, dk, dv, dtype, f"{T} {batch} {dk}x{dv} {dtype} {n}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_and_few(dtype):
    """Many chunks of few heads, where a scan may be taken apart along time."""
    for T, starts in ((4099, 0.0), (4096, 0.002)):
        q, k, v, ld, state, s = inputs(T, (1,), 2, 32, 40, dtype, T, starts)
        ld = ld * 0.05
        g = gen(1)
        g_out, g_state = torch.randn(v.shape, generator=g, device=DEV).to(dtype), torch.randn(1, 2, 32, 40, generator=g, device=DEV)
        want = both(q, k, v, ld, state, s, g_out, g_state)
        check(run(q, k, v, ld, state, s, g_out, g_state), want, T, 32, 40, dtype, f"{T} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_flags_shared_by_agents(dtype):
    for flags in ((6,), (6, 4), ()):
        q, k, v, ld, state, s = inputs(70, (6, 4), 2, 16, 24, dtype, 3, 0.1, flags)
        whole = s.view(*s.shape, *([1] * (3 - s.dim()))).expand(70, 6, 4).contiguous()
        a, b = decay_attention(q, k, v, ld, state, s), decay_attention(q, k, v, ld, state, whole)
        assert torch.equal(a.out, b.out) and torch.equal(a.state, b.state)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_start_stops_everything_and_no_step_looks_ahead(dtype):
    """NaN and infinities before a start, after a step and in the state: in the outputs exactly where
    the definition has them, and nowhere else."""
    T, H, dk, dv = 75, 2, 20, 36
    q, k, v, ld, state, _ = inputs(T, (4,), H, dk, dv, dtype, 21)
    s = torch.zeros(T, 4, dtype=torch.bool, device=DEV)
    s[0, 0] = s[40, 0] = s[50, 1] = s[10, 2] = s[12, 3] = s[33, 3] = True
    g_out, g_state = torch.randn_like(v), torch.randn_like(state)
    bad = [x.clone() for x in (q, k, v)]
    bad[2][39, 0, 0, 5] = math.nan       # just before a start
    bad[2][60, 0, 1, 7] = math.inf
    bad[1][49, 1, 0, 3] = math.nan
    bad[0][20, 1, 0, 3] = math.nan       # a query's own step alone
    bad[2][70, 2, 0, 1] = -math.inf
    state = state.clone()
    state[0, 0, 3, 3] = math.nan         # stopped at once
    state[2, 1, 0, 0] = math.inf         # stopped at step 10
    state[3, 0, 19, 35] = math.nan
    r = decay_attention(*bad, ld, state, s)
    want, S = recurrence(*(x.double() for x in bad), ld.double(), state.double(), s)
    for y, z, name in ((r.out, want, "out"), (r.state, S, "state")):
        assert torch.equal(y.isfinite(), z.isfinite()), name
        assert torch.equal(y.isnan(), z.isnan()), name
        on = z.isfinite()
        tol = 0.02 if dtype != torch.float32 and name == "out" else 1e-3
        assert bool(((y.double() - z)[on].abs() <= tol * (1 + z[on].abs())).all()), name
    # the gradients, too, are finite just where the definition's are
    x = [t.double().requires_grad_(True) for t in (*bad, state)]
    o, S = recurrence(*x[:3], ld.double(), x[3], s)
    want = torch.autograd.grad((o, S), x, (g_out.double(), g_state.double()))
    got = run(*bad, ld, state, s, g_out, g_state)[2:]
    for y, z, name in zip(got, want, ("q", "k", "v", "state")):
        assert torch.equal(y.isfinite(), z.isfinite()), name
        on = z.isfinite()
        tol = 0.02 if dtype != torch.float32 and name != "state" else 1e-3
        assert bool(((y.double() - z)[on].abs() <= tol * (1 + z[on].abs())).all()), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,batch,dk,dv", [(1, 9, 5, 7), (16, 3, 1, 1), (17, 3, 2, 33), (53, 3, 31, 100), (70, 20, 32, 32), (53, 3, 64, 65),
                                           (53, 3, 127, 3), (40, 3, 3, 127), (75, 3, 128, 128), (2100, 1, 20, 24)])
def test_what_is_not_finite_in_every_shape(T, batch, dk, dv, dtype):
    """NaN and infinities anywhere, among starts: what the definition has finite is right, and the rest is not finite."""
    H = 2
    q, k, v, ld, state, s = inputs(T, (batch,), H, dk, dv, dtype, T + dv, 0.08)
    g = gen(5)
    g_out = torch.randn(v.shape, generator=g, device=DEV).to(dtype)
    g_state = torch.randn(state.shape, generator=g, device=DEV)
    for n, x in enumerate((q, k, v, state, g_out, g_state)):
        at = torch.randint(0, x.numel(), (3,), generator=g, device=DEV)
        x.view(-1)[at[:2]], x.view(-1)[at[2]] = math.nan, math.inf
    if T > 60:  # a padded end
        for x in (q, k, v, g_out):
            x[T - 20:, 0] = math.nan
    if T > 1000:
        ld = ld * 0.1
    x = [t.double().requires_grad_(True) for t in (q, k, v, state)]
    o, S = recurrence(*x[:3], ld.double(), x[3], s)
    want = [o.detach(), S.detach(), *torch.autograd.grad((o, S), x, (g_out.double(), g_state.double()))]
    # (what is finite has none of the others in it: its terms' magnitudes are those without them)
    clean = [torch.nan_to_num(t, 0.0, 0.0, 0.0) for t in (q, k, v, ld, state, g_out, g_state)]
    mags = [m for _, m in both(*clean[:5], s, *clean[5:])]
    got = run(q, k, v, ld, state, s, g_out, g_state)
    keep = []
    for name, y, z in zip(("out", "state", "q", "k", "v", "state0"), got, want):
        assert torch.equal(y.isfinite(), z.isfinite()), name
        keep.append(torch.where(z.isfinite(), y, 0.0))
    check(keep, [(torch.where(z.isfinite(), z, 0.0), m) for z, m in zip(want, mags)], T, dk, dv, dtype, f"{T} {dk}x{dv} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,dk,dv", [(20, 24, 32), (150, 24, 32), (150, 40, 72), (2100, 16, 32)])
def test_a_start_stops_what_passed_the_largest_float(T, dk, dv, dtype):
    """Finite parts whose state, or whose products with it, are not: what a start parts from them is as if
    they had been ordinary.  `clean` has ordinary values in their place."""
    q, k, v, ld, state, _ = inputs(T, (3,), 2, dk, dv, dtype, T + dk)
    ld, cut = ld * 0.2, T * 2 // 3
    s = torch.zeros(T, 3, dtype=torch.bool, device=DEV)
    s[cut] = True
    g = gen(2)
    g_out = torch.randn(v.shape, generator=g, device=DEV).to(dtype)
    g_state = torch.randn(state.shape, generator=g, device=DEV)
    large = torch.full_like(state, 3e38)
    many = [10 * q, k, v, ld, state, s, 10 * g_out, g_state]
    many_back = [q, 10 * k, 10 * v, ld, state, s, g_out, g_state]
    late, early = slice(cut, T), slice(0, cut)
    cases = [("state", many, {4: large}, late), ("gradient of the state", many_back, {7: large}, early)]
    if dtype != torch.float16:  # (its products stay below 2^32)
        first, last = torch.ones(T, 1, 1, 1, device=DEV), torch.ones(T, 1, 1, 1, device=DEV)
        first[:cut], last[cut:] = 1e20, 1e20
        plain = [q, k, v, ld, state, s, g_out, g_state]
        cases += [("k and v", plain, {1: (k * first).to(dtype), 2: (v * first).to(dtype)}, late),
                  ("q and gradients", plain, {0: (q * last).to(dtype), 6: (g_out * last).to(dtype)}, early)]
    for what, clean, changed, part in cases:
        want = both(*clean)
        got = run(*(changed.get(n, x) for n, x in enumerate(clean)))
        assert not all(bool(x.isfinite().all()) for x in got), what  # (it did pass)
        keep = [x[part] if n in (0, 2, 3, 4) else x for n, x in enumerate(got)]
        wanted = [(x[part], y[part]) if n in (0, 2, 3, 4) else (x, y) for n, (x, y) in enumerate(want)]
        keep[1 if part is early else 5] = wanted[1 if part is early else 5][0]  # (of the other side)
        check(keep, wanted, T, dk, dv, dtype, f"{what} {T} {dk}x{dv} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_padded_ends_reach_nothing_before_them(dtype):
    q, k, v, ld, _, _ = inputs(90, (3,), 2, 32, 48, dtype, 23)
    clean = decay_attention(q, k, v, ld).out
    for t in (q, k, v):
        t[71:, 1] = math.nan
        t[13:, 2] = math.inf
    out = decay_attention(q, k, v, ld).out
    assert torch.equal(out[:, 0], clean[:, 0])
    u = 4 * torch.finfo(dtype).eps  # (a chunk with something that is not finite goes step by step)
    for b, n in ((1, 71), (2, 13)):
        assert bool(((out[:n, b] - clean[:n, b]).abs() <= u * (8 + clean[:n, b].abs())).all())


def test_decays_at_the_ends_of_their_range():
    q, k, v, ld, state, s = inputs(70, (2,), 4, 16, 16, torch.float32, 25, 0.05)
    ld[0], ld[1], ld[2], ld[3] = 0.0, -200.0, -math.inf, -1e-8
    out, S = decay_attention(q, k, v, ld, state, s)
    want, W = recurrence(q.double(), k.double(), v.double(), ld.double(), state.double(), s)
    assert bool(((out - want).abs() <= 1e-4 * (1 + want.abs())).all())
    assert bool(((S - W).abs() <= 1e-4 * (1 + W.abs())).all())


def test_large_values():
    """States beyond float16's range, from float16 inputs; scores near bfloat16's."""
    for dtype, size in ((torch.float16, 200.0), (torch.bfloat16, 1e12), (torch.float32, 1e12)):
        q, k, v, ld, state, s = inputs(80, (2,), 1, 32, 32, dtype, 27)
        k, v, ld = k * size, v * size, ld * 0.01
        q = q * 1e-6 if dtype == torch.float16 else q / size
        S = decay_attention(q, k, v, ld).state
        want, W = recurrence(q.double(), k.double(), v.double(), ld.double(), None, None)
        assert bool(((S - W).abs() <= 1e-5 * W.abs().amax()).all())
        out = decay_attention(q, k, v, ld).out
        assert bool(((out - want).abs() <= 0.02 * want.abs().amax()).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_equals_scan(dtype):
    T = 20
    q, k, v, ld, state, s = inputs(T, (5, 3), 2, 33, 20, dtype, 29, 0.2, (5,))
    mine = state.clone()
    outs = [decay_attention_step(q[t], k[t], v[t], ld, mine, s[t]) for t in range(T)]
    want = both(q, k, v, ld, state, s, v * 0, state * 0)
    check([torch.stack(outs), mine], want[:2], T, 33, 20, dtype, "step")
    r = decay_attention(q, k, v, ld, state, s)
    check([r.out, r.state], want[:2], T, 33, 20, dtype, "scan")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,H,dk,dv", [((), 1, 1, 1), ((1,), 3, 128, 128), ((7,), 2, 64, 64), ((300,), 2, 32, 32), ((9,), 1, 17, 130 - 3), ((1000,), 1, 4, 4),
                                           ((40,), 3, 33, 5), ((41,), 2, 65, 6), ((70,), 2, 32, 31), ((5, 3), 2, 9, 66)])
def test_step(batch, H, dk, dv, dtype):
    q, k, v, ld, state, s = inputs(1, batch, H, dk, dv, dtype, dk + dv, 0.3)
    mine = state.clone()
    version = mine._version
    out = decay_attention_step(q[0], k[0], v[0], ld, mine, s[0] if batch else None, scale=0.7)
    assert mine._version > version
    want = both(q, k, v, ld, state, s if batch else None, v * 0, state * 0, 0.7)
    check([out[None], mine], want[:2], 1, dk, dv, dtype, "step")
    # what a started episode's state held is not looked at
    if batch:
        dirty = torch.where(s[0].view(*batch, 1, 1, 1), math.nan, state)
        again = decay_attention_step(q[0], k[0], v[0], ld, dirty, s[0], scale=0.7)
        assert torch.equal(again, out) and torch.equal(dirty, mine)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """Parts of one projection, batch-first views, heads in front."""
    g = gen(31)
    T, B, H, D = 50, 3, 2, 16
    ld = torch.full((H,), -0.1, device=DEV)
    qkv = torch.randn(T, B, H, 3 * D, generator=g, device=DEV).to(dtype)
    first = torch.randn(B, T, 3, H, D, generator=g, device=DEV).to(dtype)
    heads = torch.randn(B, H, T, 3, D, generator=g, device=DEV).to(dtype)
    odd = torch.randn(T, B, H, D, 3, generator=g, device=DEV).to(dtype)
    for parts in (qkv.split(D, -1), first.movedim(1, 0).unbind(2), heads.permute(2, 0, 1, 3, 4).unbind(3), odd.unbind(-1)):
        plain = [t.contiguous() for t in parts]
        x = [t.detach().requires_grad_(True) for t in parts]
        y = [t.detach().requires_grad_(True) for t in plain]
        a, b = decay_attention(*x, ld), decay_attention(*y, ld)
        assert torch.equal(a.out, b.out) and torch.equal(a.state, b.state)
        go = torch.randn_like(b.out)
        for s, t in zip(torch.autograd.grad(a.out, x, go), torch.autograd.grad(b.out, y, go)):
            assert torch.equal(s, t)
        S1, S2 = torch.zeros(B, H, D, D, device=DEV), torch.zeros(B, H, D, D, device=DEV)
        o1 = decay_attention_step(*(t[0] for t in parts), ld, S1)
        assert torch.equal(o1, decay_attention_step(*(t[0] for t in plain), ld, S2)) and torch.equal(S1, S2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(32, 32), (17, 31), (8, 3)])
def test_a_scan_of_one_step(dk, dv, dtype):
    """What a started episode's state held is not looked at; the state that was given stays."""
    q, k, v, ld, state, s = inputs(1, (40, 3), 2, dk, dv, dtype, 45, 0.5)
    s = s[..., 0]  # an env's, shared by its agents
    want = both(q, k, v, ld, state, s, v * 0, state * 0, 0.7)
    dirty = torch.where(s[0].view(40, 1, 1, 1, 1), math.nan, state)
    kept = dirty.clone()
    got = decay_attention(q, k, v, ld, dirty, s, scale=0.7)
    check([got.out, got.state], want[:2], 1, dk, dv, dtype, "one step")
    assert torch.equal(dirty.nan_to_num(7.0), kept.nan_to_num(7.0))
    now = dirty.clone()
    out = decay_attention_step(q[0], k[0], v[0], ld, now, s[0], scale=0.7)
    check([out[None], now], want[:2], 1, dk, dv, dtype, "step")


def test_offsets_beyond_32_bits():
    """2^31 + elements of q, k, v at once (one tensor, 4.3 GB).  What is 60 steps away weighs e^-180: the first
    and the last steps are those of short calls."""
    T, B, D, far = (1 << 20) + 77, 16, 128, 60
    x = torch.randn(T, B, 1, D, generator=gen(46), device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    assert x.numel() > 1 << 31
    ld = torch.full((1,), -3.0, device=DEV)
    r = decay_attention(x, x.detach(), x.detach(), ld)
    one = torch.ones((), device=DEV, dtype=torch.bfloat16).expand(r.out.shape)
    d, = torch.autograd.grad(r.out, x, one)
    for part in (slice(0, 3 * far), slice(T - 3 * far, T)):
        y = x[part].detach().clone().requires_grad_(True)
        want = decay_attention(y, y.detach(), y.detach(), ld)
        w, = torch.autograd.grad(want.out, y, one[part])
        keep = slice(0, far) if part.start == 0 else slice(-far, None)
        # (chunks may begin elsewhere: products of 2^-8 halves' sums of 16 bits, and the end's rounding)
        for got, wanted in ((r.out[part][keep], want.out[keep]), (d[part][keep], w[keep])):
            assert float((got.float() - wanted.float()).abs().max()) <= 2.0 ** -7 * float(wanted.float().abs().max())
    assert torch.allclose(r.state, want.state, rtol=1e-4, atol=1e-4 * float(want.state.abs().max()))


def test_more_than_2_32_units_of_heads():
    """Three scans of 2^32 / 3 heads of one element (45 GB).  The last head's state, which a start parts it
    from, is 3e38, and its product with q past the largest float."""
    n = (1 << 32) // 3 + 99
    x = torch.randn(1, n, 1, 1, generator=gen(47), device=DEV, dtype=torch.bfloat16)
    state = torch.zeros(n, 1, 1, 1, device=DEV)
    starts = torch.zeros(1, n, dtype=torch.bool, device=DEV)
    x[0, -1], state[-1], starts[0, -1] = 10.0, 3e38, True
    q = x.requires_grad_(True)
    r = decay_attention(q, x.detach(), x.detach(), torch.full((1,), -1.0, device=DEV), state, starts)
    d, = torch.autograd.grad(r.out, q, torch.full_like(r.out, 2.0))
    assert float(r.out[0, -1]) == 1000.0 and float(d[0, -1]) == 200.0 and float(r.state[-1]) == 100.0
    for a in range(0, n, 1 << 28):
        y = x.detach()[0, a:a + (1 << 28), 0, 0].float()
        # (two terms of a score, and the end's rounding)
        for got, want in ((r.out, y * y * y), (d, 2 * y * y)):
            assert bool(((got.detach()[0, a:a + (1 << 28), 0, 0].float() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-30).all())


def test_step_under_inference_mode():
    q, k, v, ld, state, s = inputs(1, (3,), 2, 8, 8, torch.float32, 44, 0.3)
    want = decay_attention(q, k, v, ld, state, s)
    for own in (True, False):  # (a state of inference mode has no version to count)
        with torch.inference_mode():
            now = state.clone() if own else None
        now = now if own else state.clone()
        version = None if own else now._version
        with torch.inference_mode():
            out = decay_attention_step(q[0], k[0], v[0], ld, now, s[0])
        assert torch.allclose(out, want.out[0], rtol=1e-5, atol=1e-5)
        assert torch.allclose(now, want.state, rtol=1e-5, atol=1e-5)
        assert own or now._version > version


def test_step_with_parts_of_the_state():
    state = torch.randn(4, 2, 8, 8, device=DEV)
    q = torch.randn(4, 2, 8, device=DEV)
    ld = torch.full((2,), -0.5, device=DEV)
    with pytest.raises(RuntimeError, match="in the state"):
        decay_attention_step(q, q, state[:, :, 3], ld, state)
    both = torch.randn(4 * 2 * 8 + 4 * 2 * 8 * 8, device=DEV)  # beside each other
    decay_attention_step(q, q, both[:64].view(4, 2, 8), ld, both[64:].view(4, 2, 8, 8))


def test_empty_calls():
    for T, B in ((0, 3), (5, 0), (0, 0)):
        q, k, v, ld, state, s = inputs(T, (B,), 2, 8, 8, torch.float32, 1)
        x = [t.requires_grad_(True) for t in (q, k, v, state)]
        r = decay_attention(*x[:3], ld, x[3])
        assert r.out.shape == (T, B, 2, 8) and torch.equal(r.state, state)
        d = torch.autograd.grad(r.state.sum() + r.out.sum(), x)
        assert bool((d[3] == 1).all()) and not any(t.any() for t in d[:3])
        r = decay_attention(*x[:3], ld)
        assert not r.state.any()


@pytest.mark.parametrize("T", [0, 5])
@pytest.mark.parametrize("batch", [(4, 0), (0, 4), (3, 0, 2)])
def test_empty_axes_of_the_batch(T, batch):
    q, k, v, ld, state, _ = inputs(T, batch, 2, 8, 6, torch.float32, 1)
    for s in (None, torch.zeros(T, *batch[:1], dtype=torch.bool, device=DEV), torch.zeros(T, *batch, dtype=torch.bool, device=DEV)):
        x = [t.clone().requires_grad_(True) for t in (q, k, v, state)]
        r = decay_attention(*x[:3], ld, x[3], s)
        assert r.out.shape == v.shape and r.state.shape == state.shape
        d = torch.autograd.grad(r.out.sum() + r.state.sum(), x)
        assert [t.shape for t in d] == [t.shape for t in x]
    if T:
        out = decay_attention_step(q[0], k[0], v[0], ld, state, s[0])
        assert out.shape == v.shape[1:]


def test_one_result_alone_and_parts_that_want_nothing():
    q, k, v, ld, state, s = inputs(40, (2,), 2, 16, 16, torch.float32, 33, 0.1)
    x = [t.requires_grad_(True) for t in (q, k, v, state)]
    r = decay_attention(*x[:3], ld, x[3], s)
    go, gs = torch.randn_like(r.out), torch.randn_like(r.state)
    zero = torch.autograd.grad((r.out, r.state), x, (go, gs * 0), retain_graph=True)
    for a, b in zip(zero, torch.autograd.grad(r.out, x, go, retain_graph=True)):
        assert torch.equal(a, b)
    zero = torch.autograd.grad((r.out, r.state), x[1:], (go * 0, gs), retain_graph=True)
    for a, b in zip(zero, torch.autograd.grad(r.state, x[1:], gs, retain_graph=True)):
        assert torch.equal(a, b)
    full = torch.autograd.grad((r.out, r.state), x, (go, gs))
    for n in range(4):
        y = [t.detach().requires_grad_(i == n) for i, t in enumerate(x)]
        r = decay_attention(*y[:3], ld, y[3], s)
        g, = torch.autograd.grad((r.out, r.state), [y[n]], (go, gs), allow_unused=True)
        assert torch.equal(g, full[n])


def test_checkpoint_hooks_and_changed_inputs():
    q, k, v, ld, state, s = inputs(40, (3,), 2, 24, 16, torch.bfloat16, 35, 0.1)
    go = torch.randn_like(v)

    def grads(wrap):
        x = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(wrap(lambda *y: decay_attention(*(t * 1.0 for t in y), ld, state, s).out, *x), x, go)
    plain = grads(lambda f, *x: f(*x))

    def hooked(f, *x):
        with torch.autograd.graph.save_on_cpu():
            return f(*x)
    for other in (grads(lambda f, *x: checkpoint(f, *x, use_reentrant=False)), grads(hooked)):
        assert all(torch.equal(a, b) for a, b in zip(plain, other))
    x = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    mine = state.clone()
    out = decay_attention(*x, ld, mine, s).out
    decay_attention_step(q[0], k[0], v[0], ld, mine)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_streams_and_graphs():
    q, k, v, ld, state, s = inputs(100, (6,), 2, 32, 32, torch.bfloat16, 37, 0.05)
    go, gs = torch.randn_like(v), torch.randn_like(state)
    plain = run(q, k, v, ld, state, s, go, gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(q, k, v, ld, state, s, go, gs)
        mine = state.clone()
        decay_attention_step(q[0], k[0], v[0], ld, mine, s[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(plain, other))
    graph, act = torch.cuda.CUDAGraph(), state.clone()
    with torch.cuda.graph(graph):
        got = run(q, k, v, ld, state, s, go, gs)
        out = decay_attention_step(q[0], k[0], v[0], ld, act, s[0])
    torch.cuda.synchronize()
    act.copy_(state)
    eager = state.clone()
    for n in range(3):
        fresh = inputs(100, (6,), 2, 32, 32, torch.bfloat16, 40 + n, 0.05)
        for a, b in zip((q, k, v, state, s), (*fresh[:3], *fresh[4:])):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = run(q, k, v, ld, state, s, go, gs)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(out, decay_attention_step(q[0], k[0], v[0], ld, eager, s[0])) and torch.equal(act, eager)


def test_gradients_against_differences():
    q, k, v, ld, state, s = inputs(40, (1,), 1, 5, 6, torch.float32, 39, 0.05)
    go, gs = torch.randn_like(v), torch.randn_like(state)
    got = run(q, k, v, ld, state, s, go, gs)[2:]
    x = [t.double() for t in (q, k, v, state)]

    def f(y):
        o, S = recurrence(*y[:3], ld.double(), y[3], s)
        return float((o * go).sum() + (S * gs).sum())
    for n in range(4):
        d = torch.randn(x[n].shape, generator=gen(n), device=DEV, dtype=torch.float64)
        hi, lo = list(x), list(x)
        hi[n], lo[n] = x[n] + 1e-5 * d, x[n] - 1e-5 * d
        want = (f(hi) - f(lo)) / 2e-5
        # (linear in each part: the difference is off by rounding alone, 1e-16 / 1e-5 of the sum)
        assert abs(float((got[n].double() * d).sum()) - want) < 1e-4 * (1 + abs(want))


def test_refusals():
    q, k, v, ld, state, s = inputs(6, (4, 2), 2, 8, 5, torch.float32, 41, 0.1)
    ok = dict(q=q, k=k, v=v, log_decay=ld, state=state, starts=s)
    step = dict(ok, q=q[0], k=k[0], v=v[0], starts=s[0])
    for error, word, kw in [
            (TypeError, "q must be", dict(q=q.double())),
            (TypeError, "k must be", dict(k=k.half())),
            (TypeError, "log_decay must be", dict(log_decay=ld.double())),
            (TypeError, "state must be", dict(state=state.half())),
            (TypeError, "starts must be", dict(starts=s.int())),
            (ValueError, "k must be", dict(k=k[..., :4])),
            (ValueError, "v must be", dict(v=v[:3])),
            (ValueError, "q must be", dict(q=q[0, 0, 0, 0])),
            (ValueError, "log_decay must be", dict(log_decay=ld[:1])),
            (ValueError, "log_decay requires grad", dict(log_decay=ld.clone().requires_grad_(True))),
            (ValueError, "state must be", dict(state=state[:3])),
            (ValueError, "starts must be", dict(starts=s[:, :3])),
            (ValueError, "starts must be", dict(starts=s[:3])),
            (ValueError, "wide", dict(q=q.repeat(1, 1, 1, 1, 17), k=k.repeat(1, 1, 1, 1, 17))),
            (ValueError, "wide", dict(v=v[..., :0])),
            (ValueError, "scale", dict(scale=math.inf)),
            (ValueError, "is on", dict(v=v.cpu())),
            (ValueError, "is on", dict(log_decay=ld.cpu()))]:
        with pytest.raises(error, match=word):
            decay_attention(**{**ok, **kw})
    for error, word, kw in [
            (ValueError, "state must be", dict(state=state.half())),
            (ValueError, "state must be", dict(state=state[:3])),
            (ValueError, "state must be", dict(state=state.transpose(0, 1).contiguous().transpose(0, 1))),
            (ValueError, "state must be", dict(state=state[:1, :1, :1, :1, :1].expand(state.shape))),
            (RuntimeError, "not differentiable", dict(q=q[0].clone().requires_grad_(True))),
            (RuntimeError, "not differentiable", dict(state=state.clone().requires_grad_(True))),
            (ValueError, "starts must be", dict(starts=s[0, :3]))]:
        with pytest.raises(error, match=word):
            decay_attention_step(**{**step, **kw})
    with pytest.raises(RuntimeError, match="HIP device"):
        decay_attention(**dict(ok, q=q.cpu()))
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            decay_attention(**dict(ok, q=torch.autograd.forward_ad.make_dual(q, q)))
    x = q.clone().requires_grad_(True)
    one = torch.ones(v.shape, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(decay_attention(**dict(ok, q=x)).out, x, one, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_more_heads_than_a_launch_takes_are_refused():
    x = torch.zeros(1, (1 << 22) + 1, 1, device=DEV)
    with pytest.raises(ValueError, match="4194304 of them"):
        decay_attention(x, x, x, x[0, :, 0])
    with pytest.raises(ValueError, match="4194304 of them"):
        decay_attention_step(x, x, x, x[0, :, 0], x[..., None])
    y = x[:, 1:]
    assert decay_attention(y, y, y, y[0, :, 0]).out.shape == y.shape


def test_under_compile_the_graph_breaks():
    q, k, v, ld, state, s = inputs(6, (4,), 2, 8, 5, torch.float32, 43, 0.1)
    f = torch.compile(lambda x: decay_attention(x * 1.0, k, v, ld, state, s).out * 2, backend="eager")
    assert torch.equal(f(q), decay_attention(q, k, v, ld, state, s).out * 2)
    a, b = state.clone(), state.clone()
    f = torch.compile(lambda x: decay_attention_step(x * 1.0, k[0], v[0], ld, a, s[0]) * 2, backend="eager")
    assert torch.equal(f(q[0]), decay_attention_step(q[0], k[0], v[0], ld, b, s[0]) * 2) and torch.equal(a, b)
