"""The policy update on the GPU where its surroundings are unusual: saved tensors that were packed
or computed again, derivatives and views that it does not read, overlapping parameters, values at
the ends of the number range."""

import math
from fractions import Fraction

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from swarp_amd import (AdamW, adamw_state, adamw_step, categorical_policy_loss, gae,
                       gaussian_policy_loss, grad_norm)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------- packed and recomputed tensors


def poison(*like):
    """Takes the memory that tensors like these left, and fills it with NaN."""
    return [torch.full_like(t, math.nan) if t.is_floating_point() else torch.ones_like(t)
            for t in like for _ in range(4)]


def same_bits(a, b):
    """(float16 gradients of actions that the reference likes e^10 times more overflow)"""
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def packing():
    return torch.autograd.graph.saved_tensors_hooks(
        lambda x: x.detach().clone(memory_format=torch.contiguous_format), lambda x: x.clone())


def on_host():
    return torch.autograd.graph.save_on_cpu()


HEADS = [("cat", torch.float32), ("cat", torch.bfloat16), ("cat", torch.float16),
         ("shared", torch.float32), ("shared", torch.float16), ("rows", torch.bfloat16)]


def loss_case(kind, dtype, V):
    """A function from the leaves to the loss, and the leaves: the head, the deviations and all
    per-decision inputs are made inside, so that nothing but autograd keeps them."""
    g = gen(V)
    n, D = 6, V if kind == "cat" else 3
    base = torch.randn(3, n + 1, D, generator=g, device=DEV).to(dtype).requires_grad_(True)
    std = (torch.randn(D, generator=g, device=DEV) * 0.1).to(dtype).requires_grad_(True)
    act = torch.randint(0, D, (3, n), generator=g, device=DEV)
    row = [torch.randn(3, n, generator=g, device=DEV) for _ in range(3)]
    mask = torch.rand(3, n, generator=g, device=DEV) < 0.7

    def f(base, std):
        head = (base * 2)[:, :-1]
        old, adv, ref = (t + 0 for t in row)
        kw = dict(kl_coef=0.1, entropy_coef=0.1)
        if kind == "cat":
            return categorical_policy_loss(head, act + 0, old - 1, adv, ref - 1, mask & True, **kw).loss
        ls = std * 1.5
        ls = ls if kind == "shared" else ls.expand(3, n, D) * 1
        return gaussian_policy_loss(head, ls, head.detach().float() + 0.3, old - 1, adv, ref - 1,
                                    mask & True, **kw).loss
    return f, [base] if kind == "cat" else [base, std], base, std


@pytest.mark.parametrize("way", ["pack", "host", "checkpoint"])
@pytest.mark.parametrize("up", [1.0, 64.0])
@pytest.mark.parametrize("kind,dtype", HEADS)
def test_losses_under_hooks_and_checkpoints(kind, dtype, up, way):
    """The same gradients to the last bit, whoever keeps the saved tensors."""
    for V in (9, 300, 9000) if kind == "cat" else (3,):
        f, leaves, base, std = loss_case(kind, dtype, V)
        want = torch.autograd.grad(f(base, std) * up, leaves)
        if way == "checkpoint":
            loss = checkpoint(f, base, std, use_reentrant=False)
        else:
            with packing() if way == "pack" else on_host():
                loss = f(base, std)
        taken = poison(base, base[:, :-1], std, torch.zeros(3, 6, device=DEV),
                       torch.zeros(3, 6, dtype=torch.int64, device=DEV))
        got = torch.autograd.grad(loss * up, leaves)
        assert all(bool(t.any()) for t in want)
        assert all(same_bits(a, b) for a, b in zip(got, want)), (V, len(taken))


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("up", [1.0, 64.0])
@pytest.mark.parametrize("kind,dtype", HEADS)
def test_losses_whose_backward_is_a_graph_of_its_own(kind, dtype, up, apart):
    """Behind an eager forward, or one in another graph: every replay leaves what an eager backward does,
    whatever became of the gradients in between."""
    for V in (9, 300, 9000) if kind == "cat" else (3,):
        g = gen(V)
        head = torch.randn(18, V, generator=g, device=DEV).to(dtype)
        std = (torch.randn(*(() if kind == "shared" else (18,)), V, generator=g, device=DEV) * 0.1).to(dtype)
        act = torch.randint(0, V, (18,), generator=g, device=DEV) if kind == "cat" else head.float() + 0.3
        old, adv = (torch.randn(18, generator=g, device=DEV) for _ in range(2))

        def f(head, *std):
            if kind == "cat":
                return categorical_policy_loss(head, act, old - 1, adv).loss
            return gaussian_policy_loss(head, *std, act, old - 1, adv).loss
        x, y = ([t.clone().requires_grad_(True) for t in ((head,) if kind == "cat" else (head, std))] for _ in range(2))
        want = torch.autograd.grad(f(*x) * up, x)
        torch.cuda.synchronize()
        one, two, side = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(one, stream=side) if apart else torch.cuda.stream(side):
            loss = f(*y)
        torch.cuda.synchronize()
        with torch.cuda.graph(two, stream=side):
            got = torch.autograd.grad(loss * up, y, retain_graph=True)
        if apart:
            one.replay()
        for _ in range(3):
            two.replay()
            torch.cuda.synchronize()
            assert all(same_bits(a, b) for a, b in zip(got, want)), V
            for t in got:
                t.zero_()


@pytest.mark.parametrize("way", ["pack", "host", "checkpoint"])
@pytest.mark.parametrize("last", [False, True])
def test_gae_under_hooks_and_checkpoints(last, way):
    g = gen(3)
    r, v, f = (torch.randn(*s, generator=g, device=DEV) for s in ((70, 64), (71, 64), (70, 64)))
    ends = torch.rand(2, 70, 64, generator=g, device=DEV) < 0.2
    if last:
        r, v, f, ends = (t.transpose(-1, -2).contiguous() for t in (r, v, f, ends))
    x = [t.requires_grad_(True) for t in (r, v, f)]
    up = torch.randn(2, *r.shape, generator=g, device=DEV)

    def scan(r, v, f):
        return torch.stack(gae(r * 2, v, ends[0] & True, ends[1] & True, f * 1,
                               time_dim=-1 if last else 0))
    want = torch.autograd.grad(scan(*x), x, up)
    if way == "checkpoint":
        out = checkpoint(scan, *x, use_reentrant=False)
    else:
        with packing() if way == "pack" else on_host():
            out = scan(*x)
    taken = poison(ends[0], ends[0], r)
    got = torch.autograd.grad(out, x, up)
    assert all(torch.equal(a, b) for a, b in zip(got, want)), len(taken)


# ------------------------------------------------------------------------------ refusals


def test_overlapping_parameters_are_refused():
    b = torch.zeros(1000, device=DEV)
    p = [b[:300], b[100:400]]
    with pytest.raises(ValueError, match="share memory"):
        adamw_step(p, [torch.ones_like(x) for x in p], adamw_state(p), 1)
    assert not b.any()
    p = [b[:300], b[300:400]]
    adamw_step(p, [torch.ones_like(x) for x in p], adamw_state(p), 1)
    assert bool(b[:400].all()) and not b[400:].any()


def test_the_default_type_changes_nothing():
    g = [torch.randn(700, generator=gen(4), device=DEV)]

    def run():
        p = [torch.ones(700, device=DEV, dtype=torch.bfloat16)]
        state = adamw_state(p, bits=8, master=True)
        norm = adamw_step(p, g, state, 1, max_grad_norm=0.5)
        return (norm, *p, state.master, *state.moments(), *grad_norm(g, 0.5))
    want = run()
    torch.set_default_dtype(torch.float64)
    try:
        got = run()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got, want))


# --------------------------------------------------------------- without gradients, compiled


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [9, 50, 3000, 20000])
def test_losses_without_gradients(V, dtype):
    """The values of a call whose inputs need no gradient, or under no_grad, are those of one that
    leaves gradients, to the last bit (rows that are split have them formed in other workgroups,
    whose sums are joined in another order: there to 16 roundings)."""
    g = gen(V)
    x = (torch.randn(5, V, generator=g, device=DEV) * 2).to(dtype)
    act = torch.randint(0, V, (5,), generator=g, device=DEV)
    old, adv, ref = (torch.randn(5, generator=g, device=DEV) - 3 for _ in range(3))
    mask = torch.tensor([True, False, True, True, True], device=DEV)
    std = (torch.randn(5, 7, generator=g, device=DEV) * 0.2).to(dtype)

    def cat(x):
        return categorical_policy_loss(x, act, old, adv, ref, mask, kl_coef=0.1, entropy_coef=0.1)

    def gauss(x):
        return gaussian_policy_loss(x, std, x.detach().float() + 0.1, old, adv, ref, mask, kl_coef=0.1,
                                    entropy_coef=0.1)
    for f, head in ((cat, x), (gauss, x[:, :7].contiguous())):
        want = f(head.clone().requires_grad_(True))
        with torch.no_grad():
            under = f(head.clone().requires_grad_(True))
        for got in (f(head), under):
            assert not any(t.requires_grad for t in got)
            for a, b in zip(got, want):
                if V > 8192 and f is cat:
                    assert bool(((a - b).abs() <= 16 * 2.0 ** -24 * b.abs()).all())
                else:
                    assert torch.equal(a, b)


@pytest.mark.parametrize("backend", ["eager", "inductor"])
def test_compiled_callers(backend):
    """torch.compile runs functions that call the operators, with the same results: the graph
    breaks at them."""
    g = gen(8)
    r, v = torch.randn(20, 30, generator=g, device=DEV), torch.randn(21, 30, generator=g, device=DEV)
    x = torch.randn(30, 9, generator=g, device=DEV, requires_grad=True)
    act = torch.randint(0, 9, (30,), generator=g, device=DEV)

    def cat(x):
        adv = gae(r * 2, v).advantages[0] + 0
        return categorical_policy_loss(x * 2, act, adv - 3, adv, entropy_coef=0.1).loss * 4

    def gauss(x):
        adv = gae(r * 2, v).advantages[0] + 0
        return gaussian_policy_loss(x * 2, x[0] * 0.5, x.detach(), adv - 9, adv).loss * 4

    def step(x):
        p = [x.detach() * 2]
        state = adamw_state(p, bits=8)
        norm = adamw_step(p, [x.detach() * 4], state, 1, max_grad_norm=1.0)
        return (p[0], norm * 2, *grad_norm(p), *state.moments())
    for f in (cat, gauss):
        want, compiled = f(x), torch.compile(f, backend=backend)
        dwant, = torch.autograd.grad(want, x, retain_graph=True)
        for _ in range(2):
            got = compiled(x)
            assert torch.equal(want, got) and torch.equal(torch.autograd.grad(got, x)[0], dwant)
    want, compiled = step(x), torch.compile(step, backend=backend)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(compiled(x), want))


def test_compiled_optimizer():
    def go(wrap):
        p = torch.nn.Parameter(torch.ones(300, device=DEV))
        opt = AdamW([p], lr=0.1, max_grad_norm=0.5)
        step = wrap(opt.step)
        for k in range(3):
            p.grad = torch.linspace(-1, k, 300, device=DEV)
            step()
        return p.detach(), opt.last_grad_norm, opt.state_dict()["steps"]
    want, got = go(lambda f: f), go(lambda f: torch.compile(f, backend="eager"))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1]) and want[2] == got[2] == {0: 3}


# ------------------------------------------------------------- ends of the number range


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("V", [3, 40, 4100, 9000])
def test_a_reference_that_forbids_the_action(V, dtype):
    """The loss is infinite, its slope along the log-probability is -rho A + kl_coef."""
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    x = torch.zeros(4, V, device=DEV, dtype=dtype, requires_grad=True)
    act = torch.tensor([0, V - 1, 1, 0], device=DEV)
    old = torch.full((4,), -math.log(V), device=DEV, dtype=wide)
    ref = old.clone()
    ref[1] = -math.inf
    r = categorical_policy_loss(x, act, old, torch.ones_like(old), ref, kl_coef=0.25)
    r.loss.backward()
    assert float(r.loss) == math.inf and float(r.kl) == math.inf
    slope = torch.tensor([-1.0, -0.75, -1.0, -1.0], device=DEV, dtype=torch.float64)
    want = torch.full((4, V), -1 / V, device=DEV, dtype=torch.float64)
    want[torch.arange(4), act] += 1
    want *= slope[:, None] / 4
    # rho is off by a rounding of log V (9.1 at most), a handful more; one to the head's type
    tol = 16 * 2.0 ** (-53 if dtype == torch.float64 else -24) + (
        2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0.0)
    assert bool(((x.grad.double() - want).abs() <= tol).all())


def test_the_kl_term_of_small_differences():
    """With one action the log-probability is 0, and e the reference's: the mean of
    exp(e) - 1 - e to 16 roundings of itself, in float64 down to where e^2 is lost beside e."""
    for dtype, sizes in ((torch.float64, (1e-17, 1e-12, 1e-10, 1e-8, 1e-6, 1e-3, 0.1, 0.49, 0.6, 2.0)),
                         (torch.float32, (1e-12, 1e-8, 1e-4, 0.1, 0.49))):
        for e in (s * sign for s in sizes for sign in (1, -1)):
            ref = torch.full((1,), e, device=DEV, dtype=dtype)
            e = Fraction(float(ref))
            want, term = Fraction(0), Fraction(1)
            for k in range(1, 40):
                term *= e / k
                want += term if k > 1 else 0
            z = torch.zeros(1, device=DEV, dtype=dtype)
            r = categorical_policy_loss(z[:, None], z.long(), z, z, ref, kl_coef=1.0)
            tol = 16 * 2.0 ** (-53 if dtype == torch.float64 else -24)
            assert abs(float(r.kl) - float(want)) <= tol * float(want), (dtype, float(e))
            assert float(r.loss) == float(r.kl)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("lam", [0.0, 0.04, 1e-7, 0.9])
def test_what_is_not_finite_reaches_the_next_end(lam, last, dtype):
    """... and no further, wherever a stretch of the scan begins: A_t = d_t + gamma lam A_{t+1},
    whose product with 0 is NaN, and whose factors' product underflows over a long way."""
    T, N = 2500, 6
    r = torch.randint(-4, 5, (T, N), generator=gen(1), device=DEV).to(dtype)
    for n, x in enumerate((math.nan, math.inf, -math.inf) * 2):
        r[2300 - 7 * n, n] = x
    te = torch.zeros(T, N, dtype=torch.bool, device=DEV)
    te[1003, :3] = te[2400, 1] = True
    want, a, h = torch.empty(T, N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64), te.cpu()
    # (as the call rounds it)
    carry = float(torch.tensor(0.5 * lam, dtype=dtype))
    for t in reversed(range(T)):
        a = torch.where(h[t], r[t].cpu().double(), r[t].cpu().double() + carry * a)
        want[t] = a
    v = torch.zeros(T + 1, N, device=DEV, dtype=dtype)
    if last:
        r, v, te = (t.T.contiguous() for t in (r, v, te))
    got = gae(r, v, te, gamma=0.5, lam=lam, time_dim=-1 if last else 0).advantages
    got = (got.T if last else got).cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    ok = torch.isfinite(want)
    # sums of at most 4 / (1 - 0.45)
    assert float((got - want)[ok].abs().max()) <= 64 * 2.0 ** (-24 if dtype == torch.float32 else -53) * 8
    ok = torch.isinf(want)
    assert torch.equal(got[ok], want[ok])


@pytest.mark.parametrize("eps", [0.0, 1e-8])
@pytest.mark.parametrize("size", [1.0, 1e-10, 1e-18, 3e-21])
def test_adamw_where_second_moments_are_small(size, eps):
    """The update from the moments that the step stored, in float64: with eps = 0 and second moments
    down to below the smallest normal float.  A root and a reciprocal of an ulp or two each, three
    products: 8 roundings of the update, and those of the parameter."""
    n = 3000
    g = torch.randn(n, generator=gen(2), device=DEV) * size
    g = torch.where(g.abs() < 0.1 * size, 0.1 * size, g)
    p = [torch.zeros(n, device=DEV)]
    state = adamw_state(p)
    for t in (1, 2, 3):
        before = p[0].double()
        adamw_step(p, [g * t], state, t, lr=0.5, betas=(0.5, 0.75), eps=eps, weight_decay=0.0)
        m, v = (x[:n].double() for x in state.moments())
        assert bool((v > 0).all())
        update = 0.5 * (m / (1 - 0.5 ** t)) / ((v / (1 - 0.75 ** t)).sqrt() + eps)
        want = before - update
        tol = 2.0 ** -24 * (8 * update.abs() + want.abs())
        err = (p[0].double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
