"""What ``gae``, the policy losses and AdamW hand to the library, without a GPU: the library is a
stand-in that notes its arguments.  Under a saved-tensor hook or a checkpoint the forward's own
tensors are gone when the backward runs, so the addresses have to be those that autograd gives
back; and what a kernel reads at an address has to be what the tensor reads."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from swarp_amd import _lib, adamw_state, adamw_step, grad_norm, optim, policy

POINTERS = {"head", "log_std", "actions", "old_logp", "advantages", "ref_logp", "mask"}


class Library:
    """Answers every entry point with success."""

    def __init__(self):
        self.calls = []
        self.look = None  # called within each call, while its memory is alive

    def __getattr__(self, name):
        if name == "swarp_policy_work_bytes":
            return lambda rows, width: 64

        def call(arg, *rest):
            a = arg._obj if hasattr(arg, "_obj") else arg
            self.calls.append((name, type(a).from_buffer_copy(a), rest))
            if self.look is not None:
                self.look(a, rest)
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    for module in (policy, optim):
        monkeypatch.setattr(module, "_on_gpu", lambda t, what: None)
    return lib


class Packed(torch.autograd.graph.saved_tensors_hooks):
    """Keeps copies in place of the saved tensors; what it gave back is in ``given``."""

    def __init__(self, unpack=torch.clone):
        self.given = []

        def give(x):
            self.given.append(unpack(x))
            return self.given[-1]
        super().__init__(lambda x: x.detach().clone(memory_format=torch.contiguous_format), give)

    def addresses(self):
        return {t.data_ptr() for t in self.given}


def rows(n, dtype=torch.float32):
    return [torch.randn(n, dtype=dtype) for _ in range(3)]


HEADS = [("cat", torch.float32), ("cat", torch.float16), ("shared", torch.float32),
         ("rows", torch.float32), ("rows", torch.float16)]


def loss_of(kind, head, std, n):
    old, adv, ref = rows(n)
    mask = torch.ones(n, dtype=torch.bool)
    if kind == "cat":
        return policy.categorical_policy_loss(head, torch.zeros(n, dtype=torch.int64), old, adv,
                                              ref, mask).loss
    return policy.gaussian_policy_loss(head, std, torch.zeros(n, 2), old, adv, ref, mask).loss


def heads(kind, dtype, n):
    head = torch.randn(n, 2, dtype=dtype, requires_grad=True)
    std = {"cat": None, "shared": torch.zeros(2, dtype=dtype, requires_grad=True),
           "rows": torch.zeros(n, 2, dtype=dtype, requires_grad=True)}[kind]
    return head, std


@pytest.mark.parametrize("kind,dtype", HEADS)
def test_a_loss_reads_what_the_hook_gives_back(library, kind, dtype):
    head, std = heads(kind, dtype, 6)
    hook = Packed()
    with hook:
        loss = loss_of(kind, head, std, 6)
    for _ in range(2):  # the second backward computes into buffers of its own
        library.calls.clear()
        hook.given.clear()
        (loss * 0.5).backward(retain_graph=True)
        (name, a, rest), = library.calls
        assert name.endswith("_bwd")
        for field in POINTERS - ({"log_std"} if kind == "cat" else set()):
            assert getattr(a, field) in hook.addresses(), field


def test_rows_of_logits_are_read_as_they_now_lie(library):
    base = torch.randn(3, 5, 4, requires_grad=True)
    with Packed():  # gives back whole copies
        loss = policy.categorical_policy_loss(base[:, :-1], torch.zeros(3, 4, dtype=torch.int64),
                                              *(t.view(3, 4) for t in rows(12)[:2])).loss
    fwd = library.calls[-1][1]
    assert (fwd.inner, fwd.outer_stride, fwd.inner_stride) == (4, 20, 4)
    loss.backward()
    bwd = library.calls[-1][1]
    assert (bwd.inner, bwd.outer_stride, bwd.inner_stride) == (12, 0, 4)
    # a layout that two levels of strides do not reach is copied; one that they do is read
    library.calls.clear()
    with Packed(lambda x: x.repeat_interleave(2, -1)[..., ::2]):
        loss = policy.categorical_policy_loss(base[:, :-1], torch.zeros(3, 4, dtype=torch.int64),
                                              *(t.view(3, 4) for t in rows(12)[:2])).loss
    loss.backward()
    bwd = library.calls[-1][1]
    assert (bwd.inner, bwd.outer_stride, bwd.inner_stride) == (12, 0, 4)


def test_a_head_of_another_shape_is_refused(library):
    head = torch.randn(6, 2, requires_grad=True)
    with Packed(lambda x: x[:3]):
        loss = loss_of("cat", head, None, 6)
    library.calls.clear()
    with pytest.raises((RuntimeError, ValueError), match="saved"):
        loss.backward()
    assert not library.calls


@pytest.mark.parametrize("kind,dtype", HEADS)
def test_a_checkpointed_loss_reads_the_recomputed_head(library, kind, dtype):
    x, std = heads(kind, dtype, 6)
    made = []

    def f(x, std):
        made.append(x * 2)
        return loss_of(kind, made[-1], std, 6)
    (checkpoint(f, x, std, use_reentrant=False) * 0.5).backward()
    assert len(made) == 2
    name, a, _ = library.calls[-1]
    assert name.endswith("_bwd") and a.head == made[1].data_ptr() != made[0].data_ptr()


@pytest.mark.parametrize("last", [False, True])
def test_the_scan_reads_what_the_hook_gives_back(library, last):
    r, v, f = (torch.randn(*s, requires_grad=True) for s in ((4, 4), (4, 5) if last else (5, 4), (4, 4)))
    ends = torch.zeros(4, 4, dtype=torch.bool)
    hook = Packed(lambda x: x.T.contiguous().T)  # (as the flags were, in another order)
    with hook:
        out = policy.gae(r, v, ends, ends.clone(), f, time_dim=-1 if last else 0)
    g = torch.ones(4, 4)
    torch.autograd.backward(out, (g, g))
    name, a, _ = library.calls[-1]
    assert name == "swarp_gae_bwd" and a.rewards is None and a.values is None
    # made contiguous: neither the forward's flags nor the transposed ones
    gone = hook.addresses() | {ends.data_ptr()}
    assert a.terminated not in gone and a.truncated not in gone and a.terminated != a.truncated
    assert a.final_values == a.adj_advantages  # (alive; only looked at for being set)


def neg(t):
    """-t as a view that keeps its sign aside, as ``torch.conj`` makes them."""
    return torch._neg_view(t)


def floats(address, n):
    return list((ctypes.c_float * n).from_address(address))


def test_negated_views_are_handed_over_as_they_read(library):
    x = torch.arange(1.0, 13.0)
    seen = {}

    def look(a, rest):
        for name, _ in a._fields_:
            if getattr(a, name) and name in ("rewards", "values", "final_values", "head", "log_std",
                                             "old_logp", "advantages", "ref_logp"):
                seen[name] = floats(getattr(a, name), 2)
        if len(rest) == 3:
            seen["scale"] = floats(rest[1], 1)
    library.look = look
    h = neg(x.view(6, 2)).detach().requires_grad_(True)
    policy.gae(neg(x[:4]), neg(x[:5]), None, None, neg(x[:4]))
    assert all(seen[k] == [-1.0, -2.0] for k in ("rewards", "values", "final_values"))
    loss = policy.categorical_policy_loss(h, torch.zeros(6, dtype=torch.int64), neg(x[:6]), x[:6],
                                          neg(x[:6])).loss
    want = {"head": [-1.0, -2.0], "old_logp": [-1.0, -2.0], "ref_logp": [-1.0, -2.0]}
    assert {k: seen[k] for k in want} == want
    loss.backward(neg(torch.tensor(3.0)))
    assert {k: seen[k] for k in want} == want and seen["scale"] == [-3.0]
    seen.clear()
    policy.gaussian_policy_loss(h, neg(x[:2]), neg(x.view(6, 2)), x[:6], neg(x[:6])).loss.backward()
    assert seen["head"] == seen["log_std"] == seen["advantages"] == [-1.0, -2.0]
    with Packed(neg):
        loss = policy.categorical_policy_loss(h, torch.zeros(6, dtype=torch.int64), x[:6], x[:6]).loss
    loss.backward()
    assert seen["head"] == [1.0, 2.0] and seen["old_logp"] == [-1.0, -2.0]


def test_the_adjoint_of_the_scan_reads_negated_gradients(library):
    seen = []
    library.look = lambda a, rest: seen.append(a.adj_advantages and floats(a.adj_advantages, 2))
    r = torch.zeros(3, requires_grad=True)
    out = policy.gae(r, torch.zeros(4))
    torch.autograd.backward(out.advantages, neg(torch.tensor([1.0, 2.0, 3.0])))
    assert seen[-1] == [-1.0, -2.0]


def test_adamw_and_negated_views(library):
    p, g = [torch.ones(2)], [neg(torch.tensor([1.0, 2.0]))]
    seen = []

    def look(a, rest):
        table = rest[0] if isinstance(a, _lib.SwarpAdamW) else a
        seen.append(floats(table[0].grad, 2))
        if isinstance(a, _lib.SwarpAdamW) and a.grad_scale:
            seen.append(floats(a.grad_scale, 1))
    library.look = look
    adamw_step(p, g, adamw_state(p), 1, grad_scale=neg(torch.tensor([0.5])))
    grad_norm(g)
    assert seen == [[-1.0, -2.0], [-0.5], [-1.0, -2.0]]
    with pytest.raises(ValueError, match="negated"):
        adamw_step([neg(p[0])], g, adamw_state(p), 1)
    s = adamw_state(p)
    with pytest.raises(ValueError, match="exp_avg"):
        adamw_step(p, g, s._replace(exp_avg=neg(s.exp_avg)), 1)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(library, grad):
    """A tangent is not dropped in silence, whichever input has it."""
    def dual(*s):
        return forward_ad.make_dual(torch.zeros(*s), torch.ones(*s))
    act = torch.zeros(6, dtype=torch.int64)
    z = torch.zeros(6)
    with forward_ad.dual_level():
        h = torch.zeros(6, 2, requires_grad=grad)
        calls = [lambda: policy.gae(dual(3), torch.zeros(4, requires_grad=grad)),
                 lambda: policy.gae(torch.zeros(3, requires_grad=grad), dual(4)),
                 lambda: policy.gae(z[:3], torch.zeros(4), None, None, dual(3)),
                 lambda: policy.categorical_policy_loss(dual(6, 2), act, z, z),
                 lambda: policy.categorical_policy_loss(h, act, dual(6), z),
                 lambda: policy.categorical_policy_loss(h, act, z, dual(6)),
                 lambda: policy.categorical_policy_loss(h, act, z, z, dual(6)),
                 lambda: policy.gaussian_policy_loss(dual(6, 2), torch.zeros(2), h.detach(), z, z),
                 lambda: policy.gaussian_policy_loss(h, dual(2), h.detach(), z, z),
                 lambda: policy.gaussian_policy_loss(h, torch.zeros(2), dual(6, 2), z, z)]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert not library.calls
        policy.gae(z[:3], torch.zeros(4))  # nothing dual: as ever
    assert len(library.calls) == 1


def test_a_second_derivative_is_refused(library):
    """... as ``once_differentiable`` does: where the upstream gradient is to be differentiated."""
    head = torch.randn(6, 2, requires_grad=True)
    up = torch.ones((), requires_grad=True)
    g, = torch.autograd.grad(loss_of("cat", head, None, 6), head, up, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    r = torch.zeros(3, requires_grad=True)
    g, = torch.autograd.grad(policy.gae(r, torch.zeros(4)).advantages, r, up.expand(3),
                             create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_the_default_type_is_not_taken_for_float32(library, default):
    """What the kernels write as float32 is float32, whatever torch makes by default."""
    torch.set_default_dtype(default)
    try:
        p = [torch.zeros(300, dtype=torch.float32)]
        assert adamw_state(p, master=True).master.dtype == torch.float32
        assert all(x.dtype == torch.float32 for x in adamw_state(p).moments())
        assert all(x.dtype == torch.float32 for x in adamw_state(p, bits=8).moments())
        assert all(x.dtype == torch.float32 for x in grad_norm(p))
        assert adamw_step(p, p, adamw_state(p), 1, max_grad_norm=1.0).dtype == torch.float32
        out = policy.gae(p[0], torch.zeros(301, dtype=torch.float32))
        assert all(x.dtype == torch.float32 for x in out)
        z = p[0][:6]
        out = policy.categorical_policy_loss(z[:, None], z.long(), z, z)
        assert all(x.dtype == torch.float32 for x in out)
    finally:
        torch.set_default_dtype(torch.float32)
