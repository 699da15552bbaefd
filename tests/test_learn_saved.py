"""What the backwards of ``gae`` and the policy losses hand to the library, without a GPU: the
library is a stand-in that notes its arguments.  Under a saved-tensor hook or a checkpoint the
forward's own tensors are gone by then, so the addresses have to be those that autograd gives back."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from swarp_amd import _lib, policy

POINTERS = {"head", "log_std", "actions", "old_logp", "advantages", "ref_logp", "mask"}


class Library:
    """Answers every entry point with success."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name == "swarp_policy_work_bytes":
            return lambda rows, width: 64

        def call(arg, *rest):
            a = arg._obj
            self.calls.append((name, type(a).from_buffer_copy(a), rest))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    monkeypatch.setattr(policy, "_on_gpu", lambda t, what: None)
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
