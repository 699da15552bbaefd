"""The memory of a policy along an episode: linear attention with a decay for each head, as a scan
over a rollout's steps for training (:func:`decay_attention`) and as a single step for acting
(:func:`decay_attention_step`), hand-written kernels with their adjoint behind ``torch.autograd``.

In the manner of :func:`swarp_amd.gae`: time comes first, flags per env are shared by its agents,
HIP tensors only, every launch on torch's current stream, shapes and types checked before any
launch, no host synchronisation.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.compiler import is_dynamo_compiling

from . import _lib
from .policy import (_CODES, _differentiable_once, _guard, _no_tangents, _on_gpu, _plain, _ptr,
                     _same, _untraced)

_MOST_DIM, _MOST_HEADS = 128, 1 << 22


class DecayAttention(NamedTuple):
    """Result of :func:`decay_attention`."""

    out: torch.Tensor    # [T, *batch, H, Dv], of v's type
    state: torch.Tensor  # [*batch, H, Dk, Dv] after the last step, float32


def _strides(x: torch.Tensor, lead: int):
    """(step, batch, head) strides of ``x [*lead, H, D]`` with ``lead`` leading axes, the first of
    them time where there is one more than the batch's; None where one stride does not reach the
    batch or the last axis is not dense."""
    if x.numel() == 0:  # (nothing to reach)
        return 0, 0, 0
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        return None
    size, step = 1, 0
    for n, st in zip(reversed(x.shape[lead:-2]), reversed(x.stride()[lead:-2])):
        if n == 1:
            continue
        if size == 1:
            step = st
        elif st != size * step:
            return None
        size *= n
    return (x.stride(0) if lead else 0), step, x.stride(-2)


def _laid(x: torch.Tensor, lead: int):
    """``x`` as its memory reads, and its strides."""
    if x.is_neg():
        x = _plain(x)
    s = _strides(x, lead)
    if s is None:
        x = x.contiguous()
        s = _strides(x, lead)
    return x, (ctypes.c_int64 * 3)(*s)


def _arguments(what: str, q, k, v, log_decay, state, starts, scale, lead: int):
    """Everything checked, and the shape: (dtype, device, T, batch, H, Dk, Dv, scale, group)."""
    _on_gpu(q, what)
    dtype, dev, nd = q.dtype, q.device, q.dim()
    if dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"q must be float32, bfloat16 or float16; got {dtype}")
    axes = "[T, *batch, H, D]" if lead else "[*batch, H, D]"
    if nd < lead + 2:
        raise ValueError(f"q must be {axes}; got {list(q.shape)}")
    for name, t in (("k", k), ("v", v)):
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype} as q is; got {t.dtype}")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the others on {dev}")
    if k.shape != q.shape:
        raise ValueError(f"k must be {list(q.shape)} as q is; got {list(k.shape)}")
    if v.shape[:-1] != q.shape[:-1] or v.dim() != nd:
        raise ValueError(f"v must be {list(q.shape[:-1])} + [Dv]; got {list(v.shape)}")
    T = q.shape[0] if lead else 1
    batch, (H, dk), dv = q.shape[lead:-2], q.shape[-2:], v.shape[-1]
    if not (1 <= dk <= _MOST_DIM and 1 <= dv <= _MOST_DIM and 1 <= H <= _MOST_HEADS):
        raise ValueError(f"heads must be 1 to {_MOST_DIM} wide, one to {_MOST_HEADS} of them; got q "
                         f"{list(q.shape)}, v {list(v.shape)}")
    if batch.numel() * H >= 1 << 31:
        raise ValueError(f"at most 2^31 - 1 heads in all; got {batch.numel() * H}")
    log_decay = _same(log_decay, "log_decay", torch.Size((H,)), torch.float32, dev)
    if log_decay.requires_grad:
        raise ValueError("log_decay requires grad, but the decay is a constant: detach it")
    group = 1
    if starts is not None:
        n = max(starts.dim() - lead, 0)
        starts = _same(starts, "starts", torch.Size((*q.shape[:lead], *batch[:n])), torch.bool, dev)
        group = max(math.prod(batch[n:]), 1)
    scale = dk ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite; got {scale}")
    if forward_ad._current_level >= 0:
        _no_tangents(what, q, k, v, log_decay, state)
    return log_decay, starts, _lib.SwarpDecay(
        dtype=_CODES[dtype], heads=H, dk=dk, dv=dv, steps=T, batch=batch.numel(), group=group,
        scale=scale, log_decay=log_decay.data_ptr(), starts=_ptr(starts))


def _read(a: _lib.SwarpDecay, q, k, v, lead: int):
    """q, k and v into the arguments; what has to stay until the launch."""
    (q, a.q_stride), (k, a.k_stride), (v, a.v_stride) = (_laid(t, lead) for t in (q, k, v))
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    return q, k, v


def _work(a: _lib.SwarpDecay, dev):
    lib = _lib.load()
    n = lib.swarp_decay_work_bytes(ctypes.byref(a))
    work = torch.empty(n + 255, dtype=torch.uint8, device=dev)
    a.work, a.work_bytes = (work.data_ptr() + 255) // 256 * 256, n
    return lib, work


def _forward(a: _lib.SwarpDecay, q, k, v, state, stream: int):
    keep = _read(a, q, k, v, 1)
    batch = q.shape[1:-2]
    out = torch.empty((*q.shape[:-1], a.dv), dtype=q.dtype, device=q.device)
    after = torch.empty((*batch, a.heads, a.dk, a.dv), dtype=torch.float32, device=q.device)
    a.state, a.out, a.state_out = _ptr(state), out.data_ptr(), after.data_ptr()
    lib, work = _work(a, q.device)
    with _guard(q.device):
        _lib.check(lib.swarp_decay_fwd(ctypes.byref(a), stream))
    del keep, work
    return out, after


class _DecayFn(torch.autograd.Function):
    """The scan as one autograd node; the backward reads what autograd kept of its inputs."""

    @staticmethod
    def forward(ctx, a: _lib.SwarpDecay, stream: int, q, k, v, log_decay, state, starts):
        ctx.set_materialize_grads(False)
        ctx.a = a
        out, after = _forward(a, q, k, v, state, stream)
        ctx.save_for_backward(q, k, v, log_decay, state, starts)
        return out, after

    @staticmethod
    @_differentiable_once
    def backward(ctx, g_out, g_state):
        if g_out is None and g_state is None:
            return (None,) * 8
        q, k, v, log_decay, state, starts = ctx.saved_tensors
        a, dev = _lib.SwarpDecay.from_buffer_copy(ctx.a), q.device
        keep = _read(a, q, k, v, 1)
        log_decay = _plain(log_decay)
        state = None if state is None else _plain(state)
        starts = None if starts is None else starts.contiguous()
        g_out = _plain(g_out) if g_out is not None else torch.zeros(
            (*q.shape[:-1], a.dv), dtype=q.dtype, device=dev)
        g_state = None if g_state is None else _plain(g_state)
        d = [torch.empty(t.shape, dtype=q.dtype, device=dev) for t in (q, k, v)]
        d_state = None
        if state is not None and ctx.needs_input_grad[6]:
            d_state = torch.empty(state.shape, dtype=torch.float32, device=dev)
        a.log_decay, a.starts, a.state = log_decay.data_ptr(), _ptr(starts), _ptr(state)
        a.out = a.state_out = None
        a.adj_out, a.adj_state = g_out.data_ptr(), _ptr(g_state)
        (a.d_q, a.d_k, a.d_v), a.d_state = (t.data_ptr() for t in d), _ptr(d_state)
        lib, work = _work(a, dev)
        _lib.check(lib.swarp_decay_bwd(ctypes.byref(a), _lib.stream_of(dev)))
        del keep, work
        need = ctx.needs_input_grad
        return None, None, *(t if n else None for t, n in zip(d, need[2:5])), None, d_state, None


def decay_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
    state: torch.Tensor | None = None, starts: torch.Tensor | None = None, *,
    scale: float | None = None,
) -> DecayAttention:
    """Linear attention with a decay for each head along a rollout's steps: ``(out, state)``.

    ``q`` and ``k [T, *batch, H, Dk]``, ``v [T, *batch, H, Dv]`` (float32, bfloat16, float16; heads
    up to 128 wide; any strides over the steps, the batch and the heads, so the parts of one
    projection and ``x.movedim(1, 0)`` of a batch-first ``x`` are read where they lie),
    ``log_decay [H]`` (float32, not above 0), ``state [*batch, H, Dk, Dv]`` (float32) before the
    first step, or zero.  ``starts`` (bool) tells the steps that an episode starts with, and may
    leave out trailing batch axes: the ``terminated | truncated`` of the step before, ``[T, n_envs]``
    for ``q [T, n_envs, n_agents, H, Dk]``.

        S_t = (0 if starts_t else exp(log_decay) S_{t-1}) + k_t v_t^T;   out_t = scale q_t S_t

    ``scale`` is ``Dk ** -0.5`` unless given.  A start stops NaN and infinities as well, and a step
    does not look at later ones: what lies behind the end of a shorter sequence reaches only the
    outputs there and the state.  (A head with something that is not finite is done again step by
    step, some 0.7 us each: zeros behind the end are quicker.)  Sums and states are float32; with bfloat16 the products are of
    bfloat16 terms that carry 16 bits (24 in what enters the state).

    Gradients flow to ``q``, ``k``, ``v`` and ``state`` from both results, once, and backward only.
    """
    if is_dynamo_compiling():
        return _untraced(decay_attention)(q, k, v, log_decay, state, starts, scale=scale)
    log_decay, starts, a = _arguments("decay_attention", q, k, v, log_decay, state, starts, scale, 1)
    if state is not None:
        state = _same(state, "state", torch.Size((*q.shape[1:-1], a.dk, a.dv)), torch.float32,
                      q.device)
    stream = _lib.stream_of(q.device)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (
            state is not None and state.requires_grad)):
        return DecayAttention(*_DecayFn.apply(a, stream, q, k, v, log_decay, state, starts))
    return DecayAttention(*_forward(a, q, k, v, state, stream))


def decay_attention_step(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
    state: torch.Tensor, starts: torch.Tensor | None = None, *, scale: float | None = None,
) -> torch.Tensor:
    """One step of :func:`decay_attention`, for acting: ``out [*batch, H, Dv]``, with ``state``
    brought forward in place.

    ``q`` and ``k [*batch, H, Dk]``, ``v [*batch, H, Dv]``, ``state [*batch, H, Dk, Dv]`` (float32,
    contiguous), ``starts`` (bool, ``[*batch]`` or without trailing axes): which begin an episode
    with this step.  Not differentiable: call it under ``torch.no_grad()``, or with tensors that do
    not require grad.
    """
    if is_dynamo_compiling():
        return _untraced(decay_attention_step)(q, k, v, log_decay, state, starts, scale=scale)
    log_decay, starts, a = _arguments("decay_attention_step", q, k, v, log_decay, state, starts,
                                      scale, 0)
    shape = torch.Size((*q.shape[:-1], a.dk, a.dv))
    if (state.shape != shape or state.dtype != torch.float32 or state.device != q.device
            or not state.is_contiguous() or state.is_neg()):
        raise ValueError(f"state must be contiguous float32 {list(shape)} on {q.device}: it is "
                         f"changed in place; got {state.dtype} {list(state.shape)} on {state.device}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state)):
        raise RuntimeError("decay_attention_step is not differentiable: call it under "
                           "torch.no_grad(), or decay_attention with one step")
    keep = _read(a, q, k, v, 0)
    out = torch.empty((*q.shape[:-1], a.dv), dtype=q.dtype, device=q.device)
    a.state = a.state_out = state.data_ptr()
    a.out = out.data_ptr()
    with _guard(q.device):
        _lib.check(_lib.load().swarp_decay_step(ctypes.byref(a), _lib.stream_of(q.device)))
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    del keep
    return out
