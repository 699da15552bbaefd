"""The loss of imitation, and the log-probabilities of a wide head: softmax cross entropy of a linear
head over action bins or the tokens of a vocabulary, computed from the hidden states and the head's
weight by hand-written kernels that never hold the logits of all decisions.

In the manner of the policy losses: HIP tensors only, every launch on torch's current stream, shapes
and types checked before any launch, no host synchronisation.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.compiler import is_dynamo_compiling

from . import _lib
from .policy import (_CODES, _capture_of, _differentiable_once, _guard, _no_tangents, _on_gpu,
                     _plain, _ptr, _row_strides, _same, _untraced)

_MOST_DIM, _MOST_WIDTH = 65536, 1 << 21
_TYPES = {code: dtype for dtype, code in _CODES.items()}


class LinearCrossEntropy(NamedTuple):
    """Result of :func:`linear_cross_entropy`.  Gradients flow from ``loss`` only."""

    loss: torch.Tensor  # scalar, float32
    logp: torch.Tensor  # log-probability of each target (0 where masked), float32


def _call(a: _lib.SwarpLinearCe, dev, lead, shapes, complete: bool, stream: int):
    """The call: (loss, logp), the gradients that it leaves (of these shapes, or None), where their rows
    lie, its work memory."""
    loss = torch.empty((), dtype=torch.float32, device=dev)
    logp = torch.empty(lead, dtype=torch.float32, device=dev)
    kind = _TYPES[a.dtype] if complete else torch.float32
    grads = [s if s is None else torch.empty(s, dtype=kind, device=dev) for s in shapes]
    place = None
    if a.mask and not complete:
        place = torch.empty(a.rows + 1, dtype=torch.int32, device=dev)
        a.place = place.data_ptr()
    a.loss, a.logp = loss.data_ptr(), logp.data_ptr()
    a.d_hidden, a.d_weight, a.d_bias = map(_ptr, grads)
    lib = _lib.load()
    nbytes = lib.swarp_linear_ce_work_bytes(ctypes.byref(a))
    work = torch.empty(nbytes + 255, dtype=torch.uint8, device=dev)
    a.work, a.work_bytes = (work.data_ptr() + 255) // 256 * 256, nbytes
    with _guard(dev):
        _lib.check(lib.swarp_linear_ce(ctypes.byref(a), stream))
    return loss, logp, grads, place, work


def _unmoved(a: _lib.SwarpLinearCe, strides, hidden, weight, bias, targets, mask) -> bool:
    """Whether saved tensors lie where and as the forward read them (written out: this is on the path
    of every training step)."""
    return (hidden.data_ptr() == a.hidden and hidden.stride() == strides and not hidden.is_neg()
            and weight.data_ptr() == a.weight and weight.is_contiguous() and not weight.is_neg()
            and targets.data_ptr() == a.targets and targets.is_contiguous()
            and (bias is None or bias.data_ptr() == a.bias and bias.is_contiguous()
                 and not bias.is_neg())
            and (mask is None or mask.data_ptr() == a.mask and mask.is_contiguous()))


class _LinearCeFn(torch.autograd.Function):
    """The loss as one autograd node.  The forward leaves gradients for an upstream gradient of 1
    behind, while the exponentials are at hand.

    16-bit ones of a wide head are kept in float32, and the backward multiplies them by the upstream
    gradient and rounds them, once.  The others are handed out, once; where the upstream gradient is
    not 1 (the device looks) those of a wide head are multiplied by it and those of a narrow one
    computed again with it.  float16 ones of a narrow head are left to the backward: without the loss
    scale that comes with it they would vanish.  A second backward computes them again, and so does
    one that is captured into a graph without its forward."""

    @staticmethod
    def forward(ctx, a: _lib.SwarpLinearCe, stream: int, complete: bool, hidden, weight, bias,
                targets, mask):
        ctx.set_materialize_grads(False)
        need = ctx.needs_input_grad
        ctx.shapes = tuple(t.shape if n else None for t, n in zip((hidden, weight, bias), need[3:6]))
        late = complete and hidden.dtype == torch.float16
        loss, logp, grads, place, work = _call(a, hidden.device, targets.shape,
                                               (None,) * 3 if late else ctx.shapes, complete, stream)
        ctx.a, ctx.stream, ctx.complete = a, stream, complete
        ctx.like = hidden.stride(), hidden.dtype
        ctx.kept = not complete and hidden.dtype != torch.float32
        if ctx.kept:
            ctx.save_for_backward(*grads, place)
        else:
            ctx.made = None if late else (grads, place)
            ctx.capture = _capture_of(hidden, stream)
            ctx.work = work if complete else None
            ctx.save_for_backward(hidden, weight, bias, targets, mask)
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @_differentiable_once
    def backward(ctx, g, *_):
        if g is None:
            return (None,) * 8
        saved = ctx.saved_tensors  # (unchanged since, or this raises)
        a, first, keep = ctx.a, 0, None
        if g.is_neg():
            g = g.resolve_neg()
        # (autograd runs this with the forward's device and stream current)
        if ctx.kept:
            # (they may have been packed and lie elsewhere by now)
            *out, place = saved = [t if t is None else _plain(t) for t in saved]
            a = _lib.SwarpLinearCe.from_buffer_copy(a)
            a.d_hidden, a.d_weight, a.d_bias, a.place = map(_ptr, saved)
            out = [t if t is None else torch.empty(t.shape, dtype=ctx.like[1], device=g.device)
                   for t in out]
        else:
            made, ctx.made = ctx.made, None  # handed out once: the caller may change them
            if made is not None and ctx.capture != _capture_of(saved[0], ctx.stream):
                made = None  # (a graph's replays find them changed, with no forward to leave new ones)
            if not _unmoved(a, ctx.like[0], *saved):
                a = _lib.SwarpLinearCe.from_buffer_copy(a)
                keep = _point(a, *saved)
            if made is not None:
                first, (out, place) = 1, made
            elif ctx.complete:
                place = None
                out = [s if s is None else torch.empty(s, dtype=ctx.like[1], device=g.device)
                       for s in ctx.shapes]
            else:
                a = _lib.SwarpLinearCe.from_buffer_copy(a)
                out, place, work = _call(a, g.device, saved[3].shape, ctx.shapes, False,
                                         ctx.stream)[2:]
                keep = keep, work
            if place is not None and out[0] is not None:  # (its rows lie together)
                out = [torch.empty(ctx.shapes[0], dtype=ctx.like[1], device=g.device), *out[1:]]
        _lib.check(_lib.load().swarp_linear_ce_bwd(ctypes.byref(a), first, g.data_ptr(),
                                                   *map(_ptr, out), ctx.stream))
        del keep
        return None, None, None, *out, None, None


def _point(a: _lib.SwarpLinearCe, hidden, weight, bias, targets, mask):
    """The inputs into the arguments, wherever they lie; what has to stay until the launch."""
    strides = None if hidden.is_neg() else _row_strides(hidden)
    if strides is None:
        hidden = _plain(hidden)
        strides = _row_strides(hidden)
    weight, targets = _plain(weight), _plain(targets)
    bias = None if bias is None else _plain(bias)
    mask = None if mask is None else mask.contiguous()
    a.inner, a.outer_stride, a.inner_stride = strides
    a.hidden, a.weight, a.bias = hidden.data_ptr(), weight.data_ptr(), _ptr(bias)
    a.targets, a.mask = targets.data_ptr(), _ptr(mask)
    return hidden, weight, bias, targets, mask


def linear_cross_entropy(
    hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
    bias: torch.Tensor | None = None, mask: torch.Tensor | None = None, *,
    reduction: str = "mean",
) -> LinearCrossEntropy:
    """Softmax cross entropy of the head ``hidden @ weight.T + bias`` with ``targets``: the loss of
    imitating recorded actions or tokens, with its gradient, and the targets' log-probabilities,
    which under ``torch.no_grad()`` are what :func:`categorical_policy_loss` takes as ``old_logp``
    or ``ref_logp``.  The logits of all decisions are never in memory.

    ``hidden [*lead, D]`` (float32, bfloat16, float16; any strides over ``lead``, so a sequence
    model's ``hidden[:, :-1]`` is read where it lies), ``weight [V, D]`` and ``bias [V]`` of the same
    type, ``targets [*lead]`` (int64 or int32), ``mask [*lead]`` (bool: which decisions count).
    ``D`` up to 65536, ``V`` up to 2^21.

        logp = z[target] - log sum exp z,   loss = -mean (or sum) of logp over what counts

    Products and sums are in float32, whatever the type; what comes of exponentials goes into the
    gradients' products in the type of ``hidden`` (of narrow heads, up to 32 columns of 128 or 64 of 64,
    with 16 bits at least).  What a masked decision holds is not looked at, its target included
    (-100); with no decision that counts the loss and its gradients are 0.  A bias of -inf is an
    action that is not open.  A decision that counts with NaN or +inf among its logits, with all of
    them -inf, or with a target outside ``[0, V)`` makes the loss NaN.

    Gradients flow to ``hidden``, ``weight`` and ``bias``, once, and backward only.  A loss with
    float16 heads should be scaled, as mixed precision does.  A wide head's call needs work memory:
    copies of ``hidden`` and of a ``weight`` whose rows are not whole 16 bytes, 60 bytes a decision and
    up to 1 GiB; where gradients are wanted 2.1 times the exponentials of 1 GiB of rows (or of 256
    rows), 128 bytes a column and 0.13 GiB, and float32 buffers for them until the backward.
    """
    if is_dynamo_compiling():
        return _untraced(linear_cross_entropy)(hidden, weight, targets, bias, mask,
                                               reduction=reduction)
    _on_gpu(hidden, "linear_cross_entropy")
    dtype, dev = hidden.dtype, hidden.device
    if dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"hidden must be float32, bfloat16 or float16; got {dtype}")
    if hidden.dim() < 1 or not 1 <= hidden.shape[-1] <= _MOST_DIM:
        raise ValueError(f"hidden must be [*lead, D] with 1 <= D <= {_MOST_DIM}; got "
                         f"{list(hidden.shape)}")
    D, lead = hidden.shape[-1], hidden.shape[:-1]
    if weight.dim() != 2 or weight.shape[1] != D or not 1 <= weight.shape[0] <= _MOST_WIDTH:
        raise ValueError(f"weight must be [V, {D}] with 1 <= V <= {_MOST_WIDTH}; got "
                         f"{list(weight.shape)}")
    V = weight.shape[0]
    if lead.numel() >= 1 << 31:
        raise ValueError(f"at most 2^31 - 1 decisions; got {lead.numel()}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32; got {targets.dtype}")
    if reduction not in ("mean", "sum"):
        raise ValueError(f'reduction must be "mean" or "sum"; got {reduction!r}')
    weight = _same(weight, "weight", torch.Size((V, D)), dtype, dev)
    targets = _same(targets, "targets", lead, targets.dtype, dev)
    if bias is not None:
        bias = _same(bias, "bias", torch.Size((V,)), dtype, dev)
    if mask is not None:
        mask = _same(mask, "mask", lead, torch.bool, dev)
    if forward_ad._current_level >= 0:
        _no_tangents("linear_cross_entropy", hidden, weight, bias)
    a = _lib.SwarpLinearCe(
        dtype=_CODES[dtype], sum=reduction == "sum", targets32=targets.dtype == torch.int32,
        dim=D, width=V, rows=targets.numel())
    keep = _point(a, hidden, weight, bias, targets, mask)
    stream = _lib.stream_of(dev)
    complete = bool(_lib.load().swarp_linear_ce_complete(ctypes.byref(a)))
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or (
            bias is not None and bias.requires_grad)):
        return LinearCrossEntropy(*_LinearCeFn.apply(a, stream, complete, hidden, weight, bias,
                                                     targets, mask))
    loss, logp = _call(a, dev, lead, (None,) * 3, complete, stream)[:2]
    del keep
    return LinearCrossEntropy(loss, logp)
