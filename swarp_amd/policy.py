"""What a policy is trained with on the environments of this package: advantages of a rollout
(:func:`gae`) and the clipped policy loss with KL and entropy terms of a categorical or a
Gaussian head (:func:`categorical_policy_loss`, :func:`gaussian_policy_loss`), each a hand-written
kernel with its adjoint behind ``torch.autograd``.

The reference trains with torch operations (its ``swarp/rl`` package); these are this package's
own operators, in its manner: HIP tensors only, every launch on torch's current stream, shapes
and types checked before any launch, no host synchronisation.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_CODES = {torch.float32: _lib.F32, torch.float64: _lib.F64, torch.bfloat16: _lib.BF16,
          torch.float16: _lib.F16}


class Advantages(NamedTuple):
    """Result of :func:`gae`."""

    advantages: torch.Tensor
    returns: torch.Tensor


class PolicyLoss(NamedTuple):
    """Result of a policy loss.  Gradients flow from ``loss`` only; the others are for logging."""

    loss: torch.Tensor           # scalar
    logp: torch.Tensor           # log-probability of each action taken (0 where masked)
    entropy: torch.Tensor        # mean entropy of the counted decisions
    kl: torch.Tensor             # mean of exp(q - logp) - 1 - (q - logp), q the reference's
    clip_fraction: torch.Tensor  # share of counted decisions whose ratio the clip held


def _guard(device: torch.device):
    """Makes ``device`` current for the launches inside, where it is not."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _on_gpu(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what}: swarp_amd computes on the HIP device only (no CPU fallback); "
                           f"got a tensor on {t.device}")


def _same(t: torch.Tensor, name: str, shape, dtype, device) -> torch.Tensor:
    """``t``, contiguous, after checking its shape, type and device."""
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}; got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}; got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the others on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


# ----------------------------------------------------------------------------- advantages


class _Scan(NamedTuple):
    rows: int
    steps: int
    columns: int
    group: int
    gamma: float
    lam: float


def _scan_args(scan: _Scan, dtype, rewards, values, term, trunc, final) -> _lib.SwarpGae:
    return _lib.SwarpGae(
        dtype=_CODES[dtype], rows=scan.rows, steps=scan.steps, columns=scan.columns,
        group=scan.group, gamma=scan.gamma, lam=scan.lam, rewards=_ptr(rewards),
        values=_ptr(values), terminated=_ptr(term), truncated=_ptr(trunc),
        final_values=_ptr(final))


def _gae_forward(scan: _Scan, rewards, values, final, term, trunc):
    adv, ret = torch.empty_like(rewards), torch.empty_like(rewards)
    a = _scan_args(scan, rewards.dtype, rewards, values, term, trunc, final)
    a.advantages, a.returns = adv.data_ptr(), ret.data_ptr()
    with _guard(rewards.device):
        _lib.check(_lib.load().swarp_gae_fwd(ctypes.byref(a), _lib.stream_of(rewards.device)))
    return adv, ret


class _GaeFn(torch.autograd.Function):
    """The scan as one autograd node; it is linear, so only the flags are kept."""

    @staticmethod
    def forward(ctx, scan: _Scan, rewards, values, final, term, trunc):
        ctx.set_materialize_grads(False)
        ctx.scan = scan
        ctx.final = final is not None
        ctx.like = (rewards.shape, values.shape)
        ctx.save_for_backward(term, trunc)
        return _gae_forward(scan, rewards, values, final, term, trunc)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_adv, g_ret):
        if g_adv is None and g_ret is None:
            return (None,) * 6
        term, trunc = ctx.saved_tensors
        g_adv, g_ret = (None if g is None else g.contiguous() for g in (g_adv, g_ret))
        ref = g_adv if g_adv is not None else g_ret
        need = ctx.needs_input_grad
        d_r = ref.new_empty(ctx.like[0]) if need[1] else None
        d_v = ref.new_empty(ctx.like[1]) if need[2] else None
        d_f = ref.new_empty(ctx.like[0]) if ctx.final and need[3] else None
        # a final-value buffer is only looked at for being there: the adjoint reads no values
        a = _scan_args(ctx.scan, ref.dtype, None, None, term, trunc, ref if ctx.final else None)
        a.adj_advantages, a.adj_returns = _ptr(g_adv), _ptr(g_ret)
        a.adj_rewards, a.adj_values, a.adj_final_values = _ptr(d_r), _ptr(d_v), _ptr(d_f)
        with _guard(ref.device):
            _lib.check(_lib.load().swarp_gae_bwd(ctypes.byref(a), _lib.stream_of(ref.device)))
        return None, d_r, d_v, d_f, None, None


def gae(rewards: torch.Tensor, values: torch.Tensor, terminated: torch.Tensor | None = None,
        truncated: torch.Tensor | None = None, final_values: torch.Tensor | None = None, *,
        gamma: float = 0.99, lam: float = 0.95, time_dim: int = 0) -> Advantages:
    """Generalised advantage estimation of a rollout: ``(advantages, returns)``, both like
    ``rewards``.

    ``rewards [T, *batch]`` and ``values [T + 1, *batch]`` (the last is the bootstrap), float32 or
    float64; with ``time_dim=-1`` time is the last axis instead.  ``terminated`` and ``truncated``
    (bool) end an episode after a step; they may leave out trailing batch axes -- ``Environment``
    gives ``[T, n_envs]`` for rewards ``[T, n_envs, n_agents]``.  A terminated step bootstraps
    nothing.  A truncated one bootstraps ``final_values`` (like ``rewards``: the value of the
    observation the episode ended in, which an auto-reset has replaced) or, without it,
    ``values`` of the next step.  Values that no step reads may be anything, NaN included.

        delta_t = r_t + gamma next_t - V_t;   A_t = delta_t + gamma lam A_{t+1} (0 across an end)

    Gradients flow to ``rewards``, ``values`` and ``final_values`` (lambda-returns that are
    differentiated through a rollout); detach them for the usual constant targets.
    """
    _on_gpu(rewards, "gae")
    dtype, dev, nd = rewards.dtype, rewards.device, rewards.dim()
    if dtype not in (torch.float32, torch.float64):
        raise TypeError(f"gae takes float32 or float64; got {dtype}")
    if nd < 1:
        raise ValueError("rewards must have a time axis")
    if time_dim not in (0, -1, nd - 1):
        raise ValueError(f"time_dim must be 0 or -1 (the first or the last axis); got {time_dim}")
    if not (0.0 <= gamma <= 1.0 and 0.0 <= lam <= 1.0):
        raise ValueError(f"gamma and lam must lie in [0, 1]; got {gamma} and {lam}")
    last = time_dim != 0 and nd > 1
    shape = tuple(rewards.shape)
    T, batch = (shape[-1], shape[:-1]) if last else (shape[0], shape[1:])
    rewards = _same(rewards, "rewards", shape, dtype, dev)
    values = _same(values, "values", (*batch, T + 1) if last else (T + 1, *batch), dtype, dev)
    if final_values is not None:
        final_values = _same(final_values, "final_values", shape, dtype, dev)
    if terminated is not None and truncated is not None and terminated.shape != truncated.shape:
        raise ValueError(f"terminated {list(terminated.shape)} and truncated "
                         f"{list(truncated.shape)} must have the same shape")
    group, flags = 1, [terminated, truncated]
    for n, name in enumerate(("terminated", "truncated")):
        if flags[n] is not None:
            k = max(flags[n].dim() - 1, 0)
            lead = batch[:k]
            flags[n] = _same(flags[n], name, (*lead, T) if last else (T, *lead), torch.bool, dev)
            group = math.prod(batch[k:])
    scan = _Scan(int(last), T, math.prod(batch), max(group, 1), float(gamma), float(lam))
    inputs = (rewards, values, final_values)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs):
        return Advantages(*_GaeFn.apply(scan, *inputs, *flags))
    return Advantages(*_gae_forward(scan, *inputs, *flags))


# ------------------------------------------------------------------------- policy losses


class _Loss(NamedTuple):
    """The constants of a call (everything that is not a tensor)."""

    gaussian: bool
    rows: int
    width: int
    strides: tuple[int, int, int]
    clip: tuple[float, float]
    kl_coef: float
    entropy_coef: float
    sum: bool


def _loss_args(c: _Loss, head, log_std, actions, old, adv, ref, mask):
    """The C arguments of a call, without its results, and the work memory they point to."""
    nbytes = _lib.load().swarp_policy_work_bytes(c.rows, c.width)
    work = torch.empty(nbytes, dtype=torch.uint8, device=head.device)
    a = _lib.SwarpPolicy(
        dtype=_CODES[head.dtype], sum=c.sum, width=c.width,
        actions32=actions.dtype == torch.int32,
        shared_std=log_std is not None and log_std.dim() == 1 and head.dim() > 1,
        rows=c.rows, inner=c.strides[0], outer_stride=c.strides[1], inner_stride=c.strides[2],
        clip_low=c.clip[0], clip_high=c.clip[1], kl_coef=c.kl_coef, entropy_coef=c.entropy_coef,
        head=head.data_ptr(), log_std=_ptr(log_std), actions=actions.data_ptr(),
        old_logp=old.data_ptr(), advantages=adv.data_ptr(), ref_logp=_ptr(ref), mask=_ptr(mask),
        work=work.data_ptr(), work_bytes=nbytes)
    return a, work


def _loss_launch(c: _Loss, a: _lib.SwarpPolicy, dev) -> None:
    lib = _lib.load()
    call = lib.swarp_gaussian_loss if c.gaussian else lib.swarp_categorical_loss
    with _guard(dev):
        _lib.check(call(ctypes.byref(a), _lib.stream_of(dev)))


def _loss_forward(c: _Loss, head, log_std, rest, made=(None, None)):
    """(loss, stats, logp) of a call, its arguments and its work memory; ``made`` are gradient
    buffers to fill on the way."""
    a, work = _loss_args(c, head, log_std, *rest)
    old = rest[1]
    loss, stats, logp = old.new_empty(()), old.new_empty(3), torch.empty_like(old)
    a.logp, a.loss, a.stats = logp.data_ptr(), loss.data_ptr(), stats.data_ptr()
    a.d_head, a.d_log_std = _ptr(made[0]), _ptr(made[1])
    _loss_launch(c, a, head.device)
    return loss, stats, logp, a, work


def _buffers(head, log_std, need):
    """Gradient buffers of the heads that want one."""
    return (torch.empty(head.shape, dtype=head.dtype, device=head.device) if need[0] else None,
            torch.empty_like(log_std) if log_std is not None and need[1] else None)


class _LossFn(torch.autograd.Function):
    """A policy loss as one autograd node.

    The forward leaves the gradients for an upstream gradient of 1 behind, while a head's row is
    at hand: a training step then reads the heads once and writes their gradients once.  The
    backward hands them out; where the upstream gradient is not 1 (the device looks) it computes
    them again with it, so each is rounded once.  float16 gradients are left to the backward:
    without the loss scale that comes with it they would vanish.
    """

    @staticmethod
    def forward(ctx, c: _Loss, head, log_std, *rest):
        ctx.set_materialize_grads(False)
        ctx.c = c
        ctx.need = ctx.needs_input_grad[1:3]
        ctx.made = None
        if head.dtype != torch.float16:
            ctx.made = _buffers(head, log_std, ctx.need)
        loss, stats, logp, *ctx.call = _loss_forward(c, head, log_std, rest,
                                                     ctx.made or (None, None))
        ctx.save_for_backward(head, log_std, *rest)
        ctx.mark_non_differentiable(stats, logp)
        return loss, stats, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        if g is None:
            return (None,) * 8
        head, log_std = ctx.saved_tensors[:2]  # (unchanged since, or this raises)
        made, ctx.made = ctx.made, None  # handed out once: the caller may change them
        d = made or _buffers(head, log_std, ctx.need)
        a = ctx.call[0]
        a.logp = a.loss = a.stats = None
        a.d_head, a.d_log_std, a.scale = _ptr(d[0]), _ptr(d[1]), g.data_ptr()
        a.skip_unit, a.counted = made is not None, 1
        _loss_launch(ctx.c, a, head.device)
        return None, *d, *(None,) * 5


def _clip_of(clip) -> tuple[float, float]:
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    if not (0.0 <= low <= 1.0 and 0.0 <= high < math.inf):
        raise ValueError(f"clip must be >= 0 (its lower bound at most 1); got {clip}")
    return float(low), float(high)


def _per_row(lead, dtype, dev, old_logp, advantages, ref_logp, mask):
    """The per-decision inputs, checked."""
    out = []
    for name, t in (("old_logp", old_logp), ("advantages", advantages), ("ref_logp", ref_logp)):
        if t is not None:
            t = _same(t, name, lead, dtype, dev)
            if t.requires_grad:
                raise ValueError(f"{name} requires grad, but the loss treats it as a constant: "
                                 "detach it")
        out.append(t)
    if mask is not None:
        mask = _same(mask, "mask", lead, torch.bool, dev)
    return (*out, mask)


def _evaluate(c: _Loss, head, log_std, *rest) -> PolicyLoss:
    if torch.is_grad_enabled() and (head.requires_grad
                                    or (log_std is not None and log_std.requires_grad)):
        loss, stats, logp = _LossFn.apply(c, head, log_std, *rest)
    else:
        loss, stats, logp = _loss_forward(c, head, log_std, rest)[:3]
    return PolicyLoss(loss, logp, *stats.unbind(0))


def _coefs(kl_coef, entropy_coef, reduction):
    if not (math.isfinite(kl_coef) and math.isfinite(entropy_coef)):
        raise ValueError("kl_coef and entropy_coef must be finite")
    if reduction not in ("mean", "sum"):
        raise ValueError(f'reduction must be "mean" or "sum"; got {reduction!r}')
    return float(kl_coef), float(entropy_coef), reduction == "sum"


def _row_strides(x: torch.Tensor):
    """(inner, outer stride, inner stride) of the rows of ``x [*lead, V]``, or None where two
    levels of strides do not reach them."""
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        return None
    dims: list[list[int]] = []  # [size, stride], outermost first, neighbours merged
    for n, st in zip(x.shape[:-1], x.stride()[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * st:
            dims[-1] = [dims[-1][0] * n, st]
        else:
            dims.append([n, st])
    if len(dims) > 2:
        return None
    if not dims:
        return 1, 0, 0
    if len(dims) == 1:
        return dims[0][0], 0, dims[0][1]
    return dims[1][0], dims[0][1], dims[1][1]


def categorical_policy_loss(
    logits: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
    ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None, *,
    clip: float | tuple[float, float] = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
    reduction: str = "mean",
) -> PolicyLoss:
    """The clipped policy loss of a categorical head -- action bins of an agent, or tokens of a
    vocabulary -- with a KL term towards a reference policy and an entropy bonus.

    ``logits [*lead, V]`` (float32, float64, bfloat16, float16; any strides over ``lead``, so the
    slice ``logits[:, :-1]`` of a sequence model is read where it lies), ``actions`` (int64 or
    int32), ``old_logp``, ``advantages`` and ``ref_logp`` ``[*lead]`` (float32; float64 with
    float64 logits), ``mask [*lead]`` (bool: which decisions count).  Per decision, with
    ``ratio = exp(logp - old_logp)`` and ``q = ref_logp`` (``old_logp`` without it):

        -min(ratio A, clamp(ratio, 1 - low, 1 + high) A)
            + kl_coef (exp(q - logp) - 1 - (q - logp)) - entropy_coef H

    averaged (``"mean"``) or summed over the decisions that count.  ``clip`` is the bound on both
    sides, or ``(low, high)``.  Logits of -inf are actions that are not open.  What a masked
    decision holds is not looked at, its action included; with no decision that counts the loss
    and its gradients are 0.  A decision that counts with NaN or +inf among its logits, with all
    of them -inf, or with an action outside ``[0, V)`` makes the loss NaN.

    Gradients flow to ``logits`` alone (:class:`PolicyLoss`).
    """
    _on_gpu(logits, "categorical_policy_loss")
    if logits.dtype not in _CODES:
        raise TypeError(f"logits must be float32, float64, bfloat16 or float16; got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [*lead, V] with V >= 1; got {list(logits.shape)}")
    if actions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"actions must be int64 or int32; got {actions.dtype}")
    lead, dev = tuple(logits.shape[:-1]), logits.device
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32
    actions = _same(actions, "actions", lead, actions.dtype, dev)
    rest = _per_row(lead, wide, dev, old_logp, advantages, ref_logp, mask)
    low_high = _clip_of(clip)
    kl_c, ent_c, total = _coefs(kl_coef, entropy_coef, reduction)
    strides = _row_strides(logits)
    if strides is None:
        logits = logits.contiguous()
        strides = _row_strides(logits)
    c = _Loss(False, math.prod(lead), logits.shape[-1], strides, low_high, kl_c, ent_c, total)
    return _evaluate(c, logits, None, actions, *rest)


def gaussian_policy_loss(
    mean: torch.Tensor, log_std: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor,
    advantages: torch.Tensor, ref_logp: torch.Tensor | None = None,
    mask: torch.Tensor | None = None, *, clip: float | tuple[float, float] = 0.2,
    kl_coef: float = 0.0, entropy_coef: float = 0.0, reduction: str = "mean",
) -> PolicyLoss:
    """The loss of :func:`categorical_policy_loss` for a diagonal Gaussian head over continuous
    actions (an agent's accelerations, a quadrotor's thrusts).

    ``mean [*lead, D]`` (float32, float64, bfloat16, float16), ``log_std`` of the same type,
    ``[D]`` (one per dimension, whose gradient is summed over the decisions in a fixed order) or
    anything that broadcasts to ``mean``; ``actions [*lead, D]``, ``old_logp``, ``advantages``,
    ``ref_logp`` float32 (float64 with a float64 head); ``D <= 64``.  ``logp`` and the entropy are
    sums over the dimensions.  Gradients flow to ``mean`` and ``log_std``.
    """
    _on_gpu(mean, "gaussian_policy_loss")
    if mean.dtype not in _CODES:
        raise TypeError(f"mean must be float32, float64, bfloat16 or float16; got {mean.dtype}")
    if mean.dim() < 1 or not 1 <= mean.shape[-1] <= 64:
        raise ValueError(f"mean must be [*lead, D] with 1 <= D <= 64; got {list(mean.shape)}")
    D, lead, dev = mean.shape[-1], tuple(mean.shape[:-1]), mean.device
    if log_std.dtype != mean.dtype:
        raise TypeError(f"log_std must be {mean.dtype} as mean is; got {log_std.dtype}")
    if log_std.device != dev:
        raise ValueError(f"log_std is on {log_std.device}, the others on {dev}")
    if tuple(log_std.shape) != (D,):
        try:
            log_std = log_std.expand(mean.shape)
        except RuntimeError:
            raise ValueError(f"log_std {list(log_std.shape)} does not broadcast to mean "
                             f"{list(mean.shape)}") from None
    wide = torch.float64 if mean.dtype == torch.float64 else torch.float32
    actions = _same(actions, "actions", mean.shape, wide, dev)
    if actions.requires_grad:
        raise ValueError("actions requires grad, but the loss treats it as a constant: detach it")
    rest = _per_row(lead, wide, dev, old_logp, advantages, ref_logp, mask)
    kl_c, ent_c, total = _coefs(kl_coef, entropy_coef, reduction)
    c = _Loss(True, math.prod(lead), D, (1, 0, 0), _clip_of(clip), kl_c, ent_c, total)
    return _evaluate(c, mean.contiguous(), log_std.contiguous(), actions, *rest)
