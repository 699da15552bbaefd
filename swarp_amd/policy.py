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
import functools
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.compiler import is_dynamo_compiling

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
    kl: torch.Tensor             # mean of exp(q - logp) - 1 - (q - logp), q = ref_logp or old_logp
    clip_fraction: torch.Tensor  # share of counted decisions whose ratio the clip held


_HERE = contextlib.nullcontext()


def _guard(device: torch.device):
    """Makes ``device`` current for the launches inside, where it is not."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _HERE
    return torch.cuda.device(device)


def _on_gpu(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what}: swarp_amd computes on the HIP device only (no CPU fallback); "
                           f"got a tensor on {t.device}")


def _no_tangents(what: str, *tensors: torch.Tensor | None) -> None:
    """Refuses dual tensors, whose tangents the kernels would drop."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative; it is "
                                      "differentiated backward")


def _same(t: torch.Tensor, name: str, shape: torch.Size, dtype, device) -> torch.Tensor:
    """``t``, contiguous, after checking its shape, type and device."""
    if (t.shape == shape and t.dtype is dtype and t.device == device and t.is_contiguous()
            and (dtype is torch.bool or not t.is_neg())):
        return t
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}; got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}; got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the others on {device}")
    return _plain(t)


def _plain(t: torch.Tensor) -> torch.Tensor:
    """``t``, contiguous, with the values that its memory holds: a negated view (the imaginary part
    of a conjugate) reads the others' storage with its sign kept aside."""
    return (t.resolve_neg() if t.is_neg() else t).contiguous()


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


_UNTRACED: dict = {}


def _untraced(fn):
    """``fn`` as torch.compile leaves it alone, with all that it calls: the graph breaks there.
    (Made when it is first wanted: it imports the compiler.)"""
    if fn not in _UNTRACED:
        _UNTRACED[fn] = torch.compiler.disable(fn)
    return _UNTRACED[fn]


def _differentiable_once(backward):
    """``once_differentiable``, at no cost where no second derivative can be asked for."""
    guarded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


# ----------------------------------------------------------------------------- advantages


def _scan_args(rows, steps, columns, group, gamma, lam, rewards, values, final, term,
               trunc) -> _lib.SwarpGae:
    return _lib.SwarpGae(
        dtype=_CODES[rewards.dtype], rows=rows, steps=steps, columns=columns, group=group,
        gamma=gamma, lam=lam, rewards=rewards.data_ptr(), values=values.data_ptr(),
        terminated=_ptr(term), truncated=_ptr(trunc), final_values=_ptr(final))


def _gae_forward(a: _lib.SwarpGae, rewards: torch.Tensor, stream: int):
    adv, ret = torch.empty_like(rewards), torch.empty_like(rewards)
    a.advantages, a.returns = adv.data_ptr(), ret.data_ptr()
    with _guard(rewards.device):
        _lib.check(_lib.load().swarp_gae_fwd(ctypes.byref(a), stream))
    return adv, ret


class _GaeFn(torch.autograd.Function):
    """The scan as one autograd node; it is linear, so only the flags are kept.  autograd runs the
    backward with the forward's device and stream current."""

    @staticmethod
    def forward(ctx, a: _lib.SwarpGae, stream: int, rewards, values, final, term, trunc):
        ctx.set_materialize_grads(False)
        ctx.a, ctx.stream = a, stream
        ctx.like = (rewards.shape, values.shape, None if term is None else term.shape,
                    None if trunc is None else trunc.shape)
        ctx.save_for_backward(term, trunc)
        return _gae_forward(a, rewards, stream)

    @staticmethod
    @_differentiable_once
    def backward(ctx, g_adv, g_ret):
        if g_adv is None and g_ret is None:
            return (None,) * 7
        r_shape, v_shape, *flags = ctx.like
        if g_adv is not None:
            g_adv = _plain(g_adv)
        if g_ret is not None:
            g_ret = _plain(g_ret)
        ref = g_adv if g_adv is not None else g_ret
        need = ctx.needs_input_grad
        a = _lib.SwarpGae.from_buffer_copy(ctx.a)
        a.rewards = a.values = a.advantages = a.returns = None  # (read by the forward alone)
        # (unchanged since, or this raises; not the forward's memory where a hook packed them)
        term, trunc = ctx.saved_tensors
        if term is not None and not (term.data_ptr() == a.terminated and term.is_contiguous()):
            term = _same(term, "a saved tensor", flags[0], torch.bool, ref.device)
            a.terminated = term.data_ptr()
        if trunc is not None and not (trunc.data_ptr() == a.truncated and trunc.is_contiguous()):
            trunc = _same(trunc, "a saved tensor", flags[1], torch.bool, ref.device)
            a.truncated = trunc.data_ptr()
        d_r = ref.new_empty(r_shape) if need[2] else None
        d_v = ref.new_empty(v_shape) if need[3] else None
        d_f = ref.new_empty(r_shape) if a.final_values and need[4] else None
        if a.final_values:  # (only looked at for being set: an address that is alive)
            a.final_values = ref.data_ptr()
        a.adj_advantages, a.adj_returns = _ptr(g_adv), _ptr(g_ret)
        a.adj_rewards, a.adj_values, a.adj_final_values = _ptr(d_r), _ptr(d_v), _ptr(d_f)
        _lib.check(_lib.load().swarp_gae_bwd(ctypes.byref(a), ctx.stream))
        return None, None, d_r, d_v, d_f, None, None


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

    An end stops NaN and infinities as well, and nothing else does: ``0 * NaN`` is NaN with
    ``lam=0`` too.

    Gradients flow to ``rewards``, ``values`` and ``final_values`` (lambda-returns that are
    differentiated through a rollout), once, and backward only; detach them for the usual constant
    targets.
    """
    if is_dynamo_compiling():
        return _untraced(gae)(rewards, values, terminated, truncated, final_values, gamma=gamma,
                              lam=lam, time_dim=time_dim)
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
    shape = rewards.shape
    T, batch = (shape[-1], shape[:-1]) if last else (shape[0], shape[1:])

    def timed(steps, lead):
        return torch.Size((*lead, steps) if last else (steps, *lead))
    if not rewards.is_contiguous() or rewards.is_neg():
        rewards = _plain(rewards)
    values = _same(values, "values", timed(T + 1, batch), dtype, dev)
    if final_values is not None:
        final_values = _same(final_values, "final_values", shape, dtype, dev)
    if terminated is not None and truncated is not None and terminated.shape != truncated.shape:
        raise ValueError(f"terminated {list(terminated.shape)} and truncated "
                         f"{list(truncated.shape)} must have the same shape")
    group, flags = 1, [terminated, truncated]
    for n, name in enumerate(("terminated", "truncated")):
        if flags[n] is not None:
            k = max(flags[n].dim() - 1, 0)
            flags[n] = _same(flags[n], name, timed(T, batch[:k]), torch.bool, dev)
            group = math.prod(batch[k:])
    inputs = (rewards, values, final_values)
    if forward_ad._current_level >= 0:  # (a forward-mode derivative is being taken)
        _no_tangents("gae", *inputs)
    a = _scan_args(int(last), T, math.prod(batch), max(group, 1), gamma, lam, *inputs, *flags)
    stream = _lib.stream_of(dev)
    if torch.is_grad_enabled() and (rewards.requires_grad or values.requires_grad or (
            final_values is not None and final_values.requires_grad)):
        return Advantages(*_GaeFn.apply(a, stream, *inputs, *flags))
    return Advantages(*_gae_forward(a, rewards, stream))


# ------------------------------------------------------------------------- policy losses


@functools.lru_cache(maxsize=256)
def _work_bytes(lib, rows: int, width: int) -> int:
    return lib.swarp_policy_work_bytes(rows, width)


def _loss_forward(call, a: _lib.SwarpPolicy, head, old, stream: int):
    """(loss, stats, logp) of a call, and its work memory."""
    dev = head.device
    nbytes = _work_bytes(_lib.load(), a.rows, a.width)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    loss, stats, logp = old.new_empty(()), old.new_empty(3), torch.empty_like(old)
    a.logp, a.loss, a.stats = logp.data_ptr(), loss.data_ptr(), stats.data_ptr()
    a.work, a.work_bytes = work.data_ptr(), nbytes
    with _guard(dev):
        _lib.check(call(ctypes.byref(a), stream))
    return loss, stats, logp, work


def _buffers(head, log_std, need):
    """Gradient buffers of the heads that want one."""
    return (torch.empty_like(head, memory_format=torch.contiguous_format) if need[0] else None,
            torch.empty_like(log_std, memory_format=torch.contiguous_format) if need[1] else None)


def _unmoved(a: _lib.SwarpPolicy, strides, head, log_std, actions, old, adv, ref, mask) -> bool:
    """Whether saved tensors lie where and as the forward read them.  (Without a hook they do.  What
    a hook gives back has the values, size and type of what it took, but may be laid otherwise.
    Written out: this is on the path of every training step.)"""
    return (head.data_ptr() == a.head and head.stride() == strides and not head.is_neg()
            and old.data_ptr() == a.old_logp and old.is_contiguous() and not old.is_neg()
            and adv.data_ptr() == a.advantages and adv.is_contiguous() and not adv.is_neg()
            and actions.data_ptr() == a.actions and actions.is_contiguous() and not actions.is_neg()
            and (log_std is None or log_std.data_ptr() == a.log_std and log_std.is_contiguous()
                 and not log_std.is_neg())
            and (ref is None or ref.data_ptr() == a.ref_logp and ref.is_contiguous()
                 and not ref.is_neg())
            and (mask is None or mask.data_ptr() == a.mask and mask.is_contiguous()))


def _relocated(a: _lib.SwarpPolicy, like, head, log_std, actions, *rows):
    """A copy of a forward's arguments that reads saved tensors where they now lie, and all that has
    to stay until the launch."""
    shape, _, dtype, act = like
    dev, lead = rows[0].device, shape[:-1]
    if head.shape != shape or head.dtype != dtype or head.device != dev:
        raise RuntimeError(f"a saved head came back as {list(head.shape)} {head.dtype} on "
                           f"{head.device}; it was {list(shape)} {dtype} on {dev}")
    gaussian = log_std is not None
    strides = None if gaussian or head.is_neg() else _row_strides(head)
    if strides is None:
        head = _plain(head)
        strides = (1, 0, 0) if gaussian else _row_strides(head)
    if gaussian:
        log_std = _same(log_std, "a saved tensor", shape[-1:] if a.shared_std else shape, dtype, dev)
    wide = torch.float64 if dtype is torch.float64 else torch.float32
    rest = [t if t is None else _same(t, "a saved tensor", s, kind, dev) for t, s, kind in
            zip((actions, *rows), (shape if gaussian else lead, lead, lead, lead, lead),
                (act, wide, wide, wide, torch.bool))]
    a = _lib.SwarpPolicy.from_buffer_copy(a)
    a.inner, a.outer_stride, a.inner_stride = strides
    a.head, a.log_std = head.data_ptr(), _ptr(log_std)
    a.actions, a.old_logp, a.advantages, a.ref_logp, a.mask = (_ptr(t) for t in rest)
    return a, (head, log_std, rest)


class _LossFn(torch.autograd.Function):
    """A policy loss as one autograd node.

    The forward leaves the gradients for an upstream gradient of 1 behind, while a head's row is
    at hand: a training step then reads the heads once and writes their gradients once.  The
    backward hands them out; where the upstream gradient is not 1 (the device looks) it computes
    them again with it, so each is rounded once, from the tensors that autograd kept: under a
    checkpoint or a packing hook the forward's own are gone.  float16 gradients are left to the
    backward: without the loss scale that comes with it they would vanish.
    """

    @staticmethod
    def forward(ctx, calls, a: _lib.SwarpPolicy, stream: int, head, log_std, *rest):
        ctx.set_materialize_grads(False)
        ctx.call = (calls[1], a, stream)
        ctx.need = ctx.needs_input_grad[3:5]
        ctx.made = None
        if head.dtype != torch.float16:
            ctx.made = _buffers(head, log_std, ctx.need)
            a.d_head, a.d_log_std = _ptr(ctx.made[0]), _ptr(ctx.made[1])
        loss, stats, logp, ctx.work = _loss_forward(calls[0], a, head, rest[1], stream)
        ctx.like = head.shape, head.stride(), head.dtype, rest[0].dtype
        ctx.save_for_backward(head, log_std, *rest)
        ctx.mark_non_differentiable(stats, logp)
        return loss, stats, logp

    @staticmethod
    @_differentiable_once
    def backward(ctx, g, *_):
        if g is None:
            return (None,) * 10
        saved = ctx.saved_tensors  # (unchanged since, or this raises)
        call, a, stream = ctx.call
        keep = None
        if not _unmoved(a, ctx.like[1], *saved):
            a, keep = _relocated(a, ctx.like, *saved)
        if g.is_neg():
            g = g.resolve_neg()
        made, ctx.made = ctx.made, None  # handed out once: the caller may change them
        if made is None:
            d = _buffers(saved[0], saved[1], ctx.need)
            a = _lib.SwarpPolicy.from_buffer_copy(a)
            a.d_head, a.d_log_std = _ptr(d[0]), _ptr(d[1])
        else:
            d = made  # (where the forward's arguments say)
        # (autograd runs this with the forward's device and stream current)
        _lib.check(call(ctypes.byref(a), int(made is not None), g.data_ptr(), stream))
        return None, None, None, *d, None, None, None, None, None


def _clip_of(clip) -> tuple[float, float]:
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    if not (0.0 <= low <= 1.0 and 0.0 <= high < math.inf):
        raise ValueError(f"clip must be >= 0 (its lower bound at most 1); got {clip}")
    return float(low), float(high)


def _constant(t: torch.Tensor, name: str, shape, dtype, dev) -> torch.Tensor:
    t = _same(t, name, shape, dtype, dev)
    if t.requires_grad:
        raise ValueError(f"{name} requires grad, but the loss treats it as a constant: detach it")
    return t


def _per_row(lead, dtype, dev, old_logp, advantages, ref_logp, mask):
    """The per-decision inputs, checked."""
    old_logp = _constant(old_logp, "old_logp", lead, dtype, dev)
    advantages = _constant(advantages, "advantages", lead, dtype, dev)
    if ref_logp is not None:
        ref_logp = _constant(ref_logp, "ref_logp", lead, dtype, dev)
    if mask is not None:
        mask = _same(mask, "mask", lead, torch.bool, dev)
    return old_logp, advantages, ref_logp, mask


def _evaluate(gaussian: bool, width: int, strides, clip, coefs, head, log_std, actions, old, adv,
              ref, mask) -> PolicyLoss:
    if forward_ad._current_level >= 0:
        _no_tangents("the policy loss", head, log_std, actions, old, adv, ref)
    lib = _lib.load()
    stream = _lib.stream_of(head.device)
    (low, high), (kl_c, ent_c, total) = clip, coefs
    a = _lib.SwarpPolicy(
        dtype=_CODES[head.dtype], sum=total, width=width,
        actions32=actions.dtype == torch.int32,
        shared_std=gaussian and log_std.dim() == 1 and head.dim() > 1,
        rows=old.numel(), inner=strides[0], outer_stride=strides[1], inner_stride=strides[2],
        clip_low=low, clip_high=high, kl_coef=kl_c, entropy_coef=ent_c,
        head=head.data_ptr(), log_std=_ptr(log_std), actions=actions.data_ptr(),
        old_logp=old.data_ptr(), advantages=adv.data_ptr(), ref_logp=_ptr(ref), mask=_ptr(mask))
    calls = ((lib.swarp_gaussian_loss, lib.swarp_gaussian_loss_bwd) if gaussian else
             (lib.swarp_categorical_loss, lib.swarp_categorical_loss_bwd))
    if torch.is_grad_enabled() and (head.requires_grad
                                    or (gaussian and log_std.requires_grad)):
        loss, stats, logp = _LossFn.apply(calls, a, stream, head, log_std, actions, old, adv, ref,
                                          mask)
    else:
        loss, stats, logp = _loss_forward(calls[0], a, head, old, stream)[:3]
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
    if x.is_contiguous():
        return max(x.numel() // x.shape[-1], 1), 0, x.shape[-1]
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

    averaged (``"mean"``) or summed over the decisions that count.  The KL term estimates the
    divergence of this policy from the reference as far as the actions are this policy's; they are
    the old policy's, so with ``q = old_logp`` it agrees with either divergence of the two to second
    order in their difference, and is exact for neither.  ``clip`` is the bound on both
    sides, or ``(low, high)``.  Logits of -inf are actions that are not open.  What a masked
    decision holds is not looked at, its action included; with no decision that counts the loss
    and its gradients are 0.  An action that the reference forbids (``ref_logp`` of -inf) makes the
    KL term infinite, its gradient that of ``+kl_coef logp``.  A decision that counts with NaN or +inf among its logits, with all
    of them -inf, or with an action outside ``[0, V)`` makes the loss NaN.

    Gradients flow to ``logits`` alone (:class:`PolicyLoss`), once, and backward only.
    """
    if is_dynamo_compiling():
        return _untraced(categorical_policy_loss)(
            logits, actions, old_logp, advantages, ref_logp, mask, clip=clip, kl_coef=kl_coef,
            entropy_coef=entropy_coef, reduction=reduction)
    _on_gpu(logits, "categorical_policy_loss")
    if logits.dtype not in _CODES:
        raise TypeError(f"logits must be float32, float64, bfloat16 or float16; got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] < 1 << 31:
        raise ValueError(f"logits must be [*lead, V] with 1 <= V < 2^31; got {list(logits.shape)}")
    if actions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"actions must be int64 or int32; got {actions.dtype}")
    lead, dev = logits.shape[:-1], logits.device
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32
    actions = _same(actions, "actions", lead, actions.dtype, dev)
    rest = _per_row(lead, wide, dev, old_logp, advantages, ref_logp, mask)
    low_high = _clip_of(clip)
    coefs = _coefs(kl_coef, entropy_coef, reduction)
    strides = None if logits.is_neg() else _row_strides(logits)
    if strides is None:
        logits = _plain(logits)
        strides = _row_strides(logits)
    return _evaluate(False, logits.shape[-1], strides, low_high, coefs, logits, None, actions, *rest)


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
    if is_dynamo_compiling():
        return _untraced(gaussian_policy_loss)(
            mean, log_std, actions, old_logp, advantages, ref_logp, mask, clip=clip,
            kl_coef=kl_coef, entropy_coef=entropy_coef, reduction=reduction)
    _on_gpu(mean, "gaussian_policy_loss")
    if mean.dtype not in _CODES:
        raise TypeError(f"mean must be float32, float64, bfloat16 or float16; got {mean.dtype}")
    if mean.dim() < 1 or not 1 <= mean.shape[-1] <= 64:
        raise ValueError(f"mean must be [*lead, D] with 1 <= D <= 64; got {list(mean.shape)}")
    D, lead, dev = mean.shape[-1], mean.shape[:-1], mean.device
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
    actions = _constant(actions, "actions", mean.shape, wide, dev)
    rest = _per_row(lead, wide, dev, old_logp, advantages, ref_logp, mask)
    coefs = _coefs(kl_coef, entropy_coef, reduction)
    return _evaluate(True, D, (1, 0, 0), _clip_of(clip), coefs, _plain(mean),
                     _plain(log_std), actions, *rest)
