"""AdamW over all tensors of a policy at once, with moments in 32 or 8 bits.

:func:`adamw_step` is the step on given tensors, :class:`AdamW` the ``torch.optim`` optimizer
around it; :func:`grad_norm` is the norm of all gradients, with the scale that clips it, left on
the device.  The moments of all parameters lie in one flat state (:class:`AdamWState`), each
tensor's at a multiple of 256 elements, so that a step is one launch over up to 64 tensors.
"""

from __future__ import annotations

import ctypes
import operator
import struct
from typing import Iterable, NamedTuple, Sequence

import torch
from torch.compiler import is_dynamo_compiling

from . import _lib
from .policy import _CODES, _guard, _on_gpu, _plain, _ptr, _untraced

GROUP = 256  # elements that share an exponent in an 8-bit moment
_ROW = struct.Struct("QQqqii")  # a ``SwarpTensor``, written in one call
_PARAMS = {torch.float32: 4, torch.bfloat16: 2, torch.float16: 2}  # and the bytes of each


class AdamWState(NamedTuple):
    """Flat state of a list of parameters (:func:`adamw_state`): the moments as float32, or as
    uint8 codes with one uint8 base per 256 elements; a float32 copy of the parameters, or None."""

    exp_avg: torch.Tensor
    exp_avg_sq: torch.Tensor
    avg_base: torch.Tensor | None = None
    sq_base: torch.Tensor | None = None
    master: torch.Tensor | None = None

    @property
    def bits(self) -> int:
        return 8 if self.exp_avg.dtype == torch.uint8 else 32

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Both moments as flat float32 (the state's own tensors where they are)."""
        if is_dynamo_compiling():
            return _untraced(AdamWState.moments)(self)
        if self.bits == 32:
            return self.exp_avg, self.exp_avg_sq
        _on_gpu(self.exp_avg, "AdamWState.moments")
        _check_state(self, self.exp_avg.device)
        m = torch.empty(self.exp_avg.shape, device=self.exp_avg.device, dtype=torch.float32)
        v = torch.empty_like(m)
        a = _state_args(self)
        with _guard(m.device):
            _lib.check(_lib.load().swarp_adamw_unpack(ctypes.byref(a), m.data_ptr(), v.data_ptr(),
                                                      _lib.stream_of(m.device)))
        return m, v


def _slots(sizes: Iterable[int]) -> tuple[list[int], int]:
    """Where each tensor's moments start in the flat state, and its length."""
    at, n = [], 0
    for s in sizes:
        at.append(n)
        n += -(-s // GROUP) * GROUP
    return at, n


def adamw_state(params: Sequence[torch.Tensor], *, bits: int = 32,
                master: bool = False) -> AdamWState:
    """The state of ``params`` before the first step: zero moments and, with ``master``, a float32
    copy of 16-bit parameters that the steps then work on."""
    params = list(params)
    if bits not in (8, 32):
        raise ValueError(f"bits must be 8 or 32; got {bits}")
    if not params:
        raise ValueError("no parameters")
    at, n = _slots(p.numel() for p in params)
    dev = params[0].device
    z = {"device": dev, "dtype": torch.uint8 if bits == 8 else torch.float32}
    base = [torch.zeros(n // GROUP, device=dev, dtype=torch.uint8) if bits == 8 else None
            for _ in range(2)]
    copy = None
    if master:
        copy = torch.zeros(n, device=dev, dtype=torch.float32)
        for p, a in zip(params, at):
            copy[a:a + p.numel()] = p.detach().reshape(-1)
    return AdamWState(torch.zeros(n, **z), torch.zeros(n, **z), *base, copy)


def _state_args(s: AdamWState) -> _lib.SwarpAdamW:
    return _lib.SwarpAdamW(bits=s.bits, state_len=s.exp_avg.numel(), exp_avg=s.exp_avg.data_ptr(),
                           exp_avg_sq=s.exp_avg_sq.data_ptr(), avg_base=_ptr(s.avg_base),
                           sq_base=_ptr(s.sq_base), master=_ptr(s.master))


def _check_state(s: AdamWState, dev) -> None:
    n = s.exp_avg.numel()
    code = s.exp_avg.dtype
    if code not in (torch.uint8, torch.float32):
        raise TypeError(f"exp_avg must be float32 or uint8; got {code}")
    want = {"exp_avg": (n, code), "exp_avg_sq": (n, code)}
    if code == torch.uint8:
        want |= {"avg_base": (n // GROUP, torch.uint8), "sq_base": (n // GROUP, torch.uint8)}
    if s.master is not None:
        want["master"] = (n, torch.float32)
    for name, (k, dtype) in want.items():
        t = getattr(s, name)
        if (t is None or t.numel() != k or t.dtype != dtype or not t.is_contiguous()
                or t.is_neg()):
            raise ValueError(f"state.{name} must be a contiguous {dtype} tensor of {k} elements")
        if t.device != dev:
            raise ValueError(f"state.{name} is on {t.device}, the parameters on {dev}")


def _table(params, grads, dev):
    """The C table of the tensors that have a gradient, the gradients made for it, the state's
    length, and whether two of the tensors share memory."""
    rows, write, wide = bytearray(_ROW.size * max(len(params), 1)), _ROW.pack_into, _ROW.size
    at, count, keep, starts, ends = 0, 0, [], [], []
    index = -1 if dev.index is None else dev.index  # (which the CPU's tensors say, too)
    # (asked of all at once: a step's host time goes by what is asked of each)
    neg = torch.Tensor.is_neg
    negated = any(map(neg, params)) or any(map(neg, [g for g in grads if g is not None]))
    for k, (p, g) in enumerate(zip(params, grads)):
        size = p.numel()
        if g is not None and size:
            dtype, g_dtype = p.dtype, g.dtype
            if dtype not in _PARAMS:
                raise TypeError(f"parameter {k}: float32, bfloat16 or float16; got {dtype}")
            if p.get_device() != index or g.get_device() != index:
                raise ValueError(f"parameter {k} and its gradient must be on {dev}")
            if not p.is_contiguous() or negated and p.is_neg():
                raise ValueError(f"parameter {k} must be contiguous, and no negated view")
            if g.shape != p.shape or g.layout != torch.strided:
                raise ValueError(f"gradient {k} must be a dense {list(p.shape)}; got "
                                 f"{list(g.shape)}")
            if g_dtype is not dtype and g_dtype != torch.float32:
                raise TypeError(f"gradient {k} must be {dtype} or float32; got {g_dtype}")
            if not g.is_contiguous() or negated and g.is_neg():
                g = _plain(g)
                keep.append(g)
            start = p.data_ptr()
            starts.append(start)
            ends.append(start + size * _PARAMS[dtype])
            write(rows, count * wide, start, g.data_ptr(), size, at, _CODES[dtype],
                  _CODES[g_dtype])
            count += 1
        at += -(-size // GROUP) * GROUP
    # (spans are apart if, each list in order, every one ends before the next begins)
    starts.sort()
    ends.sort()
    table = (_lib.SwarpTensor * max(len(params), 1)).from_buffer(rows)
    return table, count, keep, at, any(map(operator.lt, starts[1:], ends))


_SUMS = 4096  # float32 of work memory of the norm, which its results lie behind


def _norm_of(table, count, max_norm: float, dev) -> torch.Tensor:
    """The norm and the scale, as elements ``_SUMS`` and ``_SUMS + 1``."""
    out = torch.empty(_SUMS + 2, device=dev, dtype=torch.float32)
    work = out.data_ptr()
    _lib.check(_lib.load().swarp_grad_norm(table, count, max_norm, work + 4 * _SUMS, work,
                                           _lib.stream_of(dev)))
    return out


def _check_rates(lr, betas, eps, weight_decay) -> None:
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"betas must lie in [0, 1); got {betas}")
    if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0):
        raise ValueError("lr, eps and weight_decay must be >= 0; got "
                         f"{lr}, {eps} and {weight_decay}")


def _check_norm(max_norm: float) -> None:
    if not max_norm > 0:
        raise ValueError(f"the largest norm must be > 0; got {max_norm}")


def grad_norm(grads: Sequence[torch.Tensor | None],
              max_norm: float = float("inf")) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, scale)``, float32 scalars on the device: the 2-norm of all ``grads`` together (in
    a fixed order: the same bits every time) and ``min(1, max_norm / (norm + 1e-6))``, which
    :func:`adamw_step` takes as ``grad_scale``.  No host synchronisation."""
    if is_dynamo_compiling():
        return _untraced(grad_norm)(grads, max_norm)
    grads = [_plain(g) for g in grads if g is not None]
    if not grads:
        raise ValueError("no gradients")
    _check_norm(max_norm)
    dev = grads[0].device
    _on_gpu(grads[0], "grad_norm")
    table, count, keep, *_ = _table(grads, grads, dev)
    with _guard(dev):
        out = _norm_of(table, count, max_norm, dev)
    return out[_SUMS], out[_SUMS + 1]


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor | None],
               state: AdamWState, step: int, *, lr: float = 1e-3,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.01, max_grad_norm: float | None = None,
               grad_scale: torch.Tensor | None = None, seed: int = 0) -> torch.Tensor | None:
    """Step number ``step`` (from 1 on) of AdamW with decoupled weight decay, in place, over all
    ``params``: float32, bfloat16 or float16, each gradient of its parameter's type or float32
    (None: that parameter and its moments stay as they are).

    ``max_grad_norm`` scales the gradients so that their common norm is at most that, and returns
    the norm they had; ``grad_scale`` (a float32 scalar on the device) scales them by itself.
    bfloat16 parameters without a master copy, and 8-bit moments, are rounded up or down at
    random, in proportion: an update below half a step is not lost on average.  ``seed`` is where
    those random numbers come from: give each step another one.
    """
    if is_dynamo_compiling():
        return _untraced(adamw_step)(
            params, grads, state, step, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
            max_grad_norm=max_grad_norm, grad_scale=grad_scale, seed=seed)
    params, grads = list(params), list(grads)
    if len(params) != len(grads):
        raise ValueError(f"{len(params)} parameters, {len(grads)} gradients")
    if not params:
        raise ValueError("no parameters")
    if step < 1:
        raise ValueError(f"step counts from 1; got {step}")
    _check_rates(lr, betas, eps, weight_decay)
    if max_grad_norm is not None:
        _check_norm(max_grad_norm)
        if grad_scale is not None:
            raise ValueError("give max_grad_norm or grad_scale, not both")
    dev = params[0].device
    _on_gpu(params[0], "adamw_step")
    table, count, keep, n, shared = _table(params, grads, dev)
    if shared:
        raise ValueError("two parameters share memory, or one is listed twice: their updates "
                         "would race")
    _check_state(state, dev)
    if state.exp_avg.numel() != n:
        raise ValueError(f"the state holds {state.exp_avg.numel()} elements, these parameters "
                         f"take {n}")
    if state.master is None and torch.float16 in [p.dtype for p in params]:
        raise ValueError("float16 parameters need a master copy (adamw_state(..., master=True))")
    if grad_scale is not None and (grad_scale.numel() != 1 or grad_scale.dtype != torch.float32
                                   or grad_scale.device != dev):
        raise ValueError(f"grad_scale must be one float32 on {dev}")
    if grad_scale is not None:
        grad_scale = _plain(grad_scale)
    a = _state_args(state)
    a.seed, a.step, a.lr, a.beta1, a.beta2 = seed & 0xFFFFFFFF, step, lr, betas[0], betas[1]
    a.eps, a.weight_decay, a.grad_scale = eps, weight_decay, _ptr(grad_scale)
    norm = None
    with _guard(dev):
        if max_grad_norm is not None:
            norm = _norm_of(table, count, max_grad_norm, dev)
            a.grad_scale = norm.data_ptr() + 4 * (_SUMS + 1)
        _lib.check(_lib.load().swarp_adamw(ctypes.byref(a), table, count, _lib.stream_of(dev)))
    # autograd then refuses a backward through what a graph saved of them before
    torch.autograd.graph.increment_version(
        [p for p, g in zip(params, grads) if g is not None and not p.is_inference()])
    return None if norm is None else norm[_SUMS]


class AdamW(torch.optim.Optimizer):
    """AdamW over the parameter groups (one launch per group and 64 tensors), as
    :func:`adamw_step`.  Steps are counted by group: a parameter whose first gradient comes late
    is corrected for the steps that its group has taken.

    ``bits`` (32 or 8) is the width of the moments.  ``master`` keeps a float32 copy of 16-bit
    parameters (default: where a group holds float16 ones, or the state that is loaded has one);
    after changing such parameters by other means call :meth:`sync_master`.  ``max_grad_norm`` clips the norm over all groups;
    ``last_grad_norm`` is what it was, on the device."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, *, bits: int = 32, master: bool | None = None,
                 max_grad_norm: float | None = None, seed: int = 0) -> None:
        if bits not in (8, 32):
            raise ValueError(f"bits must be 8 or 32; got {bits}")
        if max_grad_norm is not None:
            _check_norm(max_grad_norm)
        self.bits, self.master, self.max_grad_norm, self.seed = bits, master, max_grad_norm, seed
        self.last_grad_norm: torch.Tensor | None = None
        self._steps: dict[int, int] = {}          # by group: steps taken
        self._states: dict[int, AdamWState] = {}  # by group
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay))

    def add_param_group(self, param_group: dict) -> None:
        rates = self.defaults | param_group
        _check_rates(*(rates[name] for name in ("lr", "betas", "eps", "weight_decay")))
        super().add_param_group(param_group)

    def __getstate__(self) -> dict:  # (what a copy or a pickle takes along)
        own = ("bits", "master", "max_grad_norm", "seed", "last_grad_norm", "_steps", "_states")
        return super().__getstate__() | {name: getattr(self, name) for name in own}

    def _master_of(self, k: int) -> bool | None:
        """Whether group ``k`` keeps a master copy; None: it was left open, and nothing needs one."""
        if self.master is None and any(p.dtype == torch.float16
                                       for p in self.param_groups[k]["params"]):
            return True
        return self.master

    def _state_of(self, k: int) -> AdamWState:
        if k not in self._states:
            self._states[k] = adamw_state(self.param_groups[k]["params"], bits=self.bits,
                                          master=bool(self._master_of(k)))
        return self._states[k]

    def step(self, closure=None):
        return self._step(closure)

    @torch.no_grad()
    def _step(self, closure):
        if is_dynamo_compiling():
            return _untraced(AdamW._step)(self, closure)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [(k, g["params"], [p.grad for p in g["params"]])
                  for k, g in enumerate(self.param_groups)]
        every = [x for _, _, grads in groups for x in grads if x is not None]
        if not every:
            return loss
        scale = None
        if self.max_grad_norm is not None:
            self.last_grad_norm, scale = grad_norm(every, self.max_grad_norm)
        for k, params, grads in groups:
            if all(x is None for x in grads):
                continue
            g = self.param_groups[k]
            t = self._steps.get(k, 0) + 1
            adamw_step(params, grads, self._state_of(k), t, lr=float(g["lr"]),
                       betas=g["betas"], eps=g["eps"], weight_decay=g["weight_decay"],
                       grad_scale=scale, seed=self.seed + 0x51ED * t + k)
            self._steps[k] = t  # (a step that was refused is none)
        return loss

    @torch.no_grad()
    def sync_master(self) -> None:
        """Takes the parameters as they now are into the master copies."""
        for k, s in self._states.items():
            if s.master is not None:
                params = self.param_groups[k]["params"]
                for p, a in zip(params, _slots(p.numel() for p in params)[0]):
                    s.master[a:a + p.numel()] = p.reshape(-1)

    def _hooks(self, when: str) -> list:
        """What was registered by ``register_state_dict_pre_hook`` and its like."""
        return list(getattr(self, f"_optimizer_{when}_hooks", {}).values())

    def state_dict(self) -> dict:
        """Hyperparameters, step count and the flat states of the groups."""
        for hook in self._hooks("state_dict_pre"):
            hook(self)
        state = {"steps": dict(self._steps), "seed": self.seed,
                 "groups": [{k: v for k, v in g.items() if k != "params"}
                            for g in self.param_groups],
                 "states": {k: dict(s._asdict()) for k, s in self._states.items()}}
        for hook in self._hooks("state_dict_post"):
            changed = hook(self, state)
            state = state if changed is None else changed
        return state

    @torch.no_grad()
    def load_state_dict(self, state: dict) -> None:
        state = dict(state)  # (the caller's own stays as it is)
        for hook in self._hooks("load_state_dict_pre"):
            changed = hook(self, state)
            state = state if changed is None else changed
        if len(state["groups"]) != len(self.param_groups):
            raise ValueError(f"{len(state['groups'])} parameter groups in the state, "
                             f"{len(self.param_groups)} here")
        states = {}
        for k, s in state["states"].items():
            params = self.param_groups[k]["params"]
            dev, n = params[0].device, _slots(p.numel() for p in params)[1]
            s = AdamWState(**{name: None if t is None else t.to(dev).clone()
                              for name, t in s.items()})
            _check_state(s, dev)
            if s.exp_avg.numel() != n:
                raise ValueError(f"group {k}: the state holds {s.exp_avg.numel()} elements, its "
                                 f"parameters take {n}")
            if s.bits != self.bits:
                raise ValueError(f"group {k}: moments of {s.bits} bits, this optimizer keeps "
                                 f"{self.bits}")
            keeps = self._master_of(k)
            if keeps is not None and keeps != (s.master is not None):
                raise ValueError(f"group {k}: the state has {'no' if keeps else 'a'} master copy, "
                                 f"this optimizer keeps {'one' if keeps else 'none'}")
            states[k] = s
        for new in state["groups"]:
            _check_rates(*(new[name] for name in ("lr", "betas", "eps", "weight_decay")))
        for g, new in zip(self.param_groups, state["groups"]):
            g.update(new)
        self._states, self._steps, self.seed = states, dict(state["steps"]), state["seed"]
        for hook in self._hooks("load_state_dict_post"):
            hook(self)
