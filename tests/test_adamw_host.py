"""The optimizer around the AdamW step, without a GPU: what it loads, takes, refuses and tells its
hooks."""

import ctypes
import pickle

import pytest
import torch

from swarp_amd import AdamW, _lib, adamw_state
from swarp_amd.optim import _table


def params(dtype=torch.bfloat16, n=300):
    return [torch.nn.Parameter(torch.ones(n, dtype=dtype))]


def saved(dtype=torch.bfloat16, **kw):
    """The state dictionary of an optimizer that has its state."""
    opt = AdamW(params(dtype), **kw)
    opt._state_of(0)
    return opt.state_dict()


def test_a_loaded_state_has_the_master_that_the_optimizer_keeps():
    without, having = saved(), saved(master=True)
    with pytest.raises(ValueError, match="no master copy"):
        AdamW(params(), master=True).load_state_dict(without)
    with pytest.raises(ValueError, match="a master copy"):
        AdamW(params(), master=False).load_state_dict(having)
    with pytest.raises(ValueError, match="no master copy"):  # which float16 needs
        AdamW(params(torch.float16)).load_state_dict(without)
    for kw, state in (({"master": True}, having), ({"master": False}, without), ({}, without),
                      ({}, having)):
        opt = AdamW(params(), **kw)
        opt.load_state_dict(state)
        assert (opt._states[0].master is None) == (state is without)
    opt = AdamW(params(torch.float16))
    opt.load_state_dict(saved(torch.float16))
    assert opt._states[0].master is not None


def test_a_refused_state_leaves_the_optimizer_as_it_was():
    opt = AdamW(params(), master=True, seed=4)
    with pytest.raises(ValueError):
        opt.load_state_dict(saved(seed=9, lr=1.0))
    assert opt.seed == 4 and not opt._states and opt.param_groups[0]["lr"] == 1e-3


def test_a_step_that_is_refused_is_not_counted():
    opt = AdamW(params(torch.float32))
    opt.param_groups[0]["params"][0].grad = torch.ones(300)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="HIP device"):
            opt.step()
    assert opt.state_dict()["steps"] == {}


def test_parameters_that_share_memory_are_found():
    b = torch.zeros(1000)

    def shared(*spans):
        p = [b[lo:hi] for lo, hi in spans]
        return _table(p, [torch.zeros_like(x) for x in p], b.device)[4]
    assert shared((0, 300), (100, 400)) and shared((100, 400), (0, 300))
    assert shared((0, 1000), (10, 20), (30, 40)) and shared((5, 6), (5, 6))
    assert shared((0, 10), (20, 30), (29, 40), (50, 60))
    assert not shared((0, 300), (300, 400)) and not shared((500, 1000), (0, 1), (1, 500))
    assert not shared((0, 10)) and not shared((0, 0), (0, 10), (5, 5))
    h = b.view(torch.bfloat16)
    assert _table([b[:10], h[19:30]], [torch.zeros(10), torch.zeros(11).bfloat16()], b.device)[4]
    assert not _table([b[:10], h[20:30]], [torch.zeros(10), torch.zeros(10).bfloat16()], b.device)[4]
    # one without a gradient is not touched
    assert not _table([b[:300], b[100:400]], [torch.zeros(300), None], b.device)[4]


@pytest.mark.parametrize("rates", [{"lr": -1.0}, {"betas": (2.0, 2.0)}, {"betas": (0.9, 1.0)},
                                   {"eps": -1e-8}, {"weight_decay": -0.1}, {"lr": float("nan")}])
def test_rates_are_refused_when_they_are_given(rates):
    """... to the constructor, in a group, in a group that is added later, in a loaded state."""
    with pytest.raises(ValueError, match="lr, eps|betas"):
        AdamW(params(), **rates)
    with pytest.raises(ValueError, match="lr, eps|betas"):
        AdamW([{"params": params()}, {"params": params(), **rates}])
    opt = AdamW(params())
    with pytest.raises(ValueError, match="lr, eps|betas"):
        opt.add_param_group({"params": params(), **rates})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": params(), "lr": 0.5})
    assert [g["lr"] for g in opt.param_groups] == [1e-3, 0.5]
    state = AdamW(params()).state_dict()
    state["groups"][0] |= rates
    opt = AdamW(params(), seed=3)
    with pytest.raises(ValueError, match="lr, eps|betas"):
        opt.load_state_dict(state)
    assert opt.param_groups[0]["lr"] == 1e-3 and opt.seed == 3


def test_hooks_are_called():
    """Those of the state dictionary, of its loading (which may replace it) and of a step."""
    said = []
    opt = AdamW(params(), seed=3)
    opt.register_state_dict_pre_hook(lambda o: said.append(("pre", o is opt)))
    opt.register_state_dict_post_hook(lambda o, s: {**s, "note": "kept"})
    gone = opt.register_state_dict_post_hook(lambda o, s: said.append("gone"))
    gone.remove()
    state = opt.state_dict()
    assert state["note"] == "kept" and said == [("pre", True)]

    two = AdamW(params(), seed=4)
    two.register_load_state_dict_pre_hook(lambda o, s: {**s, "seed": 8})
    two.register_load_state_dict_pre_hook(lambda o, s: s.pop("note") and None)
    two.register_load_state_dict_post_hook(lambda o: said.append(o.seed))
    two.load_state_dict(state)
    assert two.seed == 8 and said[-1] == 8 and state["seed"] == 3 and state["note"] == "kept"
    opt.register_step_pre_hook(lambda o, args, kwargs: said.append("step"))
    opt.register_step_post_hook(lambda o, args, kwargs: said.append("stepped"))
    opt.step()
    assert said[-2:] == ["step", "stepped"]
    # a copy is an optimizer like another
    three = pickle.loads(pickle.dumps(AdamW(params(), seed=5)))
    assert three.state_dict()["seed"] == 5
    three.register_state_dict_pre_hook(lambda o: said.append("copy"))
    three.state_dict()
    assert said[-1] == "copy"


def test_moments_of_a_state_in_host_memory():
    """32-bit ones are the state's own; 8-bit ones are unpacked by a kernel, which is not handed
    host addresses."""
    p = params(torch.float32)
    s = adamw_state(p)
    assert s.moments()[0] is s.exp_avg
    with pytest.raises(RuntimeError, match="HIP device"):
        adamw_state(p, bits=8).moments()


def test_a_tensor_too_large_for_a_launch_is_refused_before_any():
    """2^35 elements are 2^24 workgroups of 256 threads, one thread more than a launch has: refused
    with the arguments, not by the runtime when other tensors of the step are already written."""
    lib, n = _lib.load(), 1 << 35
    s = _lib.SwarpAdamW(bits=32, state_len=n, step=1, exp_avg=256, exp_avg_sq=512)
    t = (_lib.SwarpTensor * 1)(_lib.SwarpTensor(param=64, grad=64, n=n, slot=0))
    assert lib.swarp_adamw(ctypes.byref(s), t, 1, None) != 0
    assert b"out of range" in lib.swarp_last_error()
    # (a call that is accepted clears the message)
    a = _lib.SwarpGae(dtype=0, steps=0, columns=4, group=1)
    assert lib.swarp_gae_fwd(ctypes.byref(a), None) == 0 and lib.swarp_last_error() == b""
