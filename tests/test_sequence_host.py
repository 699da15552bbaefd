"""Host side of the sequence operators, without a GPU: struct layouts, what the C entry points refuse,
and that nothing computes on the CPU."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from swarp_amd import _lib, decay_attention, decay_attention_step, linear_cross_entropy, memory

HEADER = Path(__file__).resolve().parents[1] / "include" / "swarp_hip.h"


def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    pairs = [(_lib.SwarpLinearCe, "swarp_linear_ce_t"), (_lib.SwarpDecay, "swarp_decay_t")]
    for cls, name in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join([*lines, "return 0;}"]))
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                                          check=True).stdout.split()]
    want = []
    for cls, _ in pairs:
        want += [ctypes.sizeof(cls), *(getattr(cls, f).offset for f, _ in cls._fields_)]
    assert got == want


def refused(rc, word):
    assert rc != 0 and word in _lib.load().swarp_last_error().decode(), _lib.load().swarp_last_error()


def test_linear_ce_refuses_before_any_launch():
    lib = _lib.load()

    def args(**kw):
        base = dict(dtype=0, dim=8, width=100, rows=4, inner=4, inner_stride=8, hidden=256, weight=256,
                    targets=256, logp=256, loss=256)
        return _lib.SwarpLinearCe(**{**base, **kw})

    def call(a):
        return lib.swarp_linear_ce(ctypes.byref(a), None)
    refused(lib.swarp_linear_ce(None, None), "arguments")
    for kw in (dict(dtype=1), dict(dtype=9)):
        refused(call(args(**kw)), "dtype")
        assert lib.swarp_linear_ce_work_bytes(ctypes.byref(args(**kw))) == 0
    for kw in (dict(rows=-1), dict(rows=1 << 31), dict(dim=0), dict(dim=65537), dict(width=0), dict(width=(1 << 21) + 1)):
        refused(call(args(**kw)), "sizes")
    refused(call(args(loss=None)), "loss")
    refused(call(args()), "work")
    need = lib.swarp_linear_ce_work_bytes(ctypes.byref(args()))
    assert need > 0
    refused(call(args(work=256, work_bytes=need - 1)), "work")
    refused(call(args(work=264, work_bytes=need)), "aligned")
    for kw in (dict(hidden=None), dict(weight=None), dict(targets=None), dict(logp=None), dict(inner=0)):
        refused(call(args(work=256, work_bytes=need, **kw)), "pointer")
    a = args(mask=256, work=256)
    a.work_bytes = lib.swarp_linear_ce_work_bytes(ctypes.byref(a))
    refused(call(a), "place")
    a = args(d_hidden=256)

    def back(a, *p):
        return lib.swarp_linear_ce_bwd(ctypes.byref(a), 1, *p, None)
    refused(back(a, None, 256, None, None), "pointer")
    refused(back(a, 256, None, 256, None), "pointer")
    refused(back(args(d_weight=256, dtype=2), 256, None, 256, None), "in place")
    refused(back(args(d_hidden=256, mask=256, place=256), 256, 256, None, None), "in place")
    refused(back(args(d_hidden=256, mask=256), 256, 512, None, None), "place")
    # a head that fits a workgroup is complete, and its backward computes again
    for dim, width, one in ((128, 32, 1), (129, 32, 0), (64, 64, 1), (65, 33, 0), (64, 65, 0)):
        assert lib.swarp_linear_ce_complete(ctypes.byref(args(dim=dim, width=width))) == one
    assert lib.swarp_linear_ce_complete(ctypes.byref(args(dtype=1, width=9))) == 0
    a = args(width=9)
    refused(call(a), "work")
    refused(back(a, 256, 256, None, None), "work")
    a.work, a.work_bytes = 256, lib.swarp_linear_ce_work_bytes(ctypes.byref(a))
    a.weight = None
    refused(back(a, 256, 256, None, None), "pointer")
    # gradients need room for the exponentials, a mask for its list
    grad = args(rows=5000, width=40000, d_weight=256)
    plain = args(rows=5000, width=40000)
    assert lib.swarp_linear_ce_work_bytes(ctypes.byref(grad)) > 5000 * 40000 * 4 / 4
    assert lib.swarp_linear_ce_work_bytes(ctypes.byref(plain)) < lib.swarp_linear_ce_work_bytes(ctypes.byref(grad))
    # however many rows: the exponentials stay below 1 GiB, sums of the weight's gradient aside
    big = args(rows=1 << 24, dim=64, width=1 << 16, dtype=2, d_hidden=256)
    assert lib.swarp_linear_ce_work_bytes(ctypes.byref(big)) < (1 << 30) + (1 << 24) * (64 * 2 + 40) + (1 << 29)


def test_decay_refuses_before_any_launch():
    lib = _lib.load()

    def args(**kw):
        base = dict(dtype=0, heads=2, dk=8, dv=8, steps=3, batch=4, group=1, scale=1.0, log_decay=256,
                    q=256, k=256, v=256, out=256)
        return _lib.SwarpDecay(**{**base, **kw})
    calls = (lib.swarp_decay_fwd, lib.swarp_decay_bwd, lib.swarp_decay_step)
    for f in calls:
        refused(f(None, None), "arguments")
        for kw in (dict(dtype=1), dict(dtype=-1)):
            refused(f(ctypes.byref(args(**kw)), None), "dtype")
        for kw in (dict(heads=0), dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=129), dict(steps=-1), dict(batch=-1),
                   dict(group=0), dict(group=3), dict(batch=1 << 31, group=1)):
            refused(f(ctypes.byref(args(**kw)), None), "sizes")
        a = args(log_decay=None, adj_out=256, state_out=256, steps=1)
        a.work, a.work_bytes = 256, lib.swarp_decay_work_bytes(ctypes.byref(a))
        refused(f(ctypes.byref(a), None), "pointer")
        a = args(batch=0, steps=1)
        assert f(ctypes.byref(a), None) == 0 and lib.swarp_last_error() == b""
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None)):
        a = args(**kw)
        a.work, a.work_bytes = 256, lib.swarp_decay_work_bytes(ctypes.byref(a))
        refused(lib.swarp_decay_fwd(ctypes.byref(a), None), "pointer")
    a = args(adj_out=256, d_q=256)
    a.work, a.work_bytes = 256, lib.swarp_decay_work_bytes(ctypes.byref(a))
    refused(lib.swarp_decay_bwd(ctypes.byref(a), None), "together")
    refused(lib.swarp_decay_step(ctypes.byref(args(state_out=256)), None), "one step")
    refused(lib.swarp_decay_step(ctypes.byref(args(steps=1)), None), "pointer")
    # the state: 4 x 2 x 8 x 8 floats from 1 << 20 on; q, k and v: 4 x 2 x 8
    state, n = 1 << 20, 4 * 2 * 8 * 8 * 4
    strides = {x + "_stride": (ctypes.c_int64 * 3)(0, 16, 8) for x in "qkv"}
    for name in "qkv":
        for at in (state, state - 4, state + n - 4, state - 4 * 2 * 8 * 4 + 4):
            refused(lib.swarp_decay_step(ctypes.byref(args(steps=1, state_out=state, **strides, **{name: at})), None),
                    "in the state")


@pytest.mark.parametrize("missing", ["d_q", "d_k", "d_v", "all"])
@pytest.mark.parametrize("d_state", [None, 256])
def test_the_adjoint_of_a_scan_wants_all_three_gradients(missing, d_state):
    """Its kernels write all of them, also where only the state's is wanted."""
    lib = _lib.load()
    outs = {name: None if missing in (name, "all") else 256 for name in ("d_q", "d_k", "d_v")}
    a = _lib.SwarpDecay(dtype=0, heads=2, dk=8, dv=8, steps=3, batch=4, group=1, scale=1.0, log_decay=256, q=256, k=256,
                        v=256, state=256, adj_out=256, d_state=d_state, work=256, **outs)
    a.work_bytes = lib.swarp_decay_work_bytes(ctypes.byref(a))
    refused(lib.swarp_decay_bwd(ctypes.byref(a), None), "together")


@pytest.mark.parametrize("dtype,size", [(0, 4), (2, 2), (3, 2)])
def test_linear_ce_work_memory_is_what_is_said(dtype, size):
    """Of wide heads: copies, 60 bytes a row, and with gradients 2.1 times a piece's exponentials, 128 bytes a
    column and 129 MiB; without 1 GiB."""
    lib, pad = _lib.load(), 64 // size
    for N in (1, 33, 300, 5000, 1 << 17, 1 << 24, (1 << 31) - 1):
        for D in (65, 129, 333, 2048, 65536):
            for V in (1, 33, 65, 2048, 32003, 1 << 20, 1 << 21):
                for grads in (0, 1, 2, 4, 7):
                    a = _lib.SwarpLinearCe(dtype=dtype, dim=D, width=V, rows=N, inner=1, mask=256, weight=256,
                                           d_hidden=256 * (grads & 1), d_weight=256 * (grads >> 1 & 1),
                                           d_bias=256 * (grads >> 2))
                    if lib.swarp_linear_ce_complete(ctypes.byref(a)):
                        continue
                    row = -(-D // pad) * 64
                    copies = (N + 31) * row + (V * row if D * size % 16 else 0)
                    piece = max(1 << 30, 256 * -(-V // pad) * 64)
                    rest = 2.1 * piece + 128 * V + (129 << 20) if grads else 1 << 30
                    need = lib.swarp_linear_ce_work_bytes(ctypes.byref(a))
                    assert 0 < need <= copies + 60 * N + rest + 8192, (N, D, V, grads)


def test_decay_refuses_states_in_place():
    lib = _lib.load()
    a = _lib.SwarpDecay(dtype=0, heads=2, dk=8, dv=8, steps=3, batch=4, group=1, scale=1.0, log_decay=256, q=256, k=256, v=256,
                        out=256, adj_out=256, d_q=256, d_k=256, d_v=256, work=256)
    a.work_bytes = lib.swarp_decay_work_bytes(ctypes.byref(a))
    a.state = a.state_out = 512
    refused(lib.swarp_decay_fwd(ctypes.byref(a), None), "must not be state")
    a.adj_state = a.d_state = 512
    refused(lib.swarp_decay_bwd(ctypes.byref(a), None), "must not be adj_state")


def test_a_steps_decay_and_starts_lie_outside_its_state():
    lib, state, n = _lib.load(), 1 << 20, 4 * 2 * 8 * 8 * 4
    strides = {x + "_stride": (ctypes.c_int64 * 3)(0, 16, 8) for x in "qkv"}
    for name, size in (("log_decay", 8), ("starts", 4)):
        for at in (state, state + n - 1, state - size + 1):
            a = _lib.SwarpDecay(**{**dict(dtype=0, heads=2, dk=8, dv=8, steps=1, batch=4, group=1, scale=1.0, log_decay=256, q=256,
                                          k=256, v=256, out=256, state_out=state, **strides), name: at})
            refused(lib.swarp_decay_step(ctypes.byref(a), None), "in the state")


def test_heads_beyond_a_launch_are_refused():
    lib = _lib.load()
    a = _lib.SwarpDecay(dtype=0, heads=(1 << 22) + 1, dk=8, dv=8, steps=1, batch=1, group=1)
    for f in (lib.swarp_decay_fwd, lib.swarp_decay_bwd, lib.swarp_decay_step):
        refused(f(ctypes.byref(a), None), "sizes")
    assert lib.swarp_decay_work_bytes(ctypes.byref(a)) == 0
    a.heads -= 1
    assert lib.swarp_decay_work_bytes(ctypes.byref(a)) > 0


@pytest.mark.parametrize("shape", [(5, 4, 0, 2, 8), (5, 0, 4, 2, 8), (0, 4, 3, 2, 8), (5, 3, 0, 2, 2, 8)])
def test_strides_of_what_is_empty(shape):
    x = torch.zeros(shape)
    for y in (x, x[..., ::2], x.transpose(1, 2)):
        for lead in (1, 0):
            laid, strides = memory._laid(y, lead)
            assert laid.numel() == 0 and list(strides) == [0, 0, 0]


@pytest.fixture(autouse=True)
def no_message_left_behind():
    yield
    a = _lib.SwarpDecay(dtype=0, heads=1, dk=1, dv=1, group=1)
    assert _lib.load().swarp_decay_fwd(ctypes.byref(a), None) == 0 and _lib.load().swarp_last_error() == b""


def test_nothing_computes_on_the_cpu():
    z = torch.zeros(3, 2, 4)
    with pytest.raises(RuntimeError, match="HIP device"):
        linear_cross_entropy(z, torch.zeros(5, 4), torch.zeros(3, 2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="HIP device"):
        decay_attention(z, z, z, torch.zeros(2))
    with pytest.raises(RuntimeError, match="HIP device"):
        decay_attention_step(z, z, z, torch.zeros(2), torch.zeros(3, 2, 4, 4))
