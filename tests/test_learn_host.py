"""Host side of the policy update, without a GPU: struct layouts, what the C entry points refuse,
and that nothing computes on the CPU."""

import ctypes
import pickle
import subprocess
from pathlib import Path

import pytest
import torch

from swarp_amd import (AdamW, _lib, adamw_state, adamw_step, categorical_policy_loss, gae,
                       gaussian_policy_loss, grad_norm)

HEADER = Path(__file__).resolve().parents[1] / "include" / "swarp_hip.h"


def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    pairs = [(_lib.SwarpGae, "swarp_gae_t"), (_lib.SwarpPolicy, "swarp_policy_t"),
             (_lib.SwarpTensor, "swarp_tensor_t"), (_lib.SwarpAdamW, "swarp_adamw_t")]
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


def test_c_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    a = _lib.SwarpGae(dtype=2, steps=1, columns=1, group=1)
    refused(lib.swarp_gae_fwd(ctypes.byref(a), None), "dtype")
    a = _lib.SwarpGae(dtype=0, steps=3, columns=5, group=2)
    refused(lib.swarp_gae_fwd(ctypes.byref(a), None), "sizes")
    a = _lib.SwarpGae(dtype=0, steps=3, columns=4, group=2)
    refused(lib.swarp_gae_fwd(ctypes.byref(a), None), "pointer")
    a.adj_final_values = 16
    refused(lib.swarp_gae_bwd(ctypes.byref(a), None), "final_values")
    refused(lib.swarp_gae_fwd(None, None), "arguments")
    a = _lib.SwarpGae(dtype=0, steps=0, columns=4, group=1)
    assert lib.swarp_gae_fwd(ctypes.byref(a), None) == 0

    p = _lib.SwarpPolicy(dtype=9, rows=1, width=2)
    refused(lib.swarp_categorical_loss(ctypes.byref(p), None), "dtype")
    p = _lib.SwarpPolicy(dtype=0, rows=1, width=0)
    refused(lib.swarp_categorical_loss(ctypes.byref(p), None), "sizes")
    p = _lib.SwarpPolicy(dtype=0, rows=1, width=2)
    refused(lib.swarp_categorical_loss(ctypes.byref(p), None), "work")
    need = lib.swarp_policy_work_bytes(1, 2)
    p.work, p.work_bytes = 64, need - 1
    refused(lib.swarp_categorical_loss(ctypes.byref(p), None), "work")
    p.work, p.work_bytes = 65, need
    refused(lib.swarp_categorical_loss(ctypes.byref(p), None), "aligned")
    p.work = 64
    refused(lib.swarp_categorical_loss(ctypes.byref(p), None), "pointer")
    p = _lib.SwarpPolicy(dtype=0, rows=1, width=65, work=64,
                         work_bytes=lib.swarp_policy_work_bytes(1, 65))
    refused(lib.swarp_gaussian_loss(ctypes.byref(p), None), "pointer")
    refused(lib.swarp_gaussian_loss_bwd(ctypes.byref(p), 1, None, None), "arguments")
    # a row that is split over workgroups needs room for its parts
    assert lib.swarp_policy_work_bytes(100, 131072) > lib.swarp_policy_work_bytes(100, 8192)

    s = _lib.SwarpAdamW(bits=16)
    refused(lib.swarp_adamw(ctypes.byref(s), None, 0, None), "bits")
    s = _lib.SwarpAdamW(bits=32, state_len=100, step=1)
    refused(lib.swarp_adamw(ctypes.byref(s), None, 0, None), "256")
    s = _lib.SwarpAdamW(bits=32, state_len=256, step=1, exp_avg=256, exp_avg_sq=512)
    t = (_lib.SwarpTensor * 1)(_lib.SwarpTensor(param=64, grad=64, n=257, slot=0))
    refused(lib.swarp_adamw(ctypes.byref(s), t, 1, None), "outside")
    t[0].n, t[0].slot = 10, 3
    refused(lib.swarp_adamw(ctypes.byref(s), t, 1, None), "outside")
    t[0].slot, t[0].grad_dtype = 0, 2
    refused(lib.swarp_adamw(ctypes.byref(s), t, 1, None), "type")
    t[0].param_dtype = t[0].grad_dtype = 3
    refused(lib.swarp_adamw(ctypes.byref(s), t, 1, None), "master")
    t[0].param_dtype = t[0].grad_dtype = 0
    s.step = 0
    refused(lib.swarp_adamw(ctypes.byref(s), t, 1, None), "step")
    refused(lib.swarp_adamw_unpack(ctypes.byref(s), None, None, None), "8-bit")
    refused(lib.swarp_grad_norm(t, 1, 1.0, None, None, None), "norm_scale")
    t[0].grad = None
    refused(lib.swarp_grad_norm(t, 1, 1.0, 64, 64, None), "gradient")
    # a call that is accepted clears the message
    assert lib.swarp_gae_fwd(ctypes.byref(a), None) == 0 and lib.swarp_last_error() == b""


def test_nothing_computes_on_the_cpu():
    z, f = torch.zeros(3), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="HIP device"):
        gae(z, torch.zeros(4))
    with pytest.raises(RuntimeError, match="HIP device"):
        categorical_policy_loss(torch.zeros(3, 2), f, z, z)
    with pytest.raises(RuntimeError, match="HIP device"):
        gaussian_policy_loss(torch.zeros(3, 2), torch.zeros(2), torch.zeros(3, 2), z, z)
    with pytest.raises(RuntimeError, match="HIP device"):
        grad_norm([z])
    with pytest.raises(RuntimeError, match="HIP device"):
        adamw_step([z], [z], adamw_state([z]), 1)


def test_state_layout():
    s = adamw_state([torch.zeros(1), torch.zeros(257), torch.zeros(0)], bits=8, master=True)
    assert s.exp_avg.shape == (768,) and s.avg_base.shape == (3,) and s.bits == 8
    assert s.master.dtype == torch.float32
    opt = AdamW([torch.nn.Parameter(torch.zeros(3))])
    assert opt.step() is None and opt.state_dict()["steps"] == {}


def test_a_copied_optimizer_keeps_its_settings():
    one = AdamW([torch.nn.Parameter(torch.zeros(3))], lr=2e-3, bits=8, max_grad_norm=0.5, seed=7)
    two = pickle.loads(pickle.dumps(one))
    assert (two.bits, two.max_grad_norm, two.seed, two.master) == (8, 0.5, 7, None)
    assert two.param_groups[0]["lr"] == 2e-3 and two.step() is None
