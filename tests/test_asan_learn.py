"""The policy update's kernels (gae.hip, policy.hip, adamw.hip) on the CPU under AddressSanitizer
and UBSan (tests/asan/learn.cpp): exact buffers, odd sizes, results against plain loops.  They
hold bfloat16 and float16 values, which the toolchain's clang has as types."""

import importlib.util
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
CLANG = Path("/opt/rocm/llvm/bin/clang++")


def test_policy_update_clean_under_sanitizers():
    if not CLANG.exists():
        pytest.skip("no clang++")
    spec = importlib.util.spec_from_file_location("asan_build", HERE / "asan" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.OUT.mkdir(exist_ok=True)
    mod.stage()
    exe = mod.OUT / "learn"
    flags = [f for f in mod.FLAGS if not f.startswith("-Wno")]
    r = subprocess.run([str(CLANG), *flags, "-w", f"-I{HERE / 'asan' / 'emu'}", f"-I{mod.SRC}",
                        str(HERE / "asan" / "learn.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=900, cwd="/tmp")
    assert r.returncode == 0 and "0 case(s) failed" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]
    assert "ERROR: AddressSanitizer" not in r.stderr and "runtime error" not in r.stderr
