"""The policy update's kernels on the CPU under AddressSanitizer and UBSan at the ends of the
number range (tests/asan/learn_ends.cpp), a case a run."""

import importlib.util
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
CLANG = Path("/opt/rocm/llvm/bin/clang++")


@pytest.fixture(scope="module")
def exe():
    if not CLANG.exists():
        pytest.skip("no clang++")
    spec = importlib.util.spec_from_file_location("asan_build", HERE / "asan" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.OUT.mkdir(exist_ok=True)
    mod.stage()
    exe = mod.OUT / "learn_ends"
    flags = [f for f in mod.FLAGS if not f.startswith("-Wno")]
    r = subprocess.run([str(CLANG), *flags, "-w", f"-I{HERE / 'asan' / 'emu'}", f"-I{mod.SRC}",
                        str(HERE / "asan" / "learn_ends.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return exe


@pytest.mark.parametrize("case", ["forbidden", "kl", "cut", "gradients"])
def test_at_the_ends_of_the_range(exe, case):
    r = subprocess.run([str(exe), case], capture_output=True, text=True, timeout=600, cwd="/tmp")
    assert r.returncode == 0 and f"{case}: 0 wrong" in r.stdout, r.stdout[:3000] + r.stderr[-3000:]
    assert "ERROR: AddressSanitizer" not in r.stderr and "runtime error" not in r.stderr
