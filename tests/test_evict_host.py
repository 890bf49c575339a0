"""CPU: the eviction kernels' own source, run lane by lane in several orders of the
waves (tests/cpp/wave_host), every selection kernel against a plain selection.  A barrier
that is missing, or that only some waves reach, shows here every time; on a GPU it depends
on the waves' timing, and can hang."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/llvm/bin/clang++"


def test_eviction_kernels_in_any_order_of_the_waves(tmp_path):
    if not os.path.exists(CLANG):
        pytest.skip("clang++ not found")
    exe = str(tmp_path / "test_evict_host")
    cpp = os.path.join(ROOT, "tests", "cpp")
    lib = os.path.join(ROOT, "tiny-llm_amd")
    build = subprocess.run(
        [CLANG, "-x", "c++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-Wno-unused-parameter",
         "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", os.path.join(cpp, "wave_host"),
         "-I", os.path.join(lib, "include"), "-I", os.path.join(lib, "csrc"),
         os.path.join(cpp, "test_evict_host.cpp"), "-o", exe], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split("\n")[:6] == [f"ok {x} {o}" for o in ("rising", "falling", "random") for x in ("short", "long")]
