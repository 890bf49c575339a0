"""CPU: how steps and prompts over a cache in 8 bits have their keys cut, under sanitizers
(tests/cpp/test_quant_cuts.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tiny-llm_amd", "csrc")


def test_cuts_under_sanitizers(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    exe = str(tmp_path / "test_quant_cuts")
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", "-g", "-O1", "-I", CSRC,
                    os.path.join(ROOT, "tests", "cpp", "test_quant_cuts.cpp"), os.path.join(CSRC, "quant_plan.cpp"),
                    "-o", exe], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split("\n")[:2] == ["ok prefill_cuts", "ok decode_sides"]
