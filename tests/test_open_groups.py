"""CPU: the open groups of a cache in 8 bits beside an fp16 cache's tokens, under sanitizers
(tests/cpp/test_open_groups.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tiny-llm_amd", "csrc")
CHECKS = ["advance_beyond_what_was_appended", "advance_over_another_append", "advance_where_layers_differ"]


def test_open_groups_under_sanitizers(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    exe = str(tmp_path / "test_open_groups")
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", "-g", "-O1", "-I", CSRC,
                    os.path.join(ROOT, "tests", "cpp", "test_open_groups.cpp"), os.path.join(CSRC, "quant_plan.cpp"),
                    "-o", exe], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert [line[3:] for line in r.stdout.splitlines()] == CHECKS
