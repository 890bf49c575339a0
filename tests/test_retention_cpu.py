"""CPU: the plans of the account and cross attention kernels and the block
allocator's shrink under sanitizers, the C ABI's null handles, the binding's own
checks, and the kernels' resources."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from test_kernel_resources import kernels

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tiny-llm_amd", "csrc")


def test_plans_and_allocator_under_sanitizers(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    exe = str(tmp_path / "test_retention_plan")
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", "-g", "-O1", "-I", CSRC,
                    os.path.join(ROOT, "tests", "cpp", "test_retention_plan.cpp"), os.path.join(CSRC, "stream_plan.cpp"),
                    os.path.join(CSRC, "block_allocator.cpp"), "-o", exe], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split("\n")[:4] == ["ok stream_random", "ok account_random", "ok cross_random", "ok allocator_shrink"]


@pytest.fixture(scope="module")
def tlc():
    import tinyllm_kv
    tinyllm_kv.load()
    return tinyllm_kv


def test_null_handles(tlc):
    lib, out = tlc.load(), C.c_void_p()
    bad = tlc.TL_ERR_INVALID
    assert lib.tl_kv_evict_create(None, 1, C.byref(out)) == bad
    assert lib.tl_kv_evict_prepare(None, None, None, 0, 0, None) == bad
    assert lib.tl_kv_evict_info(None, None, None) == bad
    assert lib.tl_kv_evict_run(None, 0, None, None, None, None, None) == bad
    assert lib.tl_kv_evict_commit(None) == bad and "null" in tlc.last_error()
    assert lib.tl_kv_cross_create(None, 1, 1, C.byref(out)) == bad
    assert lib.tl_kv_cross_prepare(None, None, None, None, 0, None) == bad
    assert lib.tl_kv_cross_info(None, None, None) == bad
    assert lib.tl_kv_cross_attention(None, 0, None, None, 1.0, None) == bad and "null" in tlc.last_error()
    assert lib.tl_kv_batch_decode_weights(None, 0, None, None, None, None, 1.0, None, None, None) == bad
    assert lib.tl_kv_prefill_weights(None, 0, None, 1.0, 0, None, None, None) == bad and "null" in tlc.last_error()
    assert lib.tl_kv_evicted(None, 0) == 0
    lib.tl_kv_evict_destroy(None)
    lib.tl_kv_cross_destroy(None)


def test_lists_of_different_lengths(tlc):
    ev, cr = object.__new__(tlc.EvictBatch), object.__new__(tlc.CrossBatch)
    ev._h = cr._h = None
    with pytest.raises(ValueError):
        ev.prepare([1, 2], [3])
    with pytest.raises(ValueError):
        cr.prepare([1], [3, 4])
    with pytest.raises(ValueError):
        cr.prepare([1], [3], [4, 5])


@pytest.mark.parametrize("obj", ["evict.o", "attention_stream.o", "attention_account.o", "attention_cross.o"])
def test_kernels_use_no_scratch(obj, tmp_path):
    """Registers hold the tiles and the work lists stay in the kernel arguments."""
    for name, r in kernels(obj, tmp_path).items():
        assert r["private_segment_fixed_size"] == 0 and r["vgpr_spill_count"] == 0, (name, r)
        assert r["kernarg_segment_size"] <= 4096, (name, r)
