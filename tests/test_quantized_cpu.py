"""CPU: the plans and the open groups of a cache in 8 bits under sanitizers, the C ABI's null
handles and refusals that need no GPU, and the kernels' resources."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from test_kernel_resources import kernels

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tiny-llm_amd", "csrc")


def test_plans_and_open_groups_under_sanitizers(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    exe = str(tmp_path / "test_quant_plan")
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", "-g", "-O1", "-I", CSRC,
                    os.path.join(ROOT, "tests", "cpp", "test_quant_plan.cpp"), os.path.join(CSRC, "quant_plan.cpp"),
                    "-o", exe], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split("\n")[:3] == ["ok stream_random", "ok prefill_random", "ok open_group_random"]


@pytest.fixture(scope="module")
def tlc():
    import tinyllm_kv
    tinyllm_kv.load()
    return tinyllm_kv


def test_null_handles(tlc):
    lib, out, bad = tlc.load(), C.c_void_p(), tlc.TL_ERR_INVALID
    cfg = tlc.KVConfig(1, 1, 64, 64, 1)
    assert lib.tl_kv_create_quantized(C.byref(cfg), 32, 1, None) == bad
    assert lib.tl_kv_create_quantized(None, 32, 1, C.byref(out)) == bad and "null" in tlc.last_error()
    assert lib.tl_kv_is_quantized(None) == 0
    assert lib.tl_rotary_create(64, 64, 1e4, 0, None, None, None) == bad
    assert lib.tl_rotary_apply(None, None, 0, None, 0, None, None, None, 0, 0, 0, None, None, 0.0, None) == bad
    assert "null" in tlc.last_error()
    lib.tl_rotary_destroy(None)


@pytest.mark.parametrize("cfg,block,blocks,word", [
    (dict(head_dim=64), 16, 4, "power of two >= 32"),
    (dict(head_dim=64), 48, 4, "power of two >= 32"),
    (dict(head_dim=64), 0, 4, "power of two >= 32"),
    (dict(head_dim=64), -32, 4, "power of two >= 32"),
    (dict(head_dim=64), 32, 0, "num_blocks"),
    (dict(head_dim=64), 32, 2 ** 31 - 1, "num_blocks"),
    (dict(head_dim=96), 32, 4, "head_dim 96"),
    (dict(head_dim=0), 32, 4, "invalid configuration"),
    (dict(head_dim=64, max_seq_len=0), 32, 4, "invalid configuration"),
])
def test_configurations_that_are_refused(tlc, cfg, block, blocks, word):
    args = dict(num_layers=1, num_heads=1, max_seq_len=64, max_batch_size=1, **{"head_dim": 64, **cfg})if "max_seq_len" not in cfg \
        else dict(num_layers=1, num_heads=1, max_batch_size=1, **cfg)
    mgr, err = tlc.KVCacheManager.create(block_tokens=block, num_blocks=blocks, quantized=True, **args)
    assert mgr is None and word in err, err


@pytest.mark.parametrize("args,word", [
    (dict(head_dim=80), "head_dim 80"),
    (dict(head_dim=64, rotary_dim=0), "rotary_dim"),
    (dict(head_dim=64, rotary_dim=80), "rotary_dim"),
    (dict(head_dim=64, rotary_dim=40), "rotary_dim"),
    (dict(head_dim=64, theta=0.0), "theta"),
    (dict(head_dim=64, theta=float("inf")), "theta"),
    (dict(head_dim=64, theta=float("nan")), "theta"),
    (dict(head_dim=32, rotary_dim=16, axis_of=[0] * 7 + [8]), "axis 8"),
    (dict(head_dim=32, rotary_dim=16, axis_of=[-1] + [0] * 7), "axis -1"),
    (dict(head_dim=32, rotary_dim=16, inv_freq=[1.0] * 7 + [float("nan")]), "frequency 7"),
])
def test_rotations_that_are_refused(tlc, args, word):
    with pytest.raises(tlc.TinyLLMError, match=word):
        tlc.Rotary(**args)


def test_lists_of_different_lengths(tlc):
    with pytest.raises(ValueError):
        tlc.Rotary(64, axis_of=[0] * 31)
    with pytest.raises(ValueError):
        tlc.Rotary(64, rotary_dim=32, inv_freq=[1.0] * 32)


def apply_args(**kw):
    a = dict(q=0x1000, k=0x100000, q_out=0x200000, k_out=0x300000, positions=0x400000, num_tokens=4, num_q_heads=4,
             num_kv_heads=2)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "q/q_out is null"),
    (dict(q_out=None), "q/q_out is null"),
    (dict(positions=None), "positions is null"),
    (dict(k=None), "both"),
    (dict(k_out=None), "both"),
    (dict(num_tokens=-1), "num_tokens"),
    (dict(num_q_heads=0), "heads"),
    (dict(num_kv_heads=0), "heads"),
    (dict(num_q_heads=65537), "65536"),
    (dict(eps=-1e-5), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(q_stride=255), "strides"),
    (dict(q_stride=260), "strides"),
    (dict(k_stride=64), "strides"),
    (dict(q=0x1008), "aligned"),
    (dict(k_out=0x300002), "aligned"),
    (dict(q_weight=0x500004), "aligned"),
    (dict(positions=0x400002), "aligned"),
    (dict(q_out=0x1200), "q_out overlaps q"),
    (dict(q_out=0x1000, q_stride=512), "q_out overlaps q"),
    (dict(k_out=0x100100), "k_out overlaps k"),
    (dict(q_out=0x100000), "overlap"),
    (dict(k_out=0x1000), "overlap"),
    (dict(k_out=0x200000), "overlap"),
    (dict(q_stride=(1 << 30) + 8), "2\\^30"),
    (dict(k_stride=1 << 62), "2\\^30"),
    (dict(positions=0x200000 + 4 * 256 * 2 - 4), "q_out overlaps positions"),
    (dict(positions=0x300000 - 12), "k_out overlaps positions"),
    (dict(q_weight=0x200100), "q_out overlaps positions or weights"),
    (dict(k_weight=0x300100), "k_out overlaps positions or weights"),
])
def test_rotation_calls_that_are_refused(tlc, kw, word):
    """Before anything is launched: these addresses exist on no device."""
    r = tlc.Rotary(64)
    with pytest.raises(tlc.TinyLLMError, match=word):
        r.apply(**apply_args(**kw))


def test_no_tokens_need_no_launch(tlc):
    tlc.Rotary(64).apply(**apply_args(num_tokens=0))


@pytest.mark.parametrize("obj", ["quant_copy.o", "attention_quant.o", "prefill_quant.o", "rotary.o"])
def test_kernels_use_no_scratch(obj, tmp_path):
    """Registers hold the tiles and the work lists stay in the kernel arguments."""
    for name, r in kernels(obj, tmp_path).items():
        assert r["private_segment_fixed_size"] == 0 and r["vgpr_spill_count"] == 0, (name, r)
        assert r["kernarg_segment_size"] <= 4096, (name, r)
