"""GPU: CrossBatch -- queries over cached states of another length -- against 64-bit
attention, elementwise within bounds derived from the roundings of the path."""
import numpy as np
import pytest
import torch

from retention_ref import Cache, attend, check_out, dev, even_tail

pytestmark = pytest.mark.gpu


def cross(tl, c, G, src, nq, att=None, layer=0, scale=None):
    hq, d = c.hkv * G, c.d
    scale = scale or d ** -0.5
    t = sum(nq)
    q = c.rng.standard_normal((t, hq, d)).astype(np.float16)
    b = tl.CrossBatch(c.mgr, len(src), hq)
    s = torch.cuda.current_stream().cuda_stream
    b.prepare([c.ids[j] for j in src], nq, att, s)
    assert b.info() == {"n": len(src), "tokens": t}
    dq = dev(q)
    out = torch.full((t + 3, hq, d), 9.0, dtype=torch.float16, device="cuda")
    b.attention(layer, dq.data_ptr(), out.data_ptr(), scale, s)
    torch.cuda.synchronize()
    got, at = out.cpu().numpy(), 0
    for i, (j, n) in enumerate(zip(src, nq)):
        a = len(c.k[layer][j]) if att is None else att[i]
        o, mass, _, err = attend(q[at:at + n], c.k[layer][j][:a], c.v[layer][j][:a], scale)
        check_out(got[at:at + n], o, mass, err, a)
        at += n
    assert (got[t:] == 9.0).all()  # rows behind the last entry
    return got


@pytest.mark.parametrize("d,hkv,G,block,states,src,nq", [
    (64, 8, 1, 0, [1500], [0, 0, 0], [1, 1, 1]),
    (64, 2, 1, 0, [1, 63, 64, 65, 700], [0, 1, 2, 3, 4], [1, 5, 16, 17, 100]),
    (128, 2, 4, 0, [300, 17], [1, 0, 1], [3, 130, 64]),
    (128, 1, 8, 16, [15, 16, 500], [0, 1, 2, 2], [33, 2, 1, 200]),
    (256, 1, 2, 32, [129, 40], [0, 1], [70, 9]),
    (32, 3, 8, 64, [200, 5], [1, 0], [40, 3]),
    (256, 2, 8, 0, [64], [0], [31]),
    (32, 1, 1, 0, [33], [0], [257]),
    (128, 1, 1, 16, [5000], [0], [300]),
    (128, 2, 2, 0, [2300], [0, 0], [4, 1]),
])
def test_cross(tl, d, hkv, G, block, states, src, nq):
    c = Cache(tl, states, hkv, d, block=block, seed=d + G, hq=hkv * G)
    cross(tl, c, G, src, nq)


@pytest.mark.parametrize("d,hkv,G,block,states,nq", [
    (64, 8, 1, 0, [1500, 900], [1, 3]),      # few rows, little work: pieces of four tiles
    (32, 4, 2, 16, [3000], [2]),
    (256, 4, 4, 0, [3000], [2]),
    (128, 8, 4, 0, [16500], [1]),            # more: eight waves
    (128, 1, 1, 0, [40, 700], [16, 1]),      # whole entries
    (128, 8, 4, 16, [3000], [8]),            # tiles half empty
    (64, 2, 4, 0, [3000], [30]),
    (256, 2, 4, 16, [2500], [20]),
    (32, 2, 8, 16, [3000], [40]),
    (128, 2, 4, 0, [2000], [100]),           # large workgroups, keys split
    (32, 8, 4, 0, [700, 300], [130, 257]),
    (128, 8, 1, 0, [200] * 32, [300] * 32),  # ... one round and a part of another
])
def test_cross_in_pieces(tl, d, hkv, G, block, states, nq):
    c = Cache(tl, states, hkv, d, block=block, seed=d + G + 1, hq=hkv * G)
    cross(tl, c, G, list(range(len(states))), nq)


@pytest.mark.parametrize("block", [0, 16])
@pytest.mark.parametrize("nq", [[1, 2, 1, 3], [40, 150, 64, 1]])
def test_cross_over_padded_states(tl, block, nq):
    """Attended lengths short of the states, none at all, one."""
    c = Cache(tl, [400, 90], 2, 64, block=block, seed=2, hq=4)
    got = cross(tl, c, 2, [0, 1, 0, 1], nq, [333, 0, 1, 89])
    assert not got[nq[0]:nq[0] + nq[1]].any()


def test_cross_without_any_states(tl):
    c = Cache(tl, [0, 8], 1, 64, seed=3)
    assert not cross(tl, c, 1, [0], [5])[:5].any()
    assert not cross(tl, c, 1, [0, 0], [200, 3])[:203].any()


def test_cross_more_entries_than_a_launch_takes(tl):
    c = Cache(tl, [50, 7, 200], 1, 32, block=16, seed=4, hq=2)
    cross(tl, c, 2, [i % 3 for i in range(170)], [1 + i % 2 for i in range(170)])
    cross(tl, c, 2, [i % 3 for i in range(170)], [20 + i % 60 for i in range(170)])


def test_cross_layers_scales_and_another_stream(tl):
    c = Cache(tl, [100, 333], 2, 64, layers=3, seed=5, hq=4)
    with torch.cuda.stream(torch.cuda.Stream()):
        cross(tl, c, 2, [1, 0], [3, 90], layer=2)
        cross(tl, c, 2, [1, 0], [90, 1], layer=0, scale=1.7)
        cross(tl, c, 2, [1, 0], [2, 2], layer=1, scale=-0.5)


@pytest.mark.parametrize("scale", [-0.5, 1e-30, 2.0])
@pytest.mark.parametrize("nq", [[2, 1], [90, 300]])
def test_cross_scales_of_either_sign(tl, nq, scale):
    c = Cache(tl, [100, 333], 2, 64, seed=15, hq=4)
    cross(tl, c, 2, [1, 0], nq, scale=scale)


@pytest.mark.parametrize("nq", [2, 200])
def test_cross_scale_of_zero(tl, nq):
    """Every state has the same weight, and those past the end none."""
    c = Cache(tl, [100], 1, 64, seed=16, hq=2)
    q = torch.randn((nq, 2, 64), device="cuda").half()
    out = torch.empty_like(q)
    b = tl.CrossBatch(c.mgr, 1, 2)
    b.prepare(c.ids, [nq])
    b.attention(0, q.data_ptr(), out.data_ptr(), 0.0)
    torch.cuda.synchronize()
    mean = c.v[0][0][:, 0].astype(np.float64).mean(axis=0)
    # the output's rounding, values below 1
    assert np.abs(out.cpu().numpy().astype(np.float64) - mean).max() <= 2.0 ** -11


@pytest.mark.parametrize("nq,d", [(1, 64), (16, 128), (200, 128), (300, 64), (40, 256)])
def test_cross_weights_far_below_the_largest(tl, nq, d):
    c, q, want, tol = even_tail(tl, 4096, d)
    dq = dev(np.tile(q, (nq, 1, 1)))
    out = torch.empty_like(dq)
    b = tl.CrossBatch(c.mgr, 1, 1)
    b.prepare(c.ids, [nq])
    b.attention(0, dq.data_ptr(), out.data_ptr(), 1.0)
    torch.cuda.synchronize()
    assert np.abs(out.cpu().numpy().astype(np.float64) - want).max() <= tol


def test_cross_neighbours_over_the_same_states(tl):
    """They are worked on as one, also where a padded or another one is between."""
    c = Cache(tl, [300, 40], 2, 128, seed=17, hq=8)
    cross(tl, c, 4, [0] * 7 + [1, 0, 0], [1, 1, 2, 1, 1, 1, 1, 1, 3, 90], [300, 300, 300, 10, 300, 300, 0, 40, 300, 300])


@pytest.mark.parametrize("nq", [[2, 1], [70, 300]])
def test_cross_captured(tl, nq):
    c = Cache(tl, [700, 90], 2, 64, seed=6, hq=4)
    b = tl.CrossBatch(c.mgr, 2, 4)
    b.prepare(c.ids, nq)
    q = torch.randn((sum(nq), 4, 64), device="cuda").half()
    out = torch.zeros_like(q)

    def call():
        b.attention(0, q.data_ptr(), out.data_ptr(), 0.125, torch.cuda.current_stream().cuda_stream)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(4):
        q.normal_()
        call()
        torch.cuda.synchronize()
        want = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_cross_of_one_token_is_decode_attention(tl):
    """The same attention as DecodeBatch over given lengths."""
    c = Cache(tl, [900, 64, 333], 2, 128, seed=7, hq=8)
    q = torch.randn((3, 8, 128), device="cuda").half()
    out, ref = torch.empty_like(q), torch.empty_like(q)
    b, d = tl.CrossBatch(c.mgr, 3, 8), tl.DecodeBatch(c.mgr, 3, 8)
    b.prepare(c.ids, [1, 1, 1])
    b.attention(0, q.data_ptr(), out.data_ptr(), 128 ** -0.5)
    d.prepare_lengths(c.ids, [900, 64, 333])
    d.attention(0, q.data_ptr(), ref.data_ptr(), 128 ** -0.5)
    torch.cuda.synchronize()
    # two roundings to fp16 of each: of the weights and of the outputs, which are below 4
    assert (out.float() - ref.float()).abs().max() <= 4 * 4 * 2.0 ** -11


def test_cross_refusals(tl):
    c = Cache(tl, [20, 30], 2, 64, seed=8, hq=4)
    b = tl.CrossBatch(c.mgr, 3, 4)
    a = c.ids[0]
    for ids, nq, att, msg in (([a], [0], None, "positive"), ([a], [-1], None, "positive"), ([77], [1], None, "not found"),
                              ([a], [1], [21], "outside"), ([a], [1], [-1], "outside"), ([a] * 4, [1] * 4, None, "outside"),
                              ([a, a], [2 ** 30, 2 ** 30], None, "too many")):
        with pytest.raises(tl.TinyLLMError, match=msg):
            b.prepare(ids, nq, att)
        assert b.info() == {"n": 0, "tokens": 0}
    with pytest.raises(ValueError):
        b.prepare([a], [1], [1, 2])
    q = torch.zeros((4, 4, 64), dtype=torch.float16, device="cuda")
    p = q.data_ptr()
    b.attention(0, p, p, 1.0)  # empty: nothing to do
    b.prepare([a, a], [1, 2])
    for args, msg in (((1, p, p, 1.0), "layer_idx"), ((0, None, p, 1.0), "null"), ((0, p, None, 1.0), "null"),
                      ((0, p + 2, p, 1.0), "aligned"), ((0, p, p + 8, 1.0), "aligned")):
        with pytest.raises(tl.TinyLLMError, match=msg):
            b.attention(*args)
    c.mgr.releaseSequence(a)
    with pytest.raises(tl.TinyLLMError, match="not found"):
        b.attention(0, p, p, 1.0)
    for hq in (0, 3, 32):
        with pytest.raises(tl.TinyLLMError):
            tl.CrossBatch(c.mgr, 1, hq)
    with pytest.raises(tl.TinyLLMError):
        tl.CrossBatch(c.mgr, 0, 4)
