"""GPU: cross attention of queries over no states, few and many of them."""
import pytest
import torch

from retention_ref import Cache
from test_gpu_cross import cross

pytestmark = pytest.mark.gpu


def launches(tl, call):
    """Launches of the cross and stream kernels (with their merge or finish) in the call."""
    tl.profile_enable(True)
    tl.profile_reset()
    try:
        call()
        torch.cuda.synchronize()
        return sum(tl.profile_query(k)[1] for k in ("attn_stream", "attn_cross"))
    finally:
        tl.profile_enable(False)


def test_padding_is_one_launch(tl):
    """However many queries there are over no states."""
    c = Cache(tl, [8, 100], 1, 32, seed=1, hq=8)
    for src, nq, att in (([0], [2048], [0]), ([0] * 200, [17] * 200, [0] * 200), ([0, 1, 0], [5000, 1, 70], [0, 0, 0])):
        b = tl.CrossBatch(c.mgr, len(src), 8)
        b.prepare([c.ids[j] for j in src], nq, att)
        q = torch.randn((sum(nq), 8, 32), device="cuda").half()
        out = torch.full_like(q, 9.0)
        out = torch.cat([out, out[:1]])
        assert launches(tl, lambda: b.attention(0, q.data_ptr(), out.data_ptr(), 1.0)) == 1
        assert not out[:-1].any() and (out[-1] == 9.0).all()


@pytest.mark.parametrize("d,hkv,G", [(32, 1, 1), (64, 3, 2), (128, 2, 8), (256, 1, 4)])
def test_padding_between_states(tl, d, hkv, G):
    """Ranges of one token to many, more of them than a launch takes, between attended ones."""
    c = Cache(tl, [40, 7], hkv, d, seed=2, hq=hkv * G)
    src = [i % 2 for i in range(600)]
    nq = [1 + (i * 7) % 5 for i in range(600)]
    att = [0 if i % 2 else 40 - i % 9 for i in range(600)]
    cross(tl, c, G, src, nq, att)
    cross(tl, c, G, [0, 1, 0, 1], [1, 3000, 30, 1], [0, 0, 40, 0])


def test_padding_captured(tl):
    c = Cache(tl, [90], 1, 64, seed=3)
    b = tl.CrossBatch(c.mgr, 3, 1)
    b.prepare([c.ids[0]] * 3, [5, 400, 2], [0, 90, 0])
    q = torch.randn((407, 1, 64), device="cuda").half()
    out, want = torch.empty_like(q), torch.empty_like(q)
    b.attention(0, q.data_ptr(), want.data_ptr(), 0.125)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.attention(0, q.data_ptr(), out.data_ptr(), 0.125, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and not out[:5].any() and not out[405:].any()
        b.attention(0, q.data_ptr(), want.data_ptr(), 0.125)
        torch.cuda.synchronize()
