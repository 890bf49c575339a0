"""GPU: eviction from long caches -- every selection kernel above 4096 tokens, the one
beyond 32768 among them, place by place and bit for bit -- and what a captured
eviction moves."""
import numpy as np
import pytest
import torch

from retention_ref import Cache, _Raw, evict
from test_gpu_evict import step, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["tail", "ties", "equal", "wild"])
@pytest.mark.parametrize("lens,budgets,recent", [
    ([4097, 8192], [1000, 8190], 100),      # two tokens a thread of 1024
    ([8193, 16384], [8000, 2048], 0),       # four
    ([16385, 32768], [16000, 4096], 512),   # eight
    ([32769, 20000], [9000, 500], 31),      # no end
])
@pytest.mark.parametrize("block,in_place", [(0, True), (0, False), (16, True), (32, False)])
def test_evict_of_long_caches(tl, kind, lens, budgets, recent, block, in_place):
    c = Cache(tl, lens, 1, 32, block=block, seed=len(kind) + lens[0], spare=1)
    step(tl, c, budgets, recent, [weights(c, kind)], [c.account(-9, torch.int32)], in_place, [(0, 0)] * 2)


@pytest.mark.parametrize("lens,budgets", [([8000, 30000], [300, 20000]), ([40000], [35000])])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_of_long_caches_again(tl, lens, budgets, in_place):
    """On caches that were evicted from: positions from memory below the last length."""
    n = len(lens)
    c = Cache(tl, lens, 2, 32, room=max(lens) + 6000, block=16, seed=21)
    w, pos = [weights(c, "ties")], [c.account(0, torch.int32)]
    w, pos, state = step(tl, c, budgets, 64, w, pos, in_place, [(0, 0)] * n)
    c.append([5000] * n)
    step(tl, c, [b // 2 for b in budgets], 100, [weights(c, "wild")], pos, in_place, state)


@pytest.mark.parametrize("kind", ["tail", "ties"])
def test_evict_of_131072(tl, kind):
    c = Cache(tl, [131072], 1, 32, seed=22)
    step(tl, c, [16384], 512, [weights(c, kind)], [c.account(0, torch.int32)], True, [(0, 0)])


@pytest.mark.parametrize("lens,budgets", [([500, 90], [100, 50]), ([5000], [4998]), ([33000], [700]), ([65, 12], [64, 11])])
def test_a_captured_eviction_moves_the_rows(tl, lens, budgets):
    """The cache as it was before every replay, and only the replay between it and the check."""
    n = len(lens)
    c = Cache(tl, lens, 2, 64, seed=23)
    w, pos = weights(c, "tail"), c.account(0, torch.int32)
    w_out, p_out = c.account(), c.account(0, torch.int32)
    pool = torch.as_tensor(_Raw(c.mgr, c.mgr.getTotalMemory() // 2), device="cuda")
    before = pool.clone()
    ev = tl.EvictBatch(c.mgr, n)
    ev.prepare(c.ids, budgets, 10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ev.run(0, w.data_ptr(), w_out.data_ptr(), pos.data_ptr(), p_out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    ref = w.cpu().numpy()
    for _ in range(3):
        pool.copy_(before)
        w_out.zero_(), p_out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got_w, got_p = w_out.cpu().numpy(), p_out.cpu().numpy()
        for i, (L, keep) in enumerate(zip(lens, budgets)):
            k, v = c.held(0, i, L)
            for h in range(2):
                src = evict(ref[c.slot[i], h, :L], np.arange(L), keep, L - 10)
                assert np.array_equal(k[:keep, h], c.k[0][i][src, h]) and np.array_equal(v[:keep, h], c.v[0][i][src, h])
                assert np.array_equal(k[keep:, h], c.k[0][i][keep:, h]) and np.array_equal(v[keep:, h], c.v[0][i][keep:, h])
                assert np.array_equal(got_p[c.slot[i], h, :keep], src)
                assert np.array_equal(got_w[c.slot[i], h, :keep], ref[c.slot[i], h][src])
    ev.commit()
    assert [c.mgr.getSeqLen(s) for s in c.ids] == budgets
