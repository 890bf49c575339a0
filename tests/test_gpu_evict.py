"""GPU: EvictBatch against a plain selection and compaction, bit for bit, and what
a cache is after it."""
import numpy as np
import pytest
import torch

from retention_ref import Cache, attend, check_account, check_out, dev, evict

pytestmark = pytest.mark.gpu


def weights(c, kind):
    w = c.account()
    g = torch.Generator(device="cuda").manual_seed(17)
    u = torch.rand(w.shape, generator=g, device="cuda")
    if kind == "tail":
        w.copy_(8 * u ** 6)
    elif kind == "ties":
        w.copy_((u * 5).floor())
    elif kind == "equal":
        w.fill_(0.5)
    elif kind == "wild":  # infinities, NaN, both zeros, negative values
        w.copy_(torch.where(u < 0.5, u - 0.25, -u))
        for lo, x in ((0.1, float("inf")), (0.2, float("-inf")), (0.3, float("nan")), (0.4, 0.0), (0.45, -0.0)):
            w[(u > lo) & (u < lo + 0.04)] = x
    return w


def step(tl, c, budgets, recent, w, pos, in_place, before):
    """One eviction over all layers, checked; before[i] = (base, gone)."""
    n = len(c.ids)
    ev = tl.EvictBatch(c.mgr, n)
    ev.prepare(c.ids, budgets, recent)
    lens = [c.mgr.getSeqLen(s) for s in c.ids]
    keeps = [min(a, b) for a, b in zip(lens, budgets)]
    assert ev.info() == {"n": n, "evicted": sum(lens) - sum(keeps)}
    w_new, p_new = [], []
    for layer in range(c.layers):
        w_in, p_in = w[layer], pos[layer]
        w_out = w_in if in_place else torch.full_like(w_in, 3.0)
        p_out = p_in if in_place else torch.full_like(p_in, -3)
        w0, p0, wo0, po0 = (x.cpu().numpy().copy() for x in (w_in, p_in, w_out, p_out))
        ev.run(layer, w_in.data_ptr(), w_out.data_ptr(), p_in.data_ptr(), p_out.data_ptr())
        torch.cuda.synchronize()
        w1, p1 = w_out.cpu().numpy(), p_out.cpu().numpy()
        for i, (L, keep) in enumerate(zip(lens, keeps)):
            base, gone = before[i]
            s = c.slot[i]
            got_k, got_v = c.held(layer, i, L)
            for h in range(c.hkv):
                position = np.where(np.arange(L) < base, p0[s, h, :L], np.arange(L) + gone)
                src = evict(w0[s, h, :L], position, keep, L + gone - recent)
                if in_place and keep == L:
                    assert np.array_equal(p1[s, h], po0[s, h])
                else:
                    assert np.array_equal(p1[s, h, :keep], position[src]), (layer, i, h)
                    assert np.array_equal(p1[s, h, keep:], po0[s, h, keep:])
                assert np.array_equal(w1[s, h, :keep], w0[s, h, :L][src], equal_nan=True)
                assert np.array_equal(w1[s, h, keep:], wo0[s, h, keep:], equal_nan=True)
                for got, ref in ((got_k, c.k[layer][i]), (got_v, c.v[layer][i])):
                    assert np.array_equal(got[:keep, h], ref[src, h])
                    assert np.array_equal(got[keep:, h], ref[keep:, h])
                c.k[layer][i][:keep, h] = c.k[layer][i][src, h]
                c.v[layer][i][:keep, h] = c.v[layer][i][src, h]
        for s in set(range(w1.shape[0])) - set(c.slot):
            assert np.array_equal(w1[s], wo0[s], equal_nan=True) and np.array_equal(p1[s], po0[s])
        w_new.append(w_out)
        p_new.append(p_out)
    ev.commit()
    after = []
    for i, (L, keep) in enumerate(zip(lens, keeps)):
        base, gone = before[i]
        assert c.mgr.getSeqLen(c.ids[i]) == keep and c.mgr.getEvicted(c.ids[i]) == gone + L - keep
        for layer in range(c.layers):
            c.k[layer][i], c.v[layer][i] = c.k[layer][i][:keep], c.v[layer][i][:keep]
        after.append((keep, gone + L - keep) if keep < L else (base, gone))
    assert ev.info() == {"n": 0, "evicted": 0}
    return w_new, p_new, after


@pytest.mark.parametrize("kind", ["tail", "ties", "equal", "wild"])
@pytest.mark.parametrize("d,hkv,block,lens,budgets,recent", [
    (128, 2, 0, [1, 2, 65, 300, 1025], [1, 1, 33, 299, 1024], 0),
    (64, 1, 16, [40, 17, 512, 2100], [40, 60, 100, 1000], 37),
    (32, 3, 0, [1500, 1024, 1025, 90], [3, 1023, 1, 89], 1),
    (256, 1, 32, [33, 500], [32, 250], 32),
])
def test_evict(tl, kind, d, hkv, block, lens, budgets, recent):
    c = Cache(tl, lens, hkv, d, block=block, seed=d, spare=1)
    budgets = [max(b, recent) for b in budgets]
    pos = [c.account(-9, torch.int32)]
    step(tl, c, budgets, recent, [weights(c, kind)], pos, False, [(0, 0)] * len(lens))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("block", [0, 16])
def test_evict_again_and_again(tl, block, in_place):
    """Evictions between appends, two layers: positions go on through them."""
    c = Cache(tl, [300, 20, 77], 2, 64, room=320, block=block, layers=2, seed=3)
    w, pos = [weights(c, "ties") for _ in range(2)], [c.account(0, torch.int32) for _ in range(2)]
    state = [(0, 0)] * 3
    for new, budgets, recent in (([0, 0, 0], [64, 64, 64], 8), ([1, 1, 1], [64, 64, 64], 8), ([40, 0, 3], [90, 10, 64], 10),
                                 ([200, 1, 100], [32, 64, 33], 32)):
        c.append(new)
        w, pos, state = step(tl, c, budgets, recent, w, pos, in_place, state)
    assert state[0][1] == 300 + 1 + 40 + 200 - 32


def test_evict_long(tl):
    """More tokens than a workgroup holds in one go, and more entries than a launch takes."""
    c = Cache(tl, [40000], 1, 32, seed=4)
    step(tl, c, [17000], 100, [weights(c, "tail")], [c.account(0, torch.int32)], True, [(0, 0)])
    lens = [1 + (i * 13) % 60 for i in range(150)]
    c = Cache(tl, lens, 1, 32, block=16, seed=5)
    step(tl, c, [20] * 150, 5, [weights(c, "ties")], [c.account(0, torch.int32)], True, [(0, 0)] * 150)


def test_evict_returns_blocks(tl):
    c = Cache(tl, [100, 64, 30], 1, 32, room=128, block=16, seed=6, blocks=14)
    assert c.mgr.freeBlocks() == 14 - 7 - 4 - 2
    tables = [c.mgr.blockTable(s)[0] for s in c.ids]
    w, pos = c.account(), c.account(0, torch.int32)
    step(tl, c, [33, 64, 16], 16, [w], [pos], True, [(0, 0)] * 3)
    assert c.mgr.freeBlocks() == 14 - 3 - 4 - 1
    assert [c.mgr.blockTable(s)[0] for s in c.ids] == [tables[0][:3], tables[1], tables[2][:1]]
    with pytest.raises(tl.TinyLLMError, match="exhausted"):
        c.append([0, 50, 40])  # 4 + 3 blocks of the 6
    c.append([0, 50, 30])  # 4 + 2: the freed blocks, to other sequences
    for i in range(3):
        got = c.held(0, i, c.mgr.getSeqLen(c.ids[i]))
        assert np.array_equal(got[0], c.k[0][i]) and np.array_equal(got[1], c.v[0][i])


def test_evict_with_a_block_map(tl):
    mgr = tl.KVCacheManager(num_layers=1, num_heads=2, head_dim=64, max_seq_len=64, max_batch_size=2)
    assert mgr.setBlockMap(16, np.array([5, 2, 7, 0, 3, 6, 1, 4])) is None
    sid, _ = mgr.allocateSequence(64)
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((60, 2, 64)).astype(np.float16) for _ in range(2))
    dk, dv = dev(k), dev(v)
    assert mgr.appendKV(sid, 0, dk.data_ptr(), dv.data_ptr(), 60) is None
    mgr.advanceSeqLen(sid, 60)
    w = dev(rng.random((2, 2, 64)).astype(np.float32))
    pos = torch.zeros((2, 2, 64), dtype=torch.int32, device="cuda")
    ref = w.cpu().numpy()[0]
    ev = tl.EvictBatch(mgr, 1)
    ev.prepare([sid], [25], 4)
    ev.run(0, w.data_ptr(), w.data_ptr(), pos.data_ptr(), pos.data_ptr())
    ev.commit()
    out = [torch.zeros((1, 2, 25, 64), dtype=torch.float16, device="cuda") for _ in range(2)]
    b = tl.DecodeBatch(mgr, 1, 2)
    b.prepare_lengths([sid], [25])
    b.gather(0, out[0].data_ptr(), out[1].data_ptr(), 25)
    torch.cuda.synchronize()
    for h in range(2):
        src = evict(ref[h, :60], np.arange(60), 25, 56)
        assert np.array_equal(out[0][0, h].cpu().numpy(), k[src, h])
        assert np.array_equal(out[1][0, h].cpu().numpy(), v[src, h])
        assert np.array_equal(pos[0, h, :25].cpu().numpy(), src)


def test_positions_memory_needs_no_initial_value(tl):
    """Whatever the positions hold, what is written stays in bounds and in order."""
    for garbage in (2 ** 31 - 1, -2 ** 31):
        c = Cache(tl, [200], 1, 32, seed=7)
        step(tl, c, [50], 10, [weights(c, "tail")], [c.account(garbage, torch.int32)], True, [(0, 0)])
        # a caller that hands in other positions than the last eviction wrote: still `keep` tokens
        c.append([30])
        w, pos = weights(c, "tail"), c.account(garbage, torch.int32)
        ev = tl.EvictBatch(c.mgr, 1)
        ev.prepare(c.ids, [60], 10)
        ev.run(0, w.data_ptr(), w.data_ptr(), pos.data_ptr(), pos.data_ptr())
        ev.commit()
        k, v = c.held(0, 0, 60)
        assert np.isfinite(k).all() and c.mgr.getSeqLen(c.ids[0]) == 60


def test_evict_captured(tl):
    c = Cache(tl, [500, 90], 2, 64, seed=8)
    w, pos = weights(c, "tail"), c.account(0, torch.int32)
    w_out, p_out = c.account(), c.account(0, torch.int32)
    ev = tl.EvictBatch(c.mgr, 2)
    ev.prepare(c.ids, [100, 50], 10)

    def call():
        ev.run(0, w.data_ptr(), w_out.data_ptr(), pos.data_ptr(), p_out.data_ptr(), torch.cuda.current_stream().cuda_stream)

    call()
    torch.cuda.synchronize()
    want = w_out.clone(), p_out.clone(), c.held(0, 0, 100)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):  # the moved rows' sources stay: again gives the same
        w_out.zero_(), p_out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w_out, want[0]) and torch.equal(p_out, want[1])
        call()
        torch.cuda.synchronize()
    ev.commit()
    got = c.held(0, 0, 100)
    assert np.array_equal(got[0], want[2][0]) and np.array_equal(got[1], want[2][1])


def test_evict_refusals(tl):
    c = Cache(tl, [20, 30], 1, 32, layers=2, seed=9)
    ev = tl.EvictBatch(c.mgr, 2)
    a, b = c.ids
    for ids, bud, rec, msg in (([a], [0], 0, "positive"), ([a], [-5], 0, "positive"), ([a], [5], 6, "newest"),
                               ([a], [5], -1, "recent"), ([a, a], [5, 5], 0, "duplicate"), ([99], [5], 0, "not found"),
                               ([a, b, a], [5, 5, 5], 0, "outside")):
        with pytest.raises(tl.TinyLLMError, match=msg):
            ev.prepare(ids, bud, rec)
        assert ev.info() == {"n": 0, "evicted": 0}
    with pytest.raises(ValueError):
        ev.prepare([a], [5, 6])
    w, p = c.account(), c.account(0, torch.int32)
    w2, p2 = c.account(), c.account(0, torch.int32)
    W, P, W2, P2 = (x.data_ptr() for x in (w, p, w2, p2))
    ev.prepare([a, b], [5, 30], 5)
    for args, msg in (((2, W, W, P, P), "layer_idx"), ((-1, W, W, P, P), "layer_idx"), ((0, None, W, P, P), "null"),
                      ((0, W, None, P, P), "null"), ((0, W, W, None, P), "null"), ((0, W, W, P, None), "null"),
                      ((0, W + 1, W, P, P), "aligned"), ((0, W, W + 4, P, P), "overlaps"), ((0, W, P, P, P2), "overlaps"),
                      ((0, W, W, P, P + 8), "overlaps"), ((0, W, W2, P, W2), "overlaps")):
        with pytest.raises(tl.TinyLLMError, match=msg):
            ev.run(*args)
    with pytest.raises(tl.TinyLLMError, match="layer 0 has not run"):
        ev.commit()
    ev.run(0, W, W2, P, P2)
    ev.run(0, W, W, P, P)  # the first left everything as it found it
    with pytest.raises(tl.TinyLLMError, match="in place"):
        ev.run(0, W, W, P, P)
    with pytest.raises(tl.TinyLLMError, match="layer 1 has not run"):
        ev.commit()
    ev.run(1, W2, W2, P2, P2)
    c.mgr.advanceSeqLen(a, 1)
    with pytest.raises(tl.TinyLLMError, match="changed"):
        ev.commit()
    with pytest.raises(tl.TinyLLMError, match="changed"):
        ev.run(1, W, W2, P, P2)
    assert c.mgr.getSeqLen(a) == 21 and c.mgr.getEvicted(a) == 0
    c.mgr.releaseSequence(a)
    with pytest.raises(tl.TinyLLMError, match="not found"):
        ev.commit()
    ev.prepare([b], [40], 5)  # nothing to take: every layer may be left out
    ev.commit()
    assert c.mgr.getSeqLen(b) == 30 and c.mgr.getEvicted(b) == 0 and c.mgr.getEvicted(a) == 0
    ev.commit()  # empty
    torch.cuda.synchronize()


def test_an_eviction_that_has_begun_is_committed_first(tl):
    """Its rows have moved: a second selection would read what the first overwrote."""
    c = Cache(tl, [30, 40], 1, 32, layers=2, seed=14)
    w, p = weights(c, "tail"), c.account(0, torch.int32)
    w2, p2 = c.account(), c.account(0, torch.int32)
    W, P, W2, P2 = (x.data_ptr() for x in (w, p, w2, p2))
    first, second, third = (tl.EvictBatch(c.mgr, 2) for _ in range(3))
    for ev in (first, second):
        ev.prepare(c.ids, [10, 50], 2)
    first.run(0, W, W2, P, P2)
    want = w2.clone(), p2.clone()
    with pytest.raises(tl.TinyLLMError, match="not committed"):
        second.run(0, W, W2, P, P2)
    with pytest.raises(tl.TinyLLMError, match="not committed"):
        first.prepare(c.ids, [10, 50], 2)
    assert first.info() == {"n": 2, "evicted": 20}
    with pytest.raises(tl.TinyLLMError, match="not committed"):
        third.prepare(c.ids[:1], [5], 2)
    assert third.info()["n"] == 0
    third.prepare(c.ids[1:], [5], 2)  # nothing of it was taken
    second.close()
    for layer in (0, 1):
        first.run(layer, W, W2, P, P2)
    first.commit()
    torch.cuda.synchronize()
    assert torch.equal(w2[0, :, :10], want[0][0, :, :10]) and torch.equal(p2[0, :, :10], want[1][0, :, :10])
    assert [c.mgr.getSeqLen(s) for s in c.ids] == [10, 40]
    third.close()
    third = tl.EvictBatch(c.mgr, 2)
    third.prepare(c.ids, [5, 5], 2)
    third.run(0, W2, W2, P2, P2)
    third.close()  # abandoned: the sequences are for release
    with pytest.raises(tl.TinyLLMError, match="not committed"):
        first.prepare(c.ids, [5, 5], 2)
    for s in c.ids:
        c.mgr.releaseSequence(s)
    sid, _ = c.mgr.allocateSequence(30)
    c.mgr.advanceSeqLen(sid, 6)
    first.prepare([sid], [6], 2)
    torch.cuda.synchronize()


def test_evict_prepared_in_a_capture_does_not_grow_the_workspace(tl):
    c = Cache(tl, [300], 1, 32, seed=15)
    ev = tl.EvictBatch(c.mgr, 1)
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x.add_(1)  # a capture of something
        with pytest.raises(tl.TinyLLMError, match="captured"):
            ev.prepare(c.ids, [100], 0, torch.cuda.current_stream().cuda_stream)
    assert ev.info()["n"] == 0


def test_evict_millions_of_tokens(tl):
    """More pairs than a grid has blocks for; all of the newest half stays."""
    n = 4 * 2 ** 20 + 77
    keep = n // 2
    mgr = tl.KVCacheManager(num_layers=1, num_heads=1, head_dim=32, max_seq_len=n, max_batch_size=1)
    sid, _ = mgr.allocateSequence(n)
    k, v = (torch.randn((n, 1, 32), device="cuda", dtype=torch.float16) for _ in range(2))
    assert mgr.appendKV(sid, 0, k.data_ptr(), v.data_ptr(), n) is None
    mgr.advanceSeqLen(sid, n)
    w = torch.arange(n, device="cuda", dtype=torch.float32)[None, None].contiguous()  # exact below 2^24
    pos = torch.zeros((1, 1, n), dtype=torch.int32, device="cuda")
    ev = tl.EvictBatch(mgr, 1)
    ev.prepare([sid], [keep], 0)
    ev.run(0, w.data_ptr(), w.data_ptr(), pos.data_ptr(), pos.data_ptr())
    ev.commit()
    out = [torch.empty((1, 1, keep, 32), dtype=torch.float16, device="cuda") for _ in range(2)]
    b = tl.DecodeBatch(mgr, 1, 1)
    b.prepare_lengths([sid], [keep])
    b.gather(0, out[0].data_ptr(), out[1].data_ptr(), keep)
    torch.cuda.synchronize()
    src = torch.arange(n - keep, n, device="cuda")  # movers in order to all places
    assert torch.equal(pos[0, 0, :keep].long(), src) and torch.equal(w[0, 0, :keep], src.float())
    assert torch.equal(out[0][0, 0], k[src, 0]) and torch.equal(out[1][0, 0], v[src, 0])


def test_a_slot_starts_anew(tl):
    c = Cache(tl, [30], 1, 32, room=64, seed=10)
    step(tl, c, [10], 2, [weights(c, "tail")], [c.account(0, torch.int32)], True, [(0, 0)])
    assert c.mgr.getEvicted(c.ids[0]) == 20
    c.mgr.releaseSequence(c.ids[0])
    sid, _ = c.mgr.allocateSequence(64)
    assert c.mgr.getEvicted(sid) == 0 and c.mgr.getSeqLen(sid) == 0


@pytest.mark.parametrize("block", [0, 16])
def test_a_bounded_cache_from_prompt_to_tokens(tl, block):
    """Prompt, its account, an eviction, then steps that each append, attend, count
    and evict, on two layers: every attention is the 64-bit attention over the
    tokens that the positions name."""
    hkv, G, d, budget, recent, layers = 2, 4, 64, 48, 16, 2
    hq, scale = hkv * G, d ** -0.5
    rng = np.random.default_rng(1)
    prompts, steps = [130, 40, 77], 12
    total = [p + steps for p in prompts]
    n = len(prompts)
    args = dict(num_layers=layers, num_heads=hkv, head_dim=d, max_seq_len=160, max_batch_size=n)
    if block:
        args.update(block_tokens=block, num_blocks=30)
    mgr = tl.KVCacheManager(**args)
    ids = [mgr.allocateSequence(160)[0] for _ in prompts]
    K, V = ([[rng.standard_normal((t, hkv, d)).astype(np.float16) for t in total] for _ in range(layers)] for _ in range(2))
    Q = [[rng.standard_normal((t, hq, d)).astype(np.float16) for t in total] for _ in range(layers)]
    acc = [torch.zeros((n, hkv, 160), device="cuda") for _ in range(layers)]
    pos = [torch.zeros((n, hkv, 160), dtype=torch.int32, device="cuda") for _ in range(layers)]
    slot = [mgr.slot_of(s) for s in ids]
    pf, dec, ev = tl.PrefillBatch(mgr, n, hq), tl.DecodeBatch(mgr, n, hq), tl.EvictBatch(mgr, n)
    pf.prepare(ids, prompts)
    keep_alive = []
    for layer in range(layers):
        q, k, v = (dev(np.concatenate([x[layer][i][:p] for i, p in enumerate(prompts)])) for x in (Q, K, V))
        out = torch.empty_like(q)
        pf.run(layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), scale)
        pf.weights(layer, q.data_ptr(), scale, 20, None, acc[layer].data_ptr())
        keep_alive += [q, k, v, out]
    pf.commit()

    def evict_all(recent):
        ev.prepare(ids, [budget] * n, recent)
        for layer in range(layers):
            w, p = acc[layer].data_ptr(), pos[layer].data_ptr()
            ev.run(layer, w, w, p, p)
        ev.commit()

    evict_all(recent)
    held = [min(p, budget) for p in prompts]
    left = list(held)  # lengths right after the last eviction that took something
    for t in range(steps):
        assert [mgr.getSeqLen(s) for s in ids] == held
        assert [mgr.getSeqLen(s) + mgr.getEvicted(s) for s in ids] == [p + t for p in prompts]
        dec.prepare(ids)
        for layer in range(layers):
            q, k, v = (dev(np.stack([x[layer][i][p + t] for i, p in enumerate(prompts)])) for x in (Q, K, V))
            out = torch.empty_like(q)
            before = acc[layer].cpu().numpy()
            w = acc[layer].data_ptr()
            dec.decode_weights(layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), scale, w, w)
            torch.cuda.synchronize()
            got, after, where = out.cpu().numpy(), acc[layer].cpu().numpy(), pos[layer].cpu().numpy()
            for i in range(n):
                S = held[i] + 1
                for h in range(hkv):
                    # positions below what the last eviction left are stored, later ones follow
                    src = np.arange(S) + mgr.getEvicted(ids[i])
                    if mgr.getEvicted(ids[i]):
                        src[:left[i]] = where[slot[i], h, :left[i]]
                    assert src[-1] == prompts[i] + t and len(set(src)) == S
                    qs = Q[layer][i][prompts[i] + t:prompts[i] + t + 1, h * G:h * G + G]
                    o, mass, wt, err = attend(qs, K[layer][i][src, h:h + 1], V[layer][i][src, h:h + 1], scale)
                    check_out(got[i:i + 1, h * G:h * G + G], o, mass, err, S)
                    base = before[slot[i], h:h + 1, :S].astype(np.float64)
                    base[:, -1] = 0
                    check_account(after[slot[i], h:h + 1, :S], wt.sum(axis=0) + base, wt, err, G, S, base)
        dec.commit(1)
        held = [h + 1 for h in held]
        if t % 3 != 1:  # not after every token
            evict_all(recent)
            left = [budget if h > budget else b for h, b in zip(held, left)]
            held = [min(h, budget) for h in held]
