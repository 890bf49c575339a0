"""GPU: an eviction between the other calls of a serving loop -- sequences released,
grown or appended to while it is under way."""
import numpy as np
import pytest
import torch

from retention_ref import Cache, dev, evict
from test_gpu_evict import weights

pytestmark = pytest.mark.gpu


class Running:
    """An eviction of all of a cache's sequences, run and committed by hand."""

    def __init__(self, tl, c, budgets, recent=2):
        self.c, self.budgets, self.recent, n = c, budgets, recent, len(c.ids)
        self.w, self.pos = [weights(c, "tail") for _ in range(c.layers)], [c.account(0, torch.int32) for _ in range(c.layers)]
        self.w0 = [w.cpu().numpy() for w in self.w]
        self.lens = [c.mgr.getSeqLen(s) for s in c.ids]
        self.ev = tl.EvictBatch(c.mgr, n)
        self.ev.prepare(c.ids, budgets, recent)

    def run(self, layer):
        w, p = self.w[layer].data_ptr(), self.pos[layer].data_ptr()
        self.ev.run(layer, w, w, p, p)

    def check(self, i):
        """Sequence i is what the eviction leaves of it."""
        c, L, keep = self.c, self.lens[i], min(self.lens[i], self.budgets[i])
        torch.cuda.synchronize()
        assert c.mgr.getSeqLen(c.ids[i]) == keep and c.mgr.getEvicted(c.ids[i]) == L - keep
        for layer in range(c.layers):
            k, v = c.held(layer, i, keep)
            w, p = self.w[layer].cpu().numpy(), self.pos[layer].cpu().numpy()
            for h in range(c.hkv):
                src = evict(self.w0[layer][c.slot[i], h, :L], np.arange(L), keep, L - self.recent)
                assert np.array_equal(k[:, h], c.k[layer][i][src, h]) and np.array_equal(v[:, h], c.v[layer][i][src, h])
                assert np.array_equal(w[c.slot[i], h, :keep], self.w0[layer][c.slot[i], h][src])
                assert np.array_equal(p[c.slot[i], h, :keep], src)


@pytest.mark.parametrize("block", [0, 16])
@pytest.mark.parametrize("when", [0, 1, 2])  # before the first layer, between the two, before the commit
@pytest.mark.parametrize("who", [0, 1, 2])
def test_a_released_sequence_leaves_the_eviction(tl, block, when, who):
    """The others are committed without it, and can be evicted from again."""
    c = Cache(tl, [60, 150, 90], 2, 32, block=block, layers=2, seed=31)
    r = Running(tl, c, [20, 40, 60])
    for layer in range(3):
        if layer == when:
            c.mgr.releaseSequence(c.ids[who])
            other, _ = c.mgr.allocateSequence(30)  # in its slot
            assert c.mgr.slot_of(other) == c.slot[who]
        if layer < 2:
            r.run(layer)
    r.ev.commit()
    assert r.ev.info() == {"n": 0, "evicted": 0}
    left = [i for i in range(3) if i != who]
    for i in left:
        r.check(i)
    assert c.mgr.getEvicted(other) == 0 and c.mgr.getSeqLen(other) == 0
    again = tl.EvictBatch(c.mgr, 2)
    again.prepare([c.ids[i] for i in left], [10, 10], 2)
    again.run(0, r.w[0].data_ptr(), r.w[0].data_ptr(), r.pos[0].data_ptr(), r.pos[0].data_ptr())
    again.run(1, r.w[1].data_ptr(), r.w[1].data_ptr(), r.pos[1].data_ptr(), r.pos[1].data_ptr())
    again.commit()
    assert [c.mgr.getSeqLen(c.ids[i]) for i in left] == [10, 10]
    torch.cuda.synchronize()


def test_an_eviction_of_released_sequences_only(tl):
    c = Cache(tl, [30, 40], 1, 32, seed=32)
    r = Running(tl, c, [10, 40])
    r.run(0)
    c.mgr.releaseSequence(c.ids[0])
    with pytest.raises(tl.TinyLLMError, match="not found"):
        r.ev.commit()
    r.ev.prepare(c.ids[1:], [5], 1)  # and the batch is free
    c.mgr.releaseSequence(c.ids[1])
    with pytest.raises(tl.TinyLLMError, match="not found"):
        r.run(0)
    r.ev.prepare([], [], 0)
    torch.cuda.synchronize()


@pytest.mark.parametrize("when", [0, 1, 2])
def test_a_sequence_that_keeps_all_may_change_meanwhile(tl, when):
    """It grows, or another batch evicts from it."""
    c = Cache(tl, [80, 30, 30], 2, 32, room=120, layers=2, seed=33)
    r = Running(tl, c, [20, 50, 50])
    for layer in range(3):
        if layer == when:
            p = tl.PrefillBatch(c.mgr, 1, 2)
            p.prepare([c.ids[1]], [5])
            k = dev(c.rows(5))
            for x in range(2):
                p.append(x, k.data_ptr(), k.data_ptr())
            p.commit()
            other = tl.EvictBatch(c.mgr, 1)
            other.prepare([c.ids[2]], [7], 2)
            w, pos = c.account(), c.account(0, torch.int32)
            for x in range(2):
                other.run(x, w.data_ptr(), w.data_ptr(), pos.data_ptr(), pos.data_ptr())
            other.commit()
        if layer < 2:
            r.run(layer)
    r.ev.commit()
    r.check(0)
    assert [c.mgr.getSeqLen(s) for s in c.ids] == [20, 35, 7] and [c.mgr.getEvicted(s) for s in c.ids] == [60, 0, 23]


def test_a_sequence_that_grew_after_its_rows_moved(tl):
    """It cannot be committed; once it is released the others are."""
    c = Cache(tl, [50, 80], 1, 32, room=100, seed=34)
    r = Running(tl, c, [20, 20])
    r.run(0)
    c.mgr.advanceSeqLen(c.ids[0], 1)
    with pytest.raises(tl.TinyLLMError, match="changed"):
        r.ev.commit()
    c.mgr.releaseSequence(c.ids[0])
    r.ev.commit()
    r.check(1)


@pytest.mark.parametrize("block", [0, 16])
def test_an_eviction_under_way_refuses_other_steps(tl, block):
    """Appends, steps that would append, attention to the states, and the commits of
    steps that were prepared before; after the commit all of it goes on."""
    c = Cache(tl, [50, 80, 10], 1, 32, room=112, block=block, layers=2, seed=35)
    a, b, free = c.ids  # nothing is taken from the last one
    k = dev(c.rows(4))
    K = k.data_ptr()
    dec, pf, cross = tl.DecodeBatch(c.mgr, 3, 1), tl.PrefillBatch(c.mgr, 3, 1), tl.CrossBatch(c.mgr, 2, 1)
    dec.prepare(c.ids)
    pf.prepare([b], [2])
    r = Running(tl, c, [20, 20, 20])
    r.run(0)
    msg = "eviction of sequence {} has run and is not committed"
    for call, who in ((lambda: tl.DecodeBatch(c.mgr, 1, 1).prepare([a]), a), (lambda: dec.commit(1), a), (lambda: pf.commit(), b),
                      (lambda: tl.PrefillBatch(c.mgr, 2, 1).prepare([free, b], [1, 1]), b),
                      (lambda: cross.prepare([free, b], [1, 1]), b)):
        with pytest.raises(tl.TinyLLMError, match=msg.format(who)):
            call()
    assert msg.format(a) in c.mgr.appendKV(a, 0, K, K, 2)
    assert [c.mgr.getSeqLen(s) for s in c.ids] == [50, 80, 10]  # no part of a step was committed
    assert c.mgr.appendKV(free, 0, K, K, 2) is None
    dec.prepare([free])
    cross.prepare([free], [1])
    held = tl.DecodeBatch(c.mgr, 1, 1)
    held.prepare_lengths([a], [20])
    r.run(1)
    r.ev.commit()
    for i in (0, 1):
        r.check(i)
    assert c.mgr.appendKV(a, 0, K, K, 2) is None
    dec.prepare(c.ids)
    dec.commit(1)
    pf.prepare([b], [2])
    cross.prepare([a, b], [1, 1])
    assert [c.mgr.getSeqLen(s) for s in c.ids] == [21, 21, 11]
    # a step whose sequence is gone says so, whatever its slot's next one does
    c.mgr.releaseSequence(a)
    new, _ = c.mgr.allocateSequence(30)
    c.mgr.advanceSeqLen(new, 9)
    r2 = tl.EvictBatch(c.mgr, 1)
    r2.prepare([new], [5], 1)
    w, p = r.w[0].data_ptr(), r.pos[0].data_ptr()
    r2.run(0, w, w, p, p)
    with pytest.raises(tl.TinyLLMError, match="not found"):
        dec.commit(1)
    torch.cuda.synchronize()
