"""GPU: lengths of sequences in a cache in 8 bits that do not follow the appends: beyond what was
appended, and where several batches append to the same sequences."""
import numpy as np
import pytest
import torch

from quant_ref import QuantCache, attend, check_out
from retention_ref import dev

pytestmark = pytest.mark.gpu


def check_first(c, lens, layer=0):
    """The first lens[i] tokens of every sequence that the host copy has, read at its length."""
    got = c.read(layer, [c.mgr.getSeqLen(s) for s in c.ids])
    for i, n in enumerate(lens):
        for w, x in enumerate((c.k, c.v)):
            # (a whole group that holds tokens nobody brought has a scale of theirs: none here)
            want = c.expect(layer, i)[w].astype(np.float16).transpose(1, 0, 2)[:, :n]
            assert np.array_equal(got[w][i][:, :n], want), (i, w)


def test_lengths_beyond_what_was_appended(tl):
    """Tokens that nobody brought may become visible, but none that were brought may go."""
    c = QuantCache(tl, [20, 32, 0, 70], 2, 64, seed=31, layers=2, room=200)
    m = c.mgr
    for i, far in ((0, 20), (0, 180), (3, 130)):  # the open group's tokens would be left in fp16
        err = m.advanceSeqLen(c.ids[i], far)
        assert err and "beyond the tokens up to" in err, err
    assert [m.getSeqLen(s) for s in c.ids] == [20, 32, 0, 70]
    assert m.advanceSeqLen(c.ids[0], 11) is None  # 31: the same group
    assert m.advanceSeqLen(c.ids[1], 30) is None  # nothing was open
    assert m.advanceSeqLen(c.ids[2], 1000) is None and m.getSeqLen(c.ids[2]) == 200
    for layer in range(2):
        check_first(c, [20, 32, 0, 70], layer)
    b = tl.DecodeBatch(m, 2, 2)
    b.prepare([c.ids[0], c.ids[3]])
    x = dev(c.rows(4))
    b.append(0, 2, x.data_ptr(), x.data_ptr())
    with pytest.raises(tl.TinyLLMError, match="beyond the tokens up to 71"):
        b.commit(40)
    torch.cuda.synchronize()
    check_first(c, [0, 32, 0, 70])


class Prompt:
    """A prompt of n tokens for sequence 0, and its rows in every layer."""

    def __init__(self, tl, c, n, G=1):
        self.c, self.n, self.new = c, n, c.new_rows([n])
        self.b = tl.PrefillBatch(c.mgr, 1, c.hkv * G)
        self.b.prepare(c.ids[:1], [n])
        self.kv = [tuple(dev(x[0]) for x in layer) for layer in self.new]
        self.q = dev(c.rng.standard_normal((n, c.hkv * G, c.d)).astype(np.float16))
        self.out = torch.zeros_like(self.q)

    def append(self, layer=0, s=0):
        self.b.append(layer, *(x.data_ptr() for x in self.kv[layer]), s)

    def run(self, layer=0, s=0):
        self.b.run(layer, self.q.data_ptr(), *(x.data_ptr() for x in self.kv[layer]), self.out.data_ptr(), 0.1, s)

    def attention(self, layer=0, s=0):
        self.b.attention(layer, self.q.data_ptr(), self.out.data_ptr(), 0.1, s)

    def commit(self):
        torch.cuda.synchronize()
        self.b.commit()
        self.c.note(self.new)
        self.c.check()


def test_a_replayed_append_behind_another_one(tl):
    """A prompt is captured, another batch appends less to the same sequence, the graph is replayed: the prompt
    cannot be committed before its append is made again, then it reads back and goes on."""
    c = QuantCache(tl, [95], 2, 64, seed=32, room=300)
    a = Prompt(tl, c, 40)
    a.run()  # (the workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run(0, torch.cuda.current_stream().cuda_stream)
    b = Prompt(tl, c, 1)
    b.append()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        with pytest.raises(tl.TinyLLMError, match="up to 96 of the last append, which replaced"):
            a.b.commit()
    assert c.mgr.getSeqLen(c.ids[0]) == 95
    a.run()
    a.commit()
    c.append([1], "step")
    c.check()


@pytest.mark.parametrize("less", [1, 10, 33, 70])
def test_an_append_in_between(tl, less):
    """Without a graph: what the second append replaced is neither committed nor attended to."""
    c = QuantCache(tl, [95], 2, 64, seed=33, room=300)
    a, b = Prompt(tl, c, 40), Prompt(tl, c, less)
    a.append()
    b.append()
    if less > 33:  # longer: another group is open
        with pytest.raises(tl.TinyLLMError, match="lies inside the tokens up to 165"):
            a.b.commit()
    else:
        with pytest.raises(tl.TinyLLMError, match="which replaced one that brought more"):
            a.b.commit()
    with pytest.raises(tl.TinyLLMError, match="another append to sequence"):
        a.attention()
    r = tl.DecodeBatch(c.mgr, 1, 2)
    r.prepare_lengths(c.ids, [95 + less])
    a.append()
    a.attention()
    with pytest.raises(tl.TinyLLMError, match="has changed since prepare"):
        r.attention(0, a.q.data_ptr(), a.out.data_ptr(), 0.1)
    a.commit()
    c.append([30])
    c.check()


def test_layers_that_differ(tl):
    c = QuantCache(tl, [95], 2, 64, seed=34, layers=2, room=300)
    a, b = Prompt(tl, c, 40), Prompt(tl, c, 10)
    a.append(0)
    b.append(0)
    a.append(1)
    with pytest.raises(tl.TinyLLMError, match="layers differ"):
        a.b.commit()
    r = tl.DecodeBatch(c.mgr, 1, 2)
    r.prepare_lengths(c.ids, [135])
    out = torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(tl.TinyLLMError, match="up to 105, has replaced tokens up to 135 of layer 0"):
        r.attention(0, a.q.data_ptr(), out.data_ptr(), 0.1)
    r.attention(1, a.q.data_ptr(), out.data_ptr(), 0.1)
    a.append(0)
    a.commit()
    # One layer's token alone: the other's open group would stay behind.
    c.append([24], "appendKV")
    x = dev(c.rows(2))
    assert c.mgr.appendKV(c.ids[0], 0, x.data_ptr(), x.data_ptr(), 2) is None
    assert "layers differ" in c.mgr.advanceSeqLen(c.ids[0], 2)
    torch.cuda.synchronize()
    c.check()


def test_a_commit_advances_all_or_none(tl):
    """The second of three sequences refuses: none has advanced, and after its append is made again all do, once."""
    c = QuantCache(tl, [95, 95, 40], 2, 64, seed=35, room=300)
    counts = [40, 40, 3]
    new = c.new_rows(counts)
    k, v = (dev(np.concatenate(x)) for x in new[0])
    p = tl.PrefillBatch(c.mgr, 3, 2)
    p.prepare(c.ids, counts)
    p.append(0, k.data_ptr(), v.data_ptr())
    one = tl.PrefillBatch(c.mgr, 1, 2)
    one.prepare([c.ids[1]], [10])
    one.append(0, k.data_ptr(), v.data_ptr())
    with pytest.raises(tl.TinyLLMError, match=f"sequence {c.ids[1]}"):
        p.commit()
    assert [c.mgr.getSeqLen(s) for s in c.ids] == [95, 95, 40]
    p.append(0, k.data_ptr(), v.data_ptr())
    torch.cuda.synchronize()
    p.commit()
    c.note(new)
    c.check()
    # steps: 135 and one drafted token more than fits the group of the third
    b = tl.DecodeBatch(c.mgr, 3, 2)
    b.prepare(c.ids)
    b.append(0, 1, k.data_ptr(), v.data_ptr())
    with pytest.raises(tl.TinyLLMError, match=f"sequence {c.ids[2]}"):
        b.commit(22)
    assert [c.mgr.getSeqLen(s) for s in c.ids] == [135, 135, 43]
    torch.cuda.synchronize()
    c.check()


def test_a_commit_behind_a_release_or_without_blocks(tl):
    m = tl.KVCacheManager(num_layers=1, num_heads=1, head_dim=64, max_seq_len=256, max_batch_size=3, block_tokens=32, num_blocks=6,
                          quantized=True)
    ids = [m.allocateSequence(256)[0] for _ in range(3)]
    b, p = tl.DecodeBatch(m, 3, 1), tl.PrefillBatch(m, 2, 1)
    b.prepare(ids)
    with pytest.raises(tl.TinyLLMError, match="exhausted"):
        b.commit(96)  # nine blocks
    assert [m.getSeqLen(s) for s in ids] == [0, 0, 0] and m.freeBlocks() == 3
    b.commit(64)
    assert [m.getSeqLen(s) for s in ids] == [64, 64, 64] and m.freeBlocks() == 0
    assert m.releaseSequence(ids[1]) is None
    p.prepare([ids[0], ids[2]], [1, 1])
    with pytest.raises(tl.TinyLLMError, match=f"not found: {ids[1]}"):
        b.commit(1)
    assert m.getSeqLen(ids[0]) == 64
    assert m.releaseSequence(ids[2]) is None
    with pytest.raises(tl.TinyLLMError, match=f"not found: {ids[2]}"):
        p.commit()
    assert m.getSeqLen(ids[0]) == 64
    with pytest.raises(tl.TinyLLMError, match="positive"):
        b.commit(0)


@pytest.mark.parametrize("lens", [[40, 95, 64], [20, 96, 127]])
def test_tokens_that_stand_are_read_behind_appends(tl, lens):
    """A batch that attends to tokens that its sequences have advanced over goes on doing so, whatever is
    appended behind them; one that attends to appended tokens is refused once those are others."""
    c = QuantCache(tl, lens, 2, 64, seed=36, hq=8, room=300)
    att = [n - k for n, k in zip(lens, (0, 3, 64))]
    q = c.rng.standard_normal((3, 8, 64)).astype(np.float16)
    dq, out = dev(q), torch.zeros((3, 8, 64), dtype=torch.float16, device="cuda")
    back = torch.zeros((3, 2, 128, 64), dtype=torch.float16, device="cuda")
    b, drafts = tl.DecodeBatch(c.mgr, 3, 8), tl.DecodeBatch(c.mgr, 3, 8)
    b.prepare_lengths(c.ids, att)
    for counts in ([1, 1, 1], [30, 33, 5], [70, 40, 100]):
        k, v = dev(c.rows(sum(counts))), dev(c.rows(sum(counts)))
        p = tl.PrefillBatch(c.mgr, 3, 8)
        p.prepare(c.ids, counts)
        p.append(0, k.data_ptr(), v.data_ptr())
        if counts[0] > 1:
            with pytest.raises(tl.TinyLLMError, match="has changed since prepare"):
                drafts.attention(0, dq.data_ptr(), out.data_ptr(), 0.125)
        drafts.prepare_lengths(c.ids, [n + m for n, m in zip(lens, counts)])
        out.zero_()
        b.attention(0, dq.data_ptr(), out.data_ptr(), 0.125)
        b.gather(0, back.data_ptr(), None, 128)
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        for i, a in enumerate(att):
            if a == 0:
                assert not got[i].any() and not back[i].any()
                continue
            kk, vv = (x[:a] for x in c.expect(0, i))
            assert np.array_equal(back[i, :, :a].cpu().numpy(), kk.astype(np.float16).transpose(1, 0, 2))
            o, mass, err = attend(q[i:i + 1], kk, vv, 0.125, [a - 1])
            check_out(got[i:i + 1], o, mass, err, a, np.abs(vv).max())
    assert c.mgr.advanceSeqLen(c.ids[1], 1) is None
    with pytest.raises(tl.TinyLLMError, match="has changed since prepare"):
        b.attention(0, dq.data_ptr(), out.data_ptr(), 0.125)


@pytest.mark.parametrize("pool", [dict(), dict(block_tokens=32, num_blocks=8), dict(block_tokens=32, num_blocks=8, quantized=True)])
def test_counts_at_the_end_of_an_int(tl, pool):
    """A length and a count whose sum is beyond 2^31 - 1 are an overflow of the cache."""
    m = tl.KVCacheManager(num_layers=1, num_heads=1, head_dim=64, max_seq_len=128, max_batch_size=2, **pool)
    s = m.allocateSequence(128)[0]
    x = torch.zeros((128, 64), dtype=torch.float16, device="cuda")
    assert m.appendKV(s, 0, x.data_ptr(), x.data_ptr(), 100) is None and m.advanceSeqLen(s, 100) is None
    for n in (2 ** 31 - 1, 2 ** 31 - 100, 2 ** 31 - 101, 29):
        assert f"cache overflow. Current: 100, appending: {n}, max: 128" in m.appendKV(s, 0, x.data_ptr(), x.data_ptr(), n)
        with pytest.raises(tl.TinyLLMError, match="cache overflow"):
            tl.PrefillBatch(m, 1, 1).prepare([s], [n])
    assert m.appendKV(s, 0, x.data_ptr(), x.data_ptr(), 28) is None
    torch.cuda.synchronize()


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("how", ["appendKV", "prefill", "run", "append", "decode"])
def test_tokens_that_nobody_brought_count_as_zeros(tl, d, how):
    """A sequence advances over tokens that were not appended, and its group of 32 is completed: what an
    earlier sequence left in the open group, infinite and large, has no part in the scale of those that were."""
    big = QuantCache(tl, [31, 60], 2, d, seed=37, hq=2, layers=2, spare=0, room=100)
    for i in range(2):
        for layer in range(2):
            x = torch.full((100, 2, d), float("inf") if i else 60000.0, dtype=torch.float16, device="cuda")
            big.mgr.appendKV(big.ids[i], layer, x.data_ptr(), x.data_ptr(), 35)
    torch.cuda.synchronize()
    for s in big.ids:
        assert big.mgr.releaseSequence(s) is None
    c = big
    c.ids = [c.mgr.allocateSequence(100)[0] for _ in range(2)]
    c.k, c.v = ([[np.zeros((0, 2, d), np.float16) for _ in range(2)] for _ in range(2)] for _ in range(2))
    c.append([20, 0])
    assert c.mgr.advanceSeqLen(c.ids[0], 8) is None and c.mgr.advanceSeqLen(c.ids[1], 60) is None
    zeros = [tuple([np.zeros((n, 2, d), np.float16) for n in (8, 60)] for _ in range(2)) for _ in range(2)]
    c.note(zeros)
    one, steps = how in ("append", "decode"), 4
    for k in range(steps if one else 1):
        counts = [1, 1] if one else [9, 4]
        new = c.new_rows(counts)
        if how in ("appendKV", "prefill", "append"):
            c.append(counts, {"append": "step"}.get(how, how), new)
            continue
        b = tl.DecodeBatch(c.mgr, 2, 2) if one else tl.PrefillBatch(c.mgr, 2, 2)
        b.prepare(c.ids) if one else b.prepare(c.ids, counts)
        for layer in range(2):
            kk, vv = (dev(np.concatenate(x)) for x in new[layer])
            q, out = torch.zeros((sum(counts), 2, d), dtype=torch.float16, device="cuda"), torch.zeros_like(kk)
            (b.decode if one else b.run)(layer, q.data_ptr(), kk.data_ptr(), vv.data_ptr(), out.data_ptr(), 1.0)
            torch.cuda.synchronize()
        b.commit(1) if one else b.commit()
        c.note(new)
    for layer in range(2):
        got = c.read(layer)
        for w in range(2):
            for i, first in ((0, 0), (1, 32)):  # (the second's first group was never written at all)
                want = c.expect(layer, i)[w].astype(np.float16).transpose(1, 0, 2)
                assert np.array_equal(got[w][i][:, first:want.shape[1]], want[:, first:])
