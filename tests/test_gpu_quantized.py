"""GPU: a cache in 8 bits -- written, read back, decode and prefill attention over it --
against plain 64-bit forms: what it stands for bit for bit, attention within bounds
derived from the roundings of the path."""
import numpy as np
import pytest
import torch

from quant_ref import GROUP, QuantCache, attend, check_out, held
from retention_ref import dev

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ writing, reading back
@pytest.mark.parametrize("d,hkv,block,lens", [
    (32, 1, 32, [1, 31, 32, 33]),
    (64, 3, 32, [63, 64, 65, 2]),
    (128, 8, 64, [200, 7, 96]),
    (256, 2, 128, [127, 128, 129, 300]),
    (128, 1, 256, [1000, 255]),
    (64, 32, 64, [100]),
])
def test_write_and_read_back(tl, d, hkv, block, lens):
    c = QuantCache(tl, lens, hkv, d, block=block, seed=d + block)
    assert c.mgr.isQuantized()
    c.check()
    c.append([5 + i for i in range(len(lens))])
    c.check()


@pytest.mark.parametrize("how", ["prefill", "appendKV", "step"])
def test_the_bytes_do_not_depend_on_how_tokens_came(tl, how):
    """70 tokens at once, in ragged pieces, one at a time; three layers."""
    whole = QuantCache(tl, [70, 64, 33], 2, 64, layers=3, seed=3, block=64)
    c = QuantCache(tl, [0, 0, 0], 2, 64, layers=3, seed=4, block=64, room=110)
    at = [0, 0, 0]
    pieces = [1] * 70 if how == "step" else [1, 2, 30, 31, 5, 1]
    for p in pieces:
        counts = [min(p, n - a) for a, n in zip(at, [70, 64, 33])]
        new = [tuple([rows[layer][i][at[i]:at[i] + counts[i]] for i in range(3)] for rows in (whole.k, whole.v))
               for layer in range(3)]
        c.append(counts, how, new)
        at = [a + n for a, n in zip(at, counts)]
    c.check()
    for layer in range(3):
        for x, y in zip(whole.read(layer), c.read(layer)):
            assert np.array_equal(x.view(np.uint16), y.view(np.uint16))


def special_rows(kind, d, rng):
    """32 rows of one head."""
    x = rng.standard_normal((GROUP, d)).astype(np.float16)
    if kind == "zeros":
        x[:] = 0
        x[::2] = -0.0
    elif kind == "tiny":  # subnormal halves: the scale is far below fp16's range
        x = (x * 2.0 ** -22).astype(np.float16)
    elif kind == "least":
        x[:] = 0
        x[3, 5] = 2.0 ** -24
    elif kind == "largest":
        x = (x.astype(np.float64) * 16000).clip(-65504, 65504).astype(np.float16)
        x[1, 1] = -65504
    elif kind == "halves":  # the scale is 1: halves of whole numbers go to the even one
        x = (np.arange(GROUP * d).reshape(GROUP, d) % 254 / 2 - 63).astype(np.float16)
        x[0, 0] = 127
    elif kind == "coarse":  # 127 times a number of 11 bits, and one step less
        x = (rng.integers(-127, 128, (GROUP, d)) * 2.0 ** -3).astype(np.float16)
        x[7, 0] = 127 * 2.0 ** -3
        x[8, 0] = np.nextafter(np.float16(127 * 2.0 ** -3), np.float16(0))
    elif kind in ("inf", "nan"):
        x[9, 2] = -np.inf if kind == "inf" else np.nan
    return x


KINDS = ["zeros", "tiny", "least", "largest", "halves", "coarse", "inf", "nan"]


@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_special_values(tl, d):
    """A kind per kv head, the whole numbers of every 11-bit maximum among them."""
    c = QuantCache(tl, [0], len(KINDS), d, seed=5, room=110)
    rows = np.stack([special_rows(k, d, c.rng) for k in KINDS], axis=1)
    new = [([rows], [rows[::-1].copy()])]
    c.append([GROUP], "prefill", new)
    c.check()
    c.append([3])
    c.check()


def test_every_maximum(tl):
    """2048 groups with every mantissa as the maximum, beside every smaller value."""
    d, n = 64, 2048 * GROUP
    c = QuantCache(tl, [0], 1, d, block=256, room=n)
    x = np.zeros((2048, GROUP * d), np.float16)
    mantissas = (1024 + np.arange(2048) % 1024).astype(np.float64)
    x[:, 0] = mantissas * 2.0 ** (np.arange(2048) // 1024 * 4 - 10)
    x[:, 1:] = (np.arange(1, GROUP * d) / (GROUP * d) * x[:, :1].astype(np.float64)).astype(np.float16)
    x[:, 2::3] *= -1
    x = x.reshape(n, 1, d)
    c.append([n], "prefill", [([x], [x])])
    c.check()


def test_reading_back_parts(tl):
    c = QuantCache(tl, [100, 40], 2, 64, layers=2, seed=6)
    for lens, s_max, which in [([100, 40], 128, "kv"), ([70, 33], 70, "k"), ([96, 1], 20, "v"), ([0, 32], 33, "kv"), ([64, 0], 1, "kv")]:
        got = c.read(1, lens, s_max, which)
        for w, (x, name) in enumerate(zip(got, "kv")):
            if name not in which:
                assert np.isnan(x).all()
                continue
            for i, n in enumerate(lens):
                # (a group that is complete in the cache is read there, whatever the length)
                want = c.expect(1, i)[w][:n].astype(np.float16).transpose(1, 0, 2)[:, :s_max]
                assert np.array_equal(x[i][:, :want.shape[1]], want) and not x[i][:, want.shape[1]:].any()


def test_only_the_step_is_written(tl):
    """Neighbours, other layers and released blocks stay as they were."""
    c = QuantCache(tl, [40, 50, 60], 2, 32, layers=2, seed=7)
    b = tl.PrefillBatch(c.mgr, 1, 2)
    b.prepare([c.ids[1]], [30])
    k, v = c.rows(30), c.rows(30)
    dk, dv = dev(k), dev(v)
    b.append(1, dk.data_ptr(), dv.data_ptr())
    torch.cuda.synchronize()
    for layer in range(2):
        got = c.read(layer)
        for i in range(3):
            for w in range(2):
                want = c.expect(layer, i)[w]
                if layer == 1 and i == 1:  # (its open group was closed, 50 tokens as given so far)
                    continue
                assert np.array_equal(got[w][i][:, :len(want)], want.astype(np.float16).transpose(1, 0, 2))
    c.k[1][1], c.v[1][1] = np.concatenate([c.k[1][1], k]), np.concatenate([c.v[1][1], v])
    got = c.read(1, [40, 80, 60])
    for w in range(2):
        assert np.array_equal(got[w][1], c.expect(1, 1)[w].astype(np.float16).transpose(1, 0, 2))


# ------------------------------------------------------------------ lengths that go back
def test_rejected_drafts(tl):
    """Appends of 7 of which 1 .. 7 stay, over many groups; then the same cache as one
    that never saw the rejected ones."""
    c = QuantCache(tl, [20, 31, 32], 2, 64, layers=2, seed=8, room=400)
    for step in range(25):
        new = c.new_rows([7, 7, 7])
        p = tl.PrefillBatch(c.mgr, 3, 2)
        p.prepare(c.ids, [7, 7, 7])
        for layer, (k, v) in enumerate(new):
            dk, dv = dev(np.concatenate(k)), dev(np.concatenate(v))
            p.append(layer, dk.data_ptr(), dv.data_ptr())
            p.append(layer, dk.data_ptr(), dv.data_ptr())  # once more, the same
            torch.cuda.synchronize()
        keep = 1 + step % 7
        for s in c.ids:
            assert c.mgr.advanceSeqLen(s, keep) is None
        c.note(new, keep)
        # what was advanced over, with the drafts still behind it
        k, _ = c.read(1)
        n = len(c.k[1][0])
        assert np.array_equal(k[0][:, :n], c.expect(1, 0)[0].astype(np.float16).transpose(1, 0, 2))
    c.append([1, 1, 1], "step")
    c.check()


def test_lengths_inside_an_append(tl):
    c = QuantCache(tl, [0], 1, 32, seed=9, room=200)
    new = c.new_rows([100])
    k, v = dev(new[0][0][0]), dev(new[0][1][0])
    assert c.mgr.appendKV(c.ids[0], 0, k.data_ptr(), v.data_ptr(), 100) is None
    err = c.mgr.advanceSeqLen(c.ids[0], 50)
    assert "length 50" in err and "up to 100" in err and c.mgr.getSeqLen(c.ids[0]) == 0
    assert c.mgr.advanceSeqLen(c.ids[0], 64) is None
    assert "length 74" in c.mgr.advanceSeqLen(c.ids[0], 10)
    assert c.mgr.advanceSeqLen(c.ids[0], 34) is None  # 98: the group in which the append ended
    c.note(new, 98)
    c.check()
    c.append([1], "step")
    c.check()


def test_slots_are_used_again(tl):
    c = QuantCache(tl, [45, 70], 2, 64, seed=10, blocks=8, room=100)
    used = c.mgr.getUsedMemory()
    assert used == 5 * c.mgr.blockBytes() == 5 * 2 * (64 * 64 + 8)
    assert c.mgr.releaseSequence(c.ids[0]) is None
    c.ids[0], err = c.mgr.allocateSequence(100)
    assert err is None
    c.k[0][0], c.v[0][0] = c.k[0][0][:0], c.v[0][0][:0]
    c.append([10, 0])
    c.check()


# ------------------------------------------------------------------ attention
def decode(tl, c, G, layer=0, scale=None, fused=True):
    """A step of one token per sequence: q over all of it."""
    n, hq = len(c.ids), c.hkv * G
    scale = c.d ** -0.5 if scale is None else scale
    new = c.new_rows([1] * n)
    q = c.rng.standard_normal((n, hq, c.d)).astype(np.float16)
    b = tl.DecodeBatch(c.mgr, n, hq)
    b.prepare(c.ids, stream())
    k, v, dq = dev(np.concatenate(new[layer][0])), dev(np.concatenate(new[layer][1])), dev(q)
    out = torch.full((n + 1, hq, c.d), 9.0, dtype=torch.float16, device="cuda")
    if fused:
        b.decode(layer, dq.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), scale, stream())
    else:
        b.append(layer, 1, k.data_ptr(), v.data_ptr(), stream())
        b.attention(layer, dq.data_ptr(), out.data_ptr(), scale, stream())
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[n:] == 9.0).all()
    for i in range(n):
        kk, vv = (held(np.concatenate([x[layer][i], new[layer][w][i]])) for w, x in enumerate((c.k, c.v)))
        o, mass, err = attend(q[i:i + 1], kk, vv, scale, [len(kk) - 1])
        check_out(got[i:i + 1], o, mass, err, len(kk), np.abs(vv).max())
    return b, new, got[:n]


@pytest.mark.parametrize("d,hkv,G,block,lens", [
    (64, 8, 1, 32, [0, 1, 30, 31, 32, 33]),
    (128, 2, 4, 64, [62, 63, 64, 65, 95, 96, 500]),
    (128, 8, 8, 32, [127, 128, 1000]),
    (32, 1, 2, 32, [5, 64, 191, 3000]),
    (256, 2, 8, 128, [31, 32, 63, 64, 700]),
    (256, 1, 1, 32, [2100]),
    (64, 4, 4, 256, [4000, 1, 255]),
    (128, 1, 4, 64, [9000]),
    (128, 8, 4, 128, [33000, 31]),
    (128, 64, 1, 32, [0, 31, 32, 100, 500]),                 # many short ones: 5 x 64 workgroups
    (64, 64, 2, 32, [0, 63, 64, 95, 31, 1, 300, 200, 7]),
    (256, 40, 1, 32, [0, 1, 31, 33, 128, 250, 64]),
    (32, 128, 1, 32, [3, 62, 0, 63, 1000]),
])
@pytest.mark.parametrize("fused", [True, False])
def test_decode(tl, d, hkv, G, block, lens, fused):
    c = QuantCache(tl, lens, hkv, d, block=block, seed=d + G, hq=hkv * G)
    b, new, _ = decode(tl, c, G, fused=fused)
    b.commit(1)
    c.note(new)
    c.check()
    decode(tl, c, G, fused=not fused)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales_of_either_sign(tl, scale):
    c = QuantCache(tl, [100, 31], 2, 64, seed=11, hq=8, room=200)
    decode(tl, c, 4, scale=scale)
    prefill(tl, c, 4, [3, 2], scale=scale)
    prefill(tl, c, 4, [50, 9], scale=scale)


def test_many_entries(tl):
    """More than a launch's arguments hold, lengths and slots out of order."""
    rng = np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(0, 90, 300)]
    c = QuantCache(tl, lens, 1, 32, seed=12, hq=2)
    c.check()
    b, new, _ = decode(tl, c, 2)
    b.commit(1)
    c.note(new)
    c.check()
    prefill(tl, c, 2, [9 + i % 20 for i in range(300)])


@pytest.mark.parametrize("lens,att", [([100, 64, 33], [100, 64, 33]), ([100, 64, 33], [50, 0, 32]), ([100, 64, 33], [97, 1, 1]),
                                      ([3000, 64, 0], [2500, 63, 0])])
def test_attended_lengths(tl, lens, att):
    c = QuantCache(tl, lens, 2, 64, seed=13, hq=8)
    q = c.rng.standard_normal((3, 8, 64)).astype(np.float16)
    out = torch.full((3, 8, 64), 9.0, dtype=torch.float16, device="cuda")
    b = tl.DecodeBatch(c.mgr, 3, 8)
    b.prepare_lengths(c.ids, att)
    dq = dev(q)
    b.attention(0, dq.data_ptr(), out.data_ptr(), 0.125)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    for i, a in enumerate(att):
        if a == 0:
            assert not got[i].any()
            continue
        k, v = (x[:a] for x in c.expect(0, i))
        o, mass, err = attend(q[i:i + 1], k, v, 0.125, [a - 1])
        check_out(got[i:i + 1], o, mass, err, a, np.abs(v).max())


def prefill(tl, c, G, counts, layer=0, scale=None, fused=True, commit=False):
    n, hq = len(counts), c.hkv * G
    scale = c.d ** -0.5 if scale is None else scale
    new = c.new_rows(counts)
    q = c.rng.standard_normal((sum(counts), hq, c.d)).astype(np.float16)
    p = tl.PrefillBatch(c.mgr, n, hq)
    p.prepare(c.ids[:n], counts, stream())
    out = torch.full((sum(counts) + 1, hq, c.d), 9.0, dtype=torch.float16, device="cuda")
    k, v, dq = dev(np.concatenate(new[layer][0])), dev(np.concatenate(new[layer][1])), dev(q)
    if fused:
        p.run(layer, dq.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), scale, stream())
    else:
        p.append(layer, k.data_ptr(), v.data_ptr(), stream())
        p.attention(layer, dq.data_ptr(), out.data_ptr(), scale, stream())
    torch.cuda.synchronize()
    got, at = out.cpu().numpy(), 0
    assert (got[-1] == 9.0).all()
    for i, m in enumerate(counts):
        kk, vv = (held(np.concatenate([x[layer][i], new[layer][w][i]])) for w, x in enumerate((c.k, c.v)))
        p0 = len(kk) - m
        o, mass, err = attend(q[at:at + m], kk, vv, scale, p0 + np.arange(m))
        check_out(got[at:at + m], o, mass, err, len(kk), np.abs(vv).max())
        at += m
    if commit:
        p.commit()
        c.note(new)
        c.check()
    return p, got[:-1]


@pytest.mark.parametrize("d,hkv,G,block,lens,counts", [
    (64, 2, 1, 32, [0, 5, 31], [1, 16, 2]),                 # up to 16 query rows
    (128, 2, 4, 64, [100, 60, 28, 0], [4, 4, 4, 4]),
    (128, 1, 8, 32, [2000, 31], [2, 1]),
    (128, 64, 4, 32, [0, 30, 31, 61, 100], [4, 4, 1, 3, 2]),
    (32, 2, 8, 32, [0, 0, 62], [2, 1, 2]),
    (256, 1, 2, 32, [70, 31], [8, 3]),
    (64, 2, 1, 32, [0, 0, 0, 40], [17, 31, 32, 33]),         # more
    (128, 2, 4, 64, [0, 100, 33], [5, 64, 130]),
    (128, 1, 8, 128, [500, 31], [33, 97]),
    (256, 2, 2, 32, [0, 90], [100, 9]),
    (32, 3, 4, 32, [10, 400], [70, 6]),
    (64, 1, 2, 64, [0], [700]),
    (128, 8, 4, 256, [3000], [40]),                          # keys in chunks
    (128, 1, 4, 64, [1000], [3]),
    (256, 4, 1, 64, [2000], [50]),
    (128, 1, 1, 32, [0], [1100]),
    (128, 8, 4, 64, [4000, 100, 0], [20, 40, 17]),           # of some entries
    (64, 2, 8, 32, [0, 5000], [3, 33]),
    (128, 32, 1, 64, [3000] + [0] * 8, [300] + [200] * 8),   # of the longest, while the others fill the chip
    (256, 16, 2, 64, [2500] + [10] * 9, [70] + [100] * 9),
])
@pytest.mark.parametrize("fused", [True, False])
def test_prefill(tl, d, hkv, G, block, lens, counts, fused):
    c = QuantCache(tl, lens, hkv, d, block=block, seed=d + G + 1, hq=hkv * G, room=max(lens) + 2 * max(counts))
    prefill(tl, c, G, counts, fused=fused, commit=True)


def test_mixed_row_counts(tl):
    """Entries of few and of many query rows in one step."""
    c = QuantCache(tl, [50, 0, 300, 31], 2, 128, seed=14, hq=8)
    prefill(tl, c, 4, [3, 40, 4, 33], commit=True)
    prefill(tl, c, 4, [33, 3, 1, 5], commit=True)


# ------------------------------------------------------------------ what is not finite, and where
@pytest.mark.parametrize("counts", [4, 40])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_only_who_sees_it(tl, counts, where, bad):
    """A value that is not finite at a position of the step: queries before it (before
    its group where that is complete) do not feel it; queries that see it do."""
    d, G = 64, 4
    for prefix, at in [(0, counts - 1), (64, counts - 2), (95, 3), (30, counts - 1)]:
        c = QuantCache(tl, [prefix], 1, d, seed=15, hq=G, room=300)
        new = c.new_rows([counts])
        (new[0][0] if where == "k" else new[0][1])[0][at, 0, 7] = bad
        q = c.rng.standard_normal((counts, G, d)).astype(np.float16)
        p = tl.PrefillBatch(c.mgr, 1, G)
        p.prepare(c.ids, [counts])
        out = torch.zeros((counts, G, d), dtype=torch.float16, device="cuda")
        dq, dk, dv = dev(q), dev(new[0][0][0]), dev(new[0][1][0])
        p.run(0, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), out.data_ptr(), 0.125)
        torch.cuda.synchronize()
        got, end = out.cpu().numpy(), prefix + counts
        group = (prefix + at) // GROUP * GROUP
        whole = group + GROUP <= end
        first = max(0, (group if whole else prefix + at) - prefix)  # the first query that sees some of it
        k, v = (np.concatenate([x[0][0], new[0][w][0]]) for w, x in enumerate((c.k, c.v)))
        clean = [np.where(np.isfinite(x), x, 0) for x in (k, v)]
        hk, hv = held(clean[0]), held(clean[1])
        if whole:  # the others' tokens of that group are NaN too, so are all that see it
            assert np.isnan(got[first:]).all()
        elif where == "v":
            assert not np.isfinite(got[first:, :, 7]).any()
            rest = np.delete(got, 7, axis=2)
            assert np.isfinite(rest).all()
        if first:
            o, mass, err = attend(q[:first], hk, hv, 0.125, prefix + np.arange(first))
            check_out(got[:first], o, mass, err, end, np.abs(hv).max())


def test_what_lies_behind_the_last_token(tl):
    """Rows that an earlier sequence or a rejected draft left in the open group, infinite ones."""
    c = QuantCache(tl, [40], 2, 64, seed=16, hq=8)
    new = c.new_rows([15])
    for w in range(2):
        new[0][w][0][:] = np.inf
        new[0][w][0][0] = 1.0
    k, v = dev(new[0][0][0]), dev(new[0][1][0])
    assert c.mgr.appendKV(c.ids[0], 0, k.data_ptr(), v.data_ptr(), 15) is None
    assert c.mgr.advanceSeqLen(c.ids[0], 1) is None
    c.note(new, 1)
    decode(tl, c, 4)
    prefill(tl, c, 4, [2])
    prefill(tl, c, 4, [9])
    c.check()


def test_small_and_large_scales(tl):
    """Values far below fp16's normal numbers, and at its end: relative bounds."""
    for std in (2.0 ** -16, 2.0 ** -10, 12000.0):
        c = QuantCache(tl, [0], 2, 64, seed=17, hq=8, room=300)
        real = c.rows
        c.rows = lambda n, s=1.0, real=real: real(n, std).clip(-65504, 65504)
        c.append([70])
        c.check()
        decode(tl, c, 4, scale=0.125 / max(std, 1.0) if std > 1 else 0.125)
        prefill(tl, c, 4, [30], scale=0.125 / max(std, 1.0) if std > 1 else 0.125)


# ------------------------------------------------------------------ graphs and streams
def captured(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    return graph


def test_captured_steps(tl):
    """Two batches' calls captured, replayed with eager work in between, inputs changed."""
    c = QuantCache(tl, [2000, 95, 31], 2, 128, seed=18, hq=8)
    q = dev(c.rng.standard_normal((60, 8, 128)).astype(np.float16))
    k, v = dev(c.rows(60)), dev(c.rows(60))
    outs = [torch.zeros_like(q) for _ in range(4)]
    back = [torch.zeros((3, 2, 2100, 128), dtype=torch.float16, device="cuda") for _ in range(2)]
    b, p = tl.DecodeBatch(c.mgr, 3, 8), tl.PrefillBatch(c.mgr, 2, 8)

    def step(i, s=0):
        b.decode(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[i].data_ptr(), 0.1, s)

    def prompt(i, s=0):
        p.run(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[i].data_ptr(), 0.1, s)

    b.prepare(c.ids)
    p.prepare(c.ids[:2], [40, 20])
    step(0)
    prompt(2)
    torch.cuda.synchronize()
    graphs = [captured(lambda s: step(1, s)), captured(lambda s: prompt(3, s)),
              captured(lambda s: (step(1, s), b.gather(0, back[0].data_ptr(), back[1].data_ptr(), 2100, s)))]
    for r in range(4):
        with torch.no_grad():
            q.copy_(dev(c.rng.standard_normal((60, 8, 128)).astype(np.float16)))
            k.copy_(dev(c.rows(60)))
        for g, eager, i in ((graphs[0], step, 0), (graphs[1], prompt, 2)):
            outs[i].zero_(), outs[i + 1].zero_()
            eager(i)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], outs[i + 1]) and outs[i].any()
        graphs[2].replay()
        torch.cuda.synchronize()
        assert torch.equal(back[0][0, :, 2000], k[0])  # an open group's row,
        for i, n in ((1, 95), (2, 31)):              # and those that closed theirs
            assert (back[0][i, :, n] - k[i]).abs().max() <= 0.03 and not torch.equal(back[0][i, :, n], k[i])


def test_a_capture_does_not_grow_the_workspace(tl):
    c = QuantCache(tl, [20000], 1, 64, seed=19, hq=8, block=256)
    b = tl.DecodeBatch(c.mgr, 1, 8)
    b.prepare_lengths(c.ids, [20000])
    q = torch.zeros((1, 8, 64), dtype=torch.float16, device="cuda")
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        q.zero_()
        with pytest.raises(tl.TinyLLMError, match="captured"):
            b.attention(0, q.data_ptr(), q.data_ptr(), 0.125, s.cuda_stream)


def test_a_refused_prompt_appends_nothing(tl):
    c = QuantCache(tl, [3000], 1, 64, seed=21, hq=8, block=256)
    p = tl.PrefillBatch(c.mgr, 1, 8)
    p.prepare(c.ids, [4])
    x = torch.zeros((4, 8, 64), dtype=torch.float16, device="cuda")
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        x.zero_()
        with pytest.raises(tl.TinyLLMError, match="captured"):
            p.run(0, x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), 0.125, s.cuda_stream)
    with pytest.raises(tl.TinyLLMError, match="more than the 3000 tokens"):
        tl.DecodeBatch(c.mgr, 1, 8).prepare_lengths(c.ids, [3001])
    graph.replay()
    torch.cuda.synchronize()
    c.check()


def test_beyond_4_gib(tl):
    """A sequence whose last tokens lie behind 4 GiB of the pool and of a layer: the earlier
    ones are one chunk over and over, whose scores are far below those of the last."""
    hkv, d, chunk, times, n = 8, 128, 1 << 17, 17, 200
    room = chunk * times + n + 40
    mgr = tl.KVCacheManager(num_layers=1, num_heads=hkv, head_dim=d, max_seq_len=room, max_batch_size=1, block_tokens=256,
                            num_blocks=-(-room // 256), quantized=True)
    sid, err = mgr.allocateSequence(room)
    assert err is None
    rng = np.random.default_rng(22)
    far = torch.full((chunk, hkv, d), -1.0, dtype=torch.float16, device="cuda")
    for _ in range(times):
        assert mgr.appendKV(sid, 0, far.data_ptr(), far.data_ptr(), chunk) is None
        assert mgr.advanceSeqLen(sid, chunk) is None
    assert chunk * times * hkv * d * 2 > 1 << 32
    near = [(1 + rng.random((n, hkv, d)) / 4).astype(np.float16) for _ in range(2)]
    near[1] = rng.standard_normal((n, hkv, d)).astype(np.float16)
    for count, G in ((n - 70, 4), (66, 4), (3, 4), (1, 4)):  # by the prompt kernel, then by the step's
        done = mgr.getSeqLen(sid) - chunk * times
        k, v = (dev(x[done:done + count]) for x in near)
        q = np.full((count, hkv * G, d), 0.5, dtype=np.float16)  # scores: -64 of the far tokens, 64 and more of the near ones
        dq, out = dev(q), torch.empty((count, hkv * G, d), dtype=torch.float16, device="cuda")
        b = tl.DecodeBatch(mgr, 1, hkv * G) if count == 1 else tl.PrefillBatch(mgr, 1, hkv * G)
        if count == 1:
            b.prepare([sid])
            b.decode(0, dq.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 1.0, stream())
        else:
            b.prepare([sid], [count])
            b.run(0, dq.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 1.0, stream())
        torch.cuda.synchronize()
        b.commit(1) if count == 1 else b.commit()
        kk, vv = (held(x[:done + count]) for x in near)
        o, mass, err = attend(q, kk, vv, 1.0, done + np.arange(count))
        check_out(out.cpu().numpy(), o, mass, err, done + count, np.abs(vv).max())


def test_another_stream(tl):
    c = QuantCache(tl, [500, 64], 2, 64, seed=20, hq=8)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b, new, _ = decode(tl, c, 4)
    b.commit(1)
    c.note(new)
    c.check()


# ------------------------------------------------------------------ refusals
def test_refusals(tl):
    c = QuantCache(tl, [40, 10], 2, 64, seed=21, hq=8, layers=2)
    m, bad = c.mgr, tl.TinyLLMError
    q = torch.zeros((64, 8, 64), dtype=torch.float16, device="cuda")
    a, odd = q.data_ptr(), q.data_ptr() + 2
    for make in (lambda: tl.EvictBatch(m, 1), lambda: tl.CrossBatch(m, 1, 8)):
        with pytest.raises(bad, match="fp16 caches only"):
            make()
    assert "paged" in m.getCacheChecked(c.ids[0], 0)[1]
    assert "block pool" in m.setBlockMap(32, [0])
    b, p = tl.DecodeBatch(m, 2, 8), tl.PrefillBatch(m, 2, 8)
    b.prepare(c.ids)
    p.prepare(c.ids, [2, 3])
    with pytest.raises(bad, match="8-bit cache takes projections"):
        b.project(0, a, 64, 32, a, a, a, a)
    with pytest.raises(bad, match="fp16 caches only"):
        b.decode_weights(0, a, a, a, a, 1.0, None, a)
    with pytest.raises(bad, match="fp16 caches only"):
        p.weights(0, a, 1.0, 0, None, a)
    for call in (lambda: b.append(0, 1, odd, a), lambda: b.attention(0, odd, a, 1.0), lambda: b.decode(0, a, a, odd, a, 1.0),
                 lambda: b.gather(0, odd, a, 50), lambda: p.append(0, a, odd), lambda: p.attention(0, a, odd, 1.0),
                 lambda: p.run(0, a, odd, a, a, 1.0)):
        with pytest.raises(bad, match="16-byte aligned"):
            call()
    assert "16-byte aligned" in m.appendKV(c.ids[0], 0, a, odd, 1)
    for call in (lambda: b.append(1, 2, a, a), lambda: b.append(0, 1, None, a), lambda: b.attention(2, a, a, 1.0),
                 lambda: b.gather(-1, a, a, 1), lambda: p.append(2, a, a), lambda: p.run(0, a, None, a, a, 1.0),
                 lambda: p.attention(0, a, None, 1.0), lambda: b.decode(0, None, a, a, a, 1.0)):
        with pytest.raises(bad):
            call()
    with pytest.raises(bad, match="more than the 40 tokens"):
        b.prepare_lengths([c.ids[0]], [41])
    b.prepare_lengths([c.ids[0]], [40])
    with pytest.raises(bad, match="prepare"):
        b.append(0, 1, a, a)
    # lengths that change between prepare and the calls
    b.prepare(c.ids)
    assert m.advanceSeqLen(c.ids[1], 1) is None
    for call in (lambda: b.append(0, 1, a, a), lambda: b.attention(0, a, a, 1.0), lambda: b.decode(0, a, a, a, a, 1.0),
                 lambda: b.gather(0, a, a, 4), lambda: p.append(0, a, a), lambda: p.attention(0, a, a, 1.0),
                 lambda: p.run(0, a, a, a, a, 1.0)):
        with pytest.raises(bad, match="has changed since prepare"):
            call()
    b.prepare_lengths([c.ids[0]], [40])
    assert m.releaseSequence(c.ids[0]) is None
    with pytest.raises(bad, match="has changed since prepare"):
        b.attention(0, a, a, 1.0)
    torch.cuda.synchronize()


def test_pool_without_blocks(tl):
    c = QuantCache(tl, [60, 60], 1, 32, seed=22, blocks=4, room=160)
    assert c.mgr.freeBlocks() == 0
    x = torch.zeros((40, 32), dtype=torch.float16, device="cuda")
    assert "exhausted" in c.mgr.appendKV(c.ids[0], 0, x.data_ptr(), x.data_ptr(), 5)
    p = tl.PrefillBatch(c.mgr, 2, 1)
    with pytest.raises(tl.TinyLLMError, match="exhausted"):
        p.prepare(c.ids, [5, 1])
    p.append(0, x.data_ptr(), x.data_ptr())  # an empty batch
    c.append([4, 4])
    c.check()


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("G,d", [(4, 64), (1, 128)])
def test_a_model_step_by_step(tl, G, d):
    """Prompts, then steps: rotation, append and attention, two layers, beside a cache in
    fp16 that takes the same calls."""
    layers, hkv, hq, lens, rng = 2, 2, 2 * G, [70, 33, 1], np.random.default_rng(23)
    args = dict(num_layers=layers, num_heads=hkv, head_dim=d, max_seq_len=160, max_batch_size=3, block_tokens=32, num_blocks=15)
    m8, m16 = tl.KVCacheManager(quantized=True, **args), tl.KVCacheManager(**args)
    ids = [[m.allocateSequence(160)[0] for _ in lens] for m in (m8, m16)]
    rot = tl.Rotary(d, theta=1e6)
    w = dev((1 + 0.1 * rng.standard_normal((2, d))).astype(np.float16))
    batches = [(tl.PrefillBatch(m, 3, hq), tl.DecodeBatch(m, 3, hq)) for m in (m8, m16)]
    at, seen = list(lens), [[[np.zeros((0, hkv, d), np.float16) for _ in lens] for _ in range(layers)] for _ in range(2)]
    for step in range(40):
        counts = lens if step == 0 else [1] * 3
        pos = np.concatenate([np.arange(n) + (0 if step == 0 else a) for a, n in zip(at, counts)]).astype(np.int32)
        t = len(pos)
        for (p, b), i in zip(batches, ids):
            p.prepare(i, counts) if step == 0 else b.prepare(i)
        for layer in range(layers):
            x = dev(rng.standard_normal((t, (hq + 2 * hkv) * d)).astype(np.float16))
            q, k = (torch.empty((t, h, d), dtype=torch.float16, device="cuda") for h in (hq, hkv))
            v, dp = x[:, (hq + hkv) * d:].contiguous(), dev(pos)
            rot.apply(x.data_ptr(), x[:, hq * d:].data_ptr(), q.data_ptr(), k.data_ptr(), dp.data_ptr(), t, hq, hkv,
                      w[0].data_ptr(), w[1].data_ptr(), 1e-5, x.stride(0), x.stride(0))
            outs = []
            for p, b in batches:
                o = torch.empty_like(q)
                (p.run if step == 0 else b.decode)(layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), d ** -0.5)
                outs.append(o.float())
            torch.cuda.synchronize()
            assert (outs[0] - outs[1]).norm() <= 0.03 * outs[1].norm()  # (half steps of 1 / 127 of a maximum of 3 to 4 sigma)
            first = 0
            for i, n in enumerate(counts):
                for w_, y in enumerate((k, v)):
                    seen[w_][layer][i] = np.concatenate([seen[w_][layer][i], y[first:first + n].view(n, hkv, d).cpu().numpy()])
                kk, vv = held(seen[0][layer][i]), held(seen[1][layer][i])
                o, mass, err = attend(q[first:first + n].cpu().numpy(), kk, vv, d ** -0.5, len(kk) - n + np.arange(n))
                check_out(outs[0][first:first + n].cpu().numpy(), o, mass, err, len(kk), np.abs(vv).max())
                first += n
        for p, b in batches:
            p.commit() if step == 0 else b.commit(1)
        at = [a + n for a, n in zip(at, counts)] if step else at
    assert [m8.getSeqLen(s) for s in ids[0]] == [n + 39 for n in lens]
