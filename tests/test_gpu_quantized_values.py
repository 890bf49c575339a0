"""GPU: attention over a cache in 8 bits -- the bits that the weights have, and that every
token has its part once -- against 64-bit arithmetic."""
import numpy as np
import pytest
import torch

import quant_marks as marks
from quant_ref import QuantCache, attend, check_out, held
from retention_ref import dev

pytestmark = pytest.mark.gpu


def step(tl, c, q, k, v, counts, scale):
    """counts[i] tokens for sequence i of layer 0, appended and attended to: one each by
    DecodeBatch, else by PrefillBatch.  Not committed."""
    one = set(counts) == {1}
    out = torch.zeros((len(q), q.shape[1], c.d), dtype=torch.float16, device="cuda")
    dq, dk, dv = dev(q), dev(k), dev(v)
    b = (tl.DecodeBatch if one else tl.PrefillBatch)(c.mgr, len(counts), q.shape[1])
    b.prepare(c.ids) if one else b.prepare(c.ids, counts)
    (b.decode if one else b.run)(0, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), out.data_ptr(), scale)
    torch.cuda.synchronize()
    return b, out.cpu().numpy()


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("lens,count", [([33, 63, 40, 90], 1), ([20, 30, 64, 77], 3)])
def test_weights_are_not_rounded_to_fp16(tl, d, lens, count):
    """Up to 16 query rows: a weight takes part with 22 bits, as its upper and lower half in fp16.
    With near scores every weight counts as much, so that one rounded to 11 bits would
    show: by up to 2^-12 of it on average, where the bound allows 2^-22 and what sums of fp32 lose."""
    c = QuantCache(tl, lens, 2, d, seed=d + count, hq=8)
    n = len(lens) * count
    q = (c.rng.standard_normal((n, 8, d)) / 16).astype(np.float16)
    k, v = c.rows(n), c.rows(n)
    _, got = step(tl, c, q, k, v, [count] * len(lens), d ** -0.5)
    for i, s in enumerate(lens):
        at = slice(i * count, (i + 1) * count)
        hk, hv = held(np.concatenate([c.k[0][i], k[at]])), held(np.concatenate([c.v[0][i], v[at]]))
        o, mass, err = attend(q[at], hk, hv, d ** -0.5, s + np.arange(count))
        # The weight: 2^-22 of it, 2^-32 of the largest where its lower half is below fp16's normal
        # numbers; its score's error, and twice that of the exponential (2^-22).  A product's sum is one of
        # 64 addends at most (two halves of 32 tokens), then come the groups, the waves and the row sum: 3
        # groups, 8 waves, 4 lanes' sums of 8 a group; each at most 2^-24 of the mass.  The output: 2^-11 of it.
        rel = 2 * 2.0 ** -22 + 2 * err + 2 * 2.0 ** -22 + (64 + 3 + 8 + 2 + 24 + 8) * 2.0 ** -24
        tol = 2.0 ** -11 * np.abs(o) + rel[..., None] * mass + 1e-6 * np.abs(o) + 2.0 ** -25 + s * 2.0 ** -32 * np.abs(hv).max()
        bad = ~(np.abs(got[at].astype(np.float64) - o) <= tol)
        assert not bad.any(), (bad.mean(), (np.abs(got[at] - o) / tol).max())


# d, kv heads, group, lengths before the step: whole, in few and in many chunks, of workgroups of all and of two waves
EACH_DECODE = [
    (128, 8, 4, [33000, 31]),
    (64, 1, 8, [20000]),
    (128, 1, 4, [9000]),
    (32, 2, 8, [7000, 95]),
    (256, 2, 2, [4100, 700]),
    (64, 64, 2, [0, 63, 64, 95, 31, 300]),
    (128, 64, 1, [0, 31, 500, 1279, 100]),
]
# and the tokens of the step
EACH_PREFILL = [
    (128, 8, 4, [3000], [4]),       # the decode kernel
    (64, 1, 2, [9001], [8]),
    (128, 8, 4, [30000, 40], [100, 33]),
    (128, 1, 8, [0, 4000], [500, 20]),
    (64, 2, 8, [5000, 31], [40, 90]),
    (64, 1, 4, [0], [2000]),
    (256, 2, 2, [2500, 0], [70, 300]),
    (32, 2, 4, [6000, 100], [130, 64]),
]


def marked(tl, d, hkv, G, lens, counts):
    """A cache of marked tokens, the rows of a step, and all of them: (cache, k, v, [(v, classes)])."""
    c = QuantCache(tl, [0] * len(lens), hkv, d, block=256, hq=hkv * G, room=max(n + m for n, m in zip(lens, counts)) + 1)
    old = [marks.rows(0, n, hkv, d, i) for i, n in enumerate(lens)]
    c.append(lens, "prefill", [([x[0] for x in old], [x[1] for x in old])])
    new = [marks.rows(n, m, hkv, d, i) for i, (n, m) in enumerate(zip(lens, counts))]
    whole = [(np.concatenate([o[1], n[1]]), np.concatenate([o[2], n[2]])) for o, n in zip(old, new)]
    return c, np.concatenate([x[0] for x in new]), np.concatenate([x[1] for x in new]), whole


def check_marked(got, whole, hkv, G, d, lens, counts, qcls):
    """got, [tokens][hq][d], for queries of the classes qcls [tokens][hq]: rows of every token of the step."""
    at = 0
    for i, (n, m) in enumerate(zip(lens, counts)):
        for h in range(hkv * G):
            v, cls = whole[i][0][:, h // G], whole[i][1][:, h // G]
            want, count = marks.expect(v, cls, d, n + np.arange(m), qcls[at:at + m, h])
            seen = count > 0  # (a class that no token has: the mean of whatever is there)
            err = np.abs(got[at:at + m, h][seen].astype(np.float64) - want[seen])
            assert (err <= marks.tolerance(want[seen], n + m)).all(), (i, h, err.max())
        at += m


@pytest.mark.parametrize("d,hkv,G,lens", EACH_DECODE)
def test_every_token_once_in_a_step(tl, d, hkv, G, lens):
    """Every class in turn, so every token of every sequence, the step's own among them."""
    ones, scale = [1] * len(lens), d ** -0.5
    c, k, v, whole = marked(tl, d, hkv, G, lens, ones)
    b = tl.DecodeBatch(c.mgr, len(lens), hkv * G)
    b.prepare(c.ids)
    dk, dv = dev(k), dev(v)
    out = torch.zeros((len(lens), hkv * G, d), dtype=torch.float16, device="cuda")
    for first in range(0, d, G):
        qcls = np.broadcast_to((first + np.arange(hkv * G) % G)[None], (len(lens), hkv * G))
        dq = dev(marks.queries(qcls, d, scale))
        b.decode(0, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), out.data_ptr(), scale)
        torch.cuda.synchronize()
        check_marked(out.cpu().numpy(), whole, hkv, G, d, lens, ones, qcls)


@pytest.mark.parametrize("d,hkv,G,lens,counts", EACH_PREFILL)
def test_every_token_once_in_a_prompt(tl, d, hkv, G, lens, counts):
    n, scale = sum(counts), d ** -0.5
    c, k, v, whole = marked(tl, d, hkv, G, lens, counts)
    p = tl.PrefillBatch(c.mgr, len(lens), hkv * G)
    p.prepare(c.ids, counts)
    dk, dv = dev(k), dev(v)
    out = torch.zeros((n, hkv * G, d), dtype=torch.float16, device="cuda")
    # Rows of up to 16: every class for every token; more: all classes among the rows of a tile, in two orders.
    # Then every token's own class, which it sees, and that of the next one, which it does not.
    few, heads = max(m * G for m in counts) <= 16, np.arange(hkv * G)
    classes = [(np.arange(n)[:, None] * (0 if few else G) + heads[None] % G + step) % d
               for step in (range(0, d, G) if few else (0, 37))]
    for ahead in (0, 1):
        at = [np.minimum(a + np.arange(m) + ahead, a + m - 1) for a, m in zip(lens, counts)]
        classes.append(np.concatenate([w[1][x][:, heads // G] for w, x in zip(whole, at)]).astype(np.int64))
    for qcls in classes:
        dq = dev(marks.queries(qcls, d, scale))
        p.run(0, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), out.data_ptr(), scale)
        torch.cuda.synchronize()
        check_marked(out.cpu().numpy(), whole, hkv, G, d, lens, counts, qcls)


# ------------------------------------------------------------------ what is not finite, where keys are cut
@pytest.mark.parametrize("d,hkv,G,prefix,count", [(64, 1, 8, 20000, 1), (128, 1, 4, 9000, 1), (256, 2, 2, 4100, 1), (32, 2, 8, 7000, 2),
                                                  (128, 8, 4, 3000, 40), (64, 1, 2, 5000, 20), (256, 2, 1, 2500, 20), (32, 1, 4, 6000, 33)])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_not_finite_where_keys_are_cut(tl, d, hkv, G, prefix, count, where, bad):
    """In a closed group of one chunk: NaN for all rows of that kv head, none of the others.  In the step's
    last token, in the open group: for who sees it, an infinite value its dim alone."""
    for at in (prefix // 2, prefix + count - 1):
        if (prefix + count) % 32 == 0 and at >= prefix:
            continue
        c = QuantCache(tl, [0], hkv, d, seed=41, hq=hkv * G, block=256, room=prefix + count + 8)
        old, new = c.new_rows([prefix])[0], c.new_rows([count])[0]
        rows = [np.concatenate([o[0], n[0]]) for o, n in zip(old, new)]
        rows["kv".index(where)][at, 0, 7] = bad
        c.append([prefix], "prefill", [([rows[0][:prefix]], [rows[1][:prefix]])])
        q = c.rng.standard_normal((count, hkv * G, d)).astype(np.float16)
        _, got = step(tl, c, q, rows[0][prefix:], rows[1][prefix:], [count], d ** -0.5)
        first = 0 if at < prefix else count - 1  # the first row that sees it
        if at < prefix:
            assert np.isnan(got[:, :G]).all()
        elif where == "v":
            own = got[first:, :G]
            assert not np.isfinite(own[..., 7]).any() and np.isfinite(np.delete(own, 7, axis=2)).all()
            if np.isinf(bad):
                assert (own[..., 7] == bad).all()
        else:
            sign = q[first, :G, 7].astype(np.float64) * bad  # of the infinite score
            for h in range(G):
                if not sign[h] < 0 or np.isnan(bad):
                    assert np.isnan(got[first, h]).all()
        rows["kv".index(where)][at, 0, 7] = 0
        hk, hv = held(rows[0]), held(rows[1])
        o, mass, err = attend(q, hk, hv, d ** -0.5, prefix + np.arange(count))
        sees = np.zeros((count, hkv * G), bool)
        sees[first:, :G] = True
        check_out(got[~sees][:, None], o[~sees][:, None], mass[~sees][:, None], err[~sees][:, None], prefix + count, np.abs(hv).max())
        if at >= prefix and where == "k" and np.isinf(bad):  # a score of -infinity has no weight
            for h in range(G):
                if q[first, h, 7] * bad < 0:
                    o, mass, err = attend(q[first:, h:h + 1], hk[:-1, :1], hv[:-1, :1], d ** -0.5, [prefix + count - 2])
                    check_out(got[first:, h:h + 1], o, mass, err, prefix + count, np.abs(hv).max())


def test_layers_from_one_on(tl):
    """One call's tokens for layers 1 and 2 of four: the others stay as they were."""
    c = QuantCache(tl, [31, 40, 62], 2, 64, seed=42, layers=4)
    b = tl.DecodeBatch(c.mgr, 3, 2)
    b.prepare(c.ids)
    new = c.new_rows([1, 1, 1])
    k, v = (dev(np.stack([np.concatenate(new[layer][w]) for layer in (1, 2)])) for w in (0, 1))
    b.append(1, 2, k.data_ptr(), v.data_ptr())
    torch.cuda.synchronize()
    c.check()
    for layer in (1, 2):
        for i in range(3):
            c.k[layer][i] = np.concatenate([c.k[layer][i], new[layer][0][i]])
            c.v[layer][i] = np.concatenate([c.v[layer][i], new[layer][1][i]])
        got = c.read(layer, [32, 41, 63])
        for w in range(2):
            for i, n in enumerate((32, 41, 63)):
                assert np.array_equal(got[w][i][:, :n], c.expect(layer, i)[w].astype(np.float16).transpose(1, 0, 2))
