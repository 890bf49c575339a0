"""GPU: accounts and attention to cached states on values at the edges -- infinite
scores, weights between two fp16 numbers, scores far from zero."""
import numpy as np
import pytest
import torch

from retention_ref import Cache, attend, check_account, check_out, dev

pytestmark = pytest.mark.gpu


def cache_of(tl, k, v, hq, block=0):
    """A cache of one sequence that holds these rows [S][hkv][d]."""
    c = Cache(tl, [0], k.shape[1], k.shape[2], room=len(k) + 8, block=block, hq=hq)
    parts = iter([k, v])
    c.rows = lambda n, std=1.0: next(parts)
    c.append([len(k)])
    return c


def decode(tl, c, q, scale):
    """q [1][hq][d] over all of the cache: output and account, as arrays."""
    b = tl.DecodeBatch(c.mgr, 1, q.shape[1])
    S = c.mgr.getSeqLen(c.ids[0])
    b.prepare_lengths(c.ids, [S])
    dq, w = dev(q), c.account()
    out = torch.empty_like(dq)
    b.decode_weights(0, dq.data_ptr(), None, None, out.data_ptr(), scale, None, w.data_ptr())
    torch.cuda.synchronize()
    return out.cpu().numpy(), w.cpu().numpy()[0, :, :S]


def cross(tl, c, q, scale):
    b = tl.CrossBatch(c.mgr, 1, q.shape[1])
    b.prepare(c.ids, [len(q)])
    dq = dev(q)
    out = torch.empty_like(dq)
    b.attention(0, dq.data_ptr(), out.data_ptr(), scale)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def hidden_states(d, S, hidden, seed):
    """Queries and states; the states at `hidden` have scores of -infinity."""
    rng = np.random.default_rng(seed)
    k, v = (rng.standard_normal((S, 1, d)).astype(np.float16) for _ in range(2))
    k[hidden, 0, 3] = -np.inf
    q = rng.standard_normal((40, 2, d)).astype(np.float16)
    q[..., 3] = np.abs(q[..., 3]) + np.float16(0.1)
    return q, k, v, np.setdiff1d(np.arange(S), np.arange(S)[hidden])


# All of a wave's tiles, of a work item, the first tiles of an entry, the last ones, all but one.
HIDDEN = [(64, 5000, slice(0, 700)), (128, 5000, slice(1000, 4000)), (32, 300, slice(0, 70)), (64, 200, slice(130, 200)),
          (256, 2500, slice(0, 2400)), (128, 9000, slice(1, 9000))]


@pytest.mark.parametrize("d,S,hidden", HIDDEN)
def test_scores_of_minus_infinity_in_an_account(tl, d, S, hidden):
    q, k, v, seen = hidden_states(d, S, hidden, 1)
    got, acc = decode(tl, cache_of(tl, k, v, 2), q[:1], d ** -0.5)
    o, mass, w, err = attend(q[:1], k[seen], v[seen], d ** -0.5)
    check_out(got, o, mass, err, S)
    check_account(acc[:, seen], w.sum(axis=0), w, err, 2, len(seen))
    assert not np.delete(acc, seen, axis=1).any()


@pytest.mark.parametrize("nq", [2, 7, 20, 40])
@pytest.mark.parametrize("d,S,hidden", HIDDEN)
def test_scores_of_minus_infinity_in_cross_attention(tl, d, S, hidden, nq):
    q, k, v, seen = hidden_states(d, S, hidden, 2)
    o, mass, _, err = attend(q[:nq], k[seen], v[seen], d ** -0.5)
    check_out(cross(tl, cache_of(tl, k, v, 2), q[:nq], d ** -0.5), o, mass, err, S)


@pytest.mark.parametrize("nq", [1, 3, 30])
def test_queries_whose_scores_are_all_minus_infinity(tl, nq):
    """There is nothing to attend to: zeros, as over no states."""
    for S in (40, 3000):
        q, k, v, _ = hidden_states(64, S, slice(0, S), 3)
        assert not cross(tl, cache_of(tl, k, v, 2), q[:nq], 0.125).any()


def half_step(S, d, seed=4):
    """Half of the states have weights beside the others' that fp16 does not tell apart,
    and values of the other sign: what is left of the sum is the difference, which is of
    the size of a weight's rounding to fp16.  (q, k, v, out, tolerance at a scale of 1)"""
    rng = np.random.default_rng(seed)
    k, v = np.zeros((S, 1, d), np.float16), np.ones((S, 1, d), np.float16)
    heavy = rng.permutation(S)[:S // 2]
    k[heavy, 0, 0], v[heavy] = 1.5 * 2.0 ** -12, -1.0
    q = np.zeros((40, 2, d), np.float16)
    q[..., 0] = 1.0
    s = 1.5 * 2.0 ** -12
    n, m = S - S // 2, S // 2
    out = (n - m * np.exp(s)) / (n + m * np.exp(s))
    # Scores are one product (4 roundings of 2^-24 with the logarithm's, of s < 2^-11); exp2 and
    # the division of 2 + 2; a weight in two parts 2^-22, half a step of the second one's 11 bits; sums of S
    # terms of the same size, pairwise per lane (S / 16 long) and tile; the output's rounding, and the 1e-6 beside
    # a sum of 2^7 S.
    tol = 2.0 ** -22 + (4 * s + 4 + S / 16 + 16) * 2.0 ** -24 + 2.0 ** -11 * abs(out) + 2.0 ** -24
    return q, k, v, out, tol


@pytest.mark.parametrize("d,S,block", [(64, 2, 0), (32, 64, 16), (64, 200, 16), (128, 500, 0), (256, 330, 0), (128, 1200, 16)])
def test_weights_between_two_fp16_numbers(tl, d, S, block):
    q, k, v, out, tol = half_step(S, d)
    c = cache_of(tl, k, v, 2, block)
    assert tol < 2.0 ** -12 / 4  # of what a rounding of the weights to fp16 would be
    got, acc = decode(tl, c, q[:1], 1.0)
    assert np.abs(got.astype(np.float64) - out).max() <= tol
    assert abs(acc.sum(dtype=np.float64) - 2) <= 2 * (S + 20) * 2.0 ** -23
    for nq in (1, 5, 8):
        assert np.abs(cross(tl, c, q[:nq], 1.0).astype(np.float64) - out).max() <= tol


@pytest.mark.parametrize("at", [0, 77, 199])
@pytest.mark.parametrize("nq", [1, 30])
def test_infinite_values(tl, nq, at):
    """An attended value of infinity makes its dimension infinite and no other one NaN."""
    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((200, 1, 64)).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((nq, 2, 64)).astype(np.float16)
    want, mass, _, err = attend(q, k, v, 0.125)
    v[at, 0, 5], v[at, 0, 9] = np.inf, -np.inf
    c = cache_of(tl, k, v, 2)
    for got in [cross(tl, c, q, 0.125)] + ([decode(tl, c, q, 0.125)[0]] if nq == 1 else []):
        assert (got[..., 5] == np.inf).all() and (got[..., 9] == -np.inf).all()
        rest = [i for i in range(64) if i not in (5, 9)]
        check_out(got[..., rest], want[..., rest], mass[..., rest], err, 200)


@pytest.mark.parametrize("a,b", [(40.0, 4000.0), (-77.0, 2500.0), (300.0, -515.0), (0.5, 3.0)])
@pytest.mark.parametrize("pre,new,window,G", [
    (0, 200, 0, 1), (0, 700, 0, 4),
    (3000, 3, 1, 2),       # few rows over many keys: their statistics are merged with the sums
    (5000, 130, 0, 4),     # ... in a launch of their own
])
def test_prompt_accounts_of_scores_far_from_zero(tl, pre, new, window, G, a, b):
    """Equal scores, exact in fp32: every weight is 1 / (keys that its row sees)."""
    d = 64
    c = Cache(tl, [0], 1, d, room=pre + new, hq=G)

    def same(n, std=1.0):
        k = np.zeros((n, 1, d), np.float16)
        k[..., 7] = a
        return k

    c.rows = same
    c.append([pre])
    q = np.zeros((new, G, d), np.float16)
    q[..., 7] = b
    p = tl.PrefillBatch(c.mgr, 1, G)
    p.prepare(c.ids, [new])
    dq, dk, w = dev(q), dev(same(new)), c.account()
    p.append(0, dk.data_ptr(), dk.data_ptr())
    p.weights(0, dq.data_ptr(), 0.125, window, None, w.data_ptr())
    torch.cuda.synchronize()
    S = pre + new
    weight = G / (1.0 + np.arange(S))
    weight[:S - (window or new)] = 0  # rows that are not counted
    want = np.cumsum(weight[::-1])[::-1]
    got = w.cpu().numpy()[0, 0, :S].astype(np.float64)
    # exp2 and the multiply-adds of both passes (12 roundings), and fp32 sums of S and of G * new terms; a score
    # and its reference are one product, whose rounding both have
    assert np.abs(got / want - 1).max() <= (12 + S + G * new) * 2.0 ** -24


@pytest.mark.parametrize("pre,new,window,hidden", [(70, 300, 0, slice(64, 256)), (3000, 4, 0, slice(10, 2990)), (500, 200, 30, slice(1, 690))])
def test_scores_of_minus_infinity_in_a_prompt_account(tl, pre, new, window, hidden):
    q, k, v, seen = hidden_states(64, pre + new, hidden, 6)
    q = np.random.default_rng(7).standard_normal((new, 2, 64)).astype(np.float16)
    q[..., 3] = np.abs(q[..., 3]) + np.float16(0.1)
    c = Cache(tl, [0], 1, 64, room=pre + new, hq=2)
    parts = iter([k[:pre], v[:pre]])
    c.rows = lambda n, std=1.0: next(parts)
    c.append([pre])
    p = tl.PrefillBatch(c.mgr, 1, 2)
    p.prepare(c.ids, [new])
    dq, dk, w = dev(q), dev(k[pre:]), c.account()
    p.append(0, dk.data_ptr(), dk.data_ptr())
    p.weights(0, dq.data_ptr(), 0.125, window, None, w.data_ptr())
    torch.cuda.synchronize()
    n = window or new
    positions = np.arange(pre + new - n, pre + new)
    last = np.searchsorted(seen, positions, side="right") - 1  # among the keys that have weights
    _, _, weights, err = attend(q[new - n:], k[seen], k[seen], 0.125, last)
    got = w.cpu().numpy()[0, :, :pre + new]
    check_account(got[:, seen], weights.reshape(1, 2 * n, len(seen)).sum(axis=1), weights, err, 2 * n, len(seen))
    assert not np.delete(got, seen, axis=1).any()


@pytest.mark.parametrize("S", [40, 3000])
def test_a_query_without_finite_scores_counts_nothing(tl, S):
    """Zeros for an output, and the account as the other heads' queries leave it."""
    rng = np.random.default_rng(8)
    k, v = (rng.standard_normal((S, 1, 64)).astype(np.float16) for _ in range(2))
    k[:, 0, 3] = -np.inf
    q = rng.standard_normal((1, 2, 64)).astype(np.float16)
    q[0, :, 3] = [1.0, 0.5]
    c = cache_of(tl, k, v, 2)
    got, acc = decode(tl, c, q, 0.125)
    assert not got.any() and not acc.any()
    # a prompt's first rows see hidden keys only, the others also the last ones
    new = S // 2
    k[new:, 0, 3] = 0.0
    c = Cache(tl, [0], 1, 64, room=S, hq=2)
    p = tl.PrefillBatch(c.mgr, 1, 2)
    p.prepare(c.ids, [S])
    qs = rng.standard_normal((S, 2, 64)).astype(np.float16)
    qs[..., 3] = 1.0
    dq, dk, w = dev(qs), dev(k), c.account()
    p.append(0, dk.data_ptr(), dk.data_ptr())
    p.weights(0, dq.data_ptr(), 0.125, 0, None, w.data_ptr())
    torch.cuda.synchronize()
    rows = np.arange(new, S)
    _, _, weights, err = attend(qs[new:], k[new:], k[new:], 0.125, rows - new)
    got = w.cpu().numpy()[0, :, :S]
    check_account(got[:, new:], weights.reshape(1, 2 * len(rows), S - new).sum(axis=1), weights, err, 2 * len(rows), S - new)
    assert not got[:, :new].any()
