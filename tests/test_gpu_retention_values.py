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
