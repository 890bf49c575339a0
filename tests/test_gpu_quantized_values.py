"""GPU: attention over a cache in 8 bits -- the bits that the weights have, and that every
token has its part once -- against 64-bit arithmetic."""
import numpy as np
import pytest
import torch

from quant_ref import QuantCache, attend, held
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
