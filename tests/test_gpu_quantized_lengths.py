"""GPU: lengths of sequences in a cache in 8 bits that do not follow the appends: beyond what was
appended, and where several batches append to the same sequences."""
import numpy as np
import pytest
import torch

from quant_ref import QuantCache
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
