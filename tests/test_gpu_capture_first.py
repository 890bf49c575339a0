"""GPU: a captured call whose kernels have not run before, where the workspace is large
enough from other calls of the batch."""
import numpy as np
import pytest
import torch

from retention_ref import Cache, dev

pytestmark = pytest.mark.gpu


def captured(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    return graph


@pytest.mark.parametrize("d,G", [(32, 8), (256, 8), (64, 8)])
def test_a_plan_that_has_not_run(tl, d, G):
    """Split entries first, then whole ones on eight waves (four at 256), captured at once."""
    c = Cache(tl, [6000, 600], 4, d, seed=d, hq=4 * G)
    b, x = tl.DecodeBatch(c.mgr, 2, 4 * G), tl.CrossBatch(c.mgr, 2, 4 * G)
    q = dev(c.rng.standard_normal((300, 4 * G, d)).astype(np.float16))
    outs = [torch.zeros_like(q) for _ in range(4)]
    accs = [c.account() for _ in range(2)]
    b.prepare_lengths(c.ids, [6000, 600])
    b.decode_weights(0, q.data_ptr(), None, None, outs[0].data_ptr(), d ** -0.5, None, accs[0].data_ptr())
    x.prepare(c.ids, [100, 200])
    x.attention(0, q.data_ptr(), outs[0].data_ptr(), d ** -0.5)
    torch.cuda.synchronize()
    b.prepare_lengths(c.ids[1:], [600])
    x.prepare(c.ids[1:] * 2, [1, 1], [500, 600])

    def decode(i):
        return lambda s=0: b.decode_weights(0, q.data_ptr(), None, None, outs[i].data_ptr(), d ** -0.5, None, accs[i].data_ptr(), s)

    def cross(i):
        return lambda s=0: x.attention(0, q.data_ptr(), outs[i].data_ptr(), d ** -0.5, s)

    outs[0].zero_(), accs[0].zero_()
    torch.cuda.synchronize()
    graphs = [captured(decode(0)), captured(cross(2))]
    decode(1)()
    cross(3)()
    torch.cuda.synchronize()
    for _ in range(3):
        outs[0].zero_(), outs[2].zero_(), accs[0].zero_()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0][:1], outs[1][:1]) and torch.equal(outs[2][:2], outs[3][:2]) and outs[1][0].any()
        assert torch.equal(accs[0], accs[1]) and accs[0].any()
        decode(1)()
        cross(3)()
        torch.cuda.synchronize()
