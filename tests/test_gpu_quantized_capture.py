"""GPU: captured calls over a cache in 8 bits whose kernels have not run before (in a process of their own)."""
import numpy as np
import pytest
import torch

from quant_ref import QuantCache
from retention_ref import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_first_calls_captured(tl, d):
    """Steps of whole entries, on workgroups of all and of two waves, append, prompt and gather: one launch each."""
    many = 600 // 64 + 1  # entries of 64 kv heads: more than two a CU
    for hkv, n in ((2, 3), (64, many)):
        c = QuantCache(tl, [0] * n, hkv, d, seed=d + n, hq=2 * hkv, room=200)
        k, v = dev(c.rows(60 * n)), dev(c.rows(60 * n))
        q = dev(c.rng.standard_normal((60 * n, 2 * hkv, d)).astype(np.float16))
        outs = [torch.zeros_like(q) for _ in range(2)]
        back = [torch.zeros((n, hkv, 70, d), dtype=torch.float16, device="cuda") for _ in range(2)]
        p, b = tl.PrefillBatch(c.mgr, n, 2 * hkv), tl.DecodeBatch(c.mgr, n, 2 * hkv)

        def prompt(i, s=0):
            p.run(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[i].data_ptr(), 0.1, s)

        def one(i, s=0):
            b.decode(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[i].data_ptr(), 0.1, s)
            b.append(0, 1, k.data_ptr(), v.data_ptr(), s)
            b.attention(0, q.data_ptr(), outs[i][n:].data_ptr(), 0.1, s)
            b.gather(0, back[i].data_ptr(), None, 70, s)

        for step, prepare in ((prompt, lambda: p.prepare(c.ids, [60] * n)), (one, lambda: b.prepare(c.ids))):
            prepare()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step(0, torch.cuda.current_stream().cuda_stream)
            for _ in range(3):
                outs[0].zero_(), outs[1].zero_(), back[0].zero_(), back[1].zero_()
                step(1)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(*outs) and outs[0].any() and torch.equal(*back)
            p.commit() if step is prompt else b.commit(1)
        assert [c.mgr.getSeqLen(s) for s in c.ids] == [61] * n
