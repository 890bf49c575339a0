"""GPU: what the accounts of a decode step allocate, and results where only some of a
step's entries need it."""
import pytest
import torch

from retention_ref import Cache
from test_gpu_accounts import decode_step

pytestmark = pytest.mark.gpu


def test_scores_of_whole_entries_have_no_workspace(tl):
    """They stay in a workgroup's LDS: 64 MiB here, if they were counted."""
    n, S, hkv, d, hq = 64, 4096, 8, 32, 64
    mgr = tl.KVCacheManager(num_layers=1, num_heads=hkv, head_dim=d, max_seq_len=S, max_batch_size=n)
    ids = [mgr.allocateSequence(S)[0] for _ in range(n)]
    b = tl.DecodeBatch(mgr, n, hq)
    b.prepare_lengths(ids, [S] * n)
    q, acc = torch.randn((n, hq, d), device="cuda").half(), torch.zeros((n, hkv, S), device="cuda")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    b.decode_weights(0, q.data_ptr(), None, None, out.data_ptr(), 0.1, None, acc.data_ptr())
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] < 8 << 20
    # an empty cache of zeros: even weights
    assert (acc * (S / 8) - 1).abs().max() <= (S + 20) * 2.0 ** -23


@pytest.mark.parametrize("block", [0, 16])
@pytest.mark.parametrize("d,hkv,G,lens", [
    (64, 8, 2, [50] * 20 + [4000, 3000] + [700] * 10),  # several chunks among whole entries, of one launch
    (128, 8, 8, [9000] + [600, 0, 5000] * 20),
    (32, 2, 8, [3000] * 3 + [20] * 150 + [2500]),       # ... of two
])
def test_whole_entries_between_split_ones(tl, d, hkv, G, lens, block):
    c = Cache(tl, lens, hkv, d, block=block, seed=d + 5, hq=hkv * G)
    decode_step(tl, c, lens, G)
