"""GPU: Rotary over rows of zeros."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [1e-6, 0.0])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_rows_of_zeros(tl, d, eps):
    """With eps they stay zeros; without, 0 / 0 is NaN, as the formula's.  Other rows of the call do not feel it."""
    x = torch.zeros((3, 2, d), dtype=torch.float16, device="cuda")
    x[1, 1] = 1.0
    w, pos = torch.ones(d, dtype=torch.float16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    out = torch.ones_like(x)
    tl.Rotary(d).apply(x.data_ptr(), None, out.data_ptr(), None, pos.data_ptr(), 3, 2, 0, w.data_ptr(), eps=eps)
    torch.cuda.synchronize()
    assert (out[1, 1] == 1.0).all()  # (1 / sqrt(1 + eps) rounds to 1)
    out[1, 1] = out[0, 0]
    assert not out.any() if eps else torch.isnan(out).all()
