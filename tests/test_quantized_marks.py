"""CPU: the marked sequences of the 8-bit cache's GPU tests show one token too many or too few, at
every length that those tests use; the plain form of attention agrees with them."""
import numpy as np
import pytest

import quant_marks as marks
from quant_ref import attend, held
from test_gpu_quantized_values import EACH_DECODE, EACH_PREFILL


@pytest.mark.parametrize("d,length,hkv", sorted({(d, n + (1 if np.isscalar(m) else m[i]), hkv)
                                                  for d, hkv, _, lens, m in [(*x, 1) for x in EACH_DECODE] + EACH_PREFILL
                                                  for i, n in enumerate(lens)}))
def test_every_token_shows(d, length, hkv):
    """Leaving out, or doubling, any one of them moves some dim by more than twice the bound."""
    _, v, cls = marks.rows(0, length, hkv, d, 0)
    for h in {0, hkv - 1}:
        vv, cc = v[:, h].astype(np.float64), cls[:, h].astype(np.int64)
        count = np.bincount(cc, minlength=d)
        mean = np.zeros((d, d))
        np.add.at(mean, cc, vv)
        mean /= np.maximum(count, 1)[:, None]
        n, o = count[cc][:, None], mean[cc]
        tol = 2 * marks.tolerance(o, length)
        alone = n[:, 0] == 1  # (without its only token a class has some other mean: of all the rest)
        without = np.abs((n * o - vv) / np.maximum(n - 1, 1) - o)
        twice = np.abs((n * o + vv) / (n + 1) - o)
        assert ((without > tol).any(1) | alone).all()
        assert ((twice > tol).any(1) | alone).all()


@pytest.mark.parametrize("d,length", [(32, 70), (64, 33), (128, 400)])
def test_plain_attention_of_marked_tokens(d, length):
    k, v, cls = marks.rows(0, length, 2, d, 5)
    assert np.array_equal(held(k), k) and np.array_equal(held(v), v)  # nothing is rounded
    a = [np.concatenate(x) for x in zip(marks.rows(0, 7, 2, d, 5), marks.rows(7, length - 7, 2, d, 5))]
    assert all(np.array_equal(x, y) for x, y in zip(a, (k, v, cls)))
    qcls = np.stack([cls[:, h][np.arange(20) % length] for h in range(2)], axis=1)  # classes that some token has
    last = np.full(20, length - 1)
    o, _, _ = attend(marks.queries(qcls, d, 0.125), held(k), held(v), 0.125, last)
    for h in range(2):
        want, count = marks.expect(v[:, h], cls[:, h], d, last, qcls[:, h])
        assert (count > 0).all() and np.abs(o[:, h] - want).max() < 1e-9
