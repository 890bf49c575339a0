"""GPU: Rotary -- RMS norm of query and key heads and their rotation by position -- against
64-bit arithmetic."""
import numpy as np
import pytest
import torch

from retention_ref import dev

pytestmark = pytest.mark.gpu


def reference(x, w, pos, eps, rd, theta, interleaved, axis_of, inv_freq):
    """x [T][H][D] in 64 bits, and a bound of the error before the last rounding."""
    y = x.astype(np.float64)
    d, n = x.shape[-1], rd // 2
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    f = np.asarray(inv_freq) if inv_freq is not None else theta ** (-np.arange(n) / n)
    a = (pos.astype(np.float64)[axis_of].T * f)[:, None]
    i = (np.arange(0, rd, 2), np.arange(1, rd, 2)) if interleaved else (np.arange(n), np.arange(n, rd))
    z, size = y.copy(), np.abs(y)
    z[..., i[0]] = y[..., i[0]] * np.cos(a) - y[..., i[1]] * np.sin(a)
    z[..., i[1]] = y[..., i[0]] * np.sin(a) + y[..., i[1]] * np.cos(a)
    for u in i:
        size[..., u] = np.abs(y[..., i[0]]) + np.abs(y[..., i[1]])
    # fp32: a sum of d squares, its root, reciprocal and two products; sine and cosine of an angle that is
    # half a step of 2^-24 turns off (2 pi 2^-25) and a few steps wrong; two products and a sum
    return z, size * (d + 24) * 2.0 ** -24


def check(tl, t, hq, hkv, d, rd=None, theta=1e4, interleaved=False, axis_of=None, inv_freq=None, weights=(True, True), eps=1e-5,
          extra=0, far=2 ** 17, std=2.0, seed=0, pos=None, in_place=False):
    rng = np.random.default_rng(seed)
    rd = rd or d
    axes = 1 + (max(axis_of) if axis_of else 0)
    rows = (rng.standard_normal((t, (hq + hkv) * d + extra)) * std).astype(np.float16)
    w = [(1 + 0.3 * rng.standard_normal(d)).astype(np.float16) if on else None for on in weights]
    pos = rng.integers(-5, far, (axes, t)).astype(np.int32) if pos is None else pos
    x, dw, dp = dev(rows), [None if a is None else dev(a) for a in w], dev(pos)
    q, k = rows[:, :hq * d].reshape(t, hq, d), rows[:, hq * d:(hq + hkv) * d].reshape(t, hkv, d)
    outs = [torch.full((t + 1, h, d), 9.0, dtype=torch.float16, device="cuda") for h in (hq, hkv)]
    src, strides = (x.data_ptr(), x[:, hq * d:].data_ptr()), (x.stride(0), x.stride(0))
    if in_place:
        outs[0][:t], outs[1][:t] = dev(q), dev(k)
        src, strides = tuple(o.data_ptr() for o in outs), (0, 0)
    r = tl.Rotary(d, rd, theta, interleaved, axis_of, inv_freq)
    r.apply(*src, *(o.data_ptr() for o in outs), dp.data_ptr(), t, hq, hkv, *(None if a is None else a.data_ptr() for a in dw),
            eps, *strides, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for got, a, b in zip(outs, (q, k), w):
        got = got.cpu().numpy()
        assert (got[t:] == 9.0).all()
        want, err = reference(a, b, pos, eps, rd, theta, interleaved, axis_of or [0] * (rd // 2), inv_freq)
        tol = err + np.abs(want) * 2.0 ** -11 * 1.001 + 2.0 ** -25
        bad = ~(np.abs(got[:t].astype(np.float64) - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got[:t] - want).max())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rd", [(32, 32), (32, 16), (64, 64), (64, 48), (128, 128), (128, 64), (128, 16), (256, 256), (256, 208)])
def test_dims(tl, d, rd, interleaved):
    for t, hq, hkv in [(1, 1, 1), (3, 8, 2), (37, 5, 3)]:
        check(tl, t, hq, hkv, d, rd, interleaved=interleaved, seed=d + rd + t)


@pytest.mark.parametrize("weights", [(True, True), (False, False), (True, False), (False, True)])
def test_norms(tl, weights):
    for std in (2.0 ** -12, 1.0, 3000.0):
        check(tl, 9, 6, 2, 128, weights=weights, std=std, seed=1)
    check(tl, 9, 6, 2, 128, weights=weights, eps=0.5, seed=2)


@pytest.mark.parametrize("t,hq,hkv,d", [(64, 32, 8, 128), (700, 40, 40, 64), (5000, 32, 8, 128), (2500, 71, 1, 64), (9000, 4, 4, 256),
                                        (20000, 3, 1, 32), (2, 300, 200, 32)])
def test_sizes(tl, t, hq, hkv, d):
    """One head a thread to several, more heads than a workgroup's rows, tokens that fill no workgroup."""
    check(tl, t, hq, hkv, d, seed=t, extra=hkv * d)


@pytest.mark.parametrize("axis_of", [[0] * 16 + [1] * 24 + [2] * 24, [i % 3 for i in range(64)], [7] * 64, [1] * 32 + [0] * 32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(tl, axis_of, interleaved):
    check(tl, 50, 4, 2, 128, axis_of=axis_of, interleaved=interleaved, seed=3)


def test_far_positions(tl):
    pos = np.array([[0, 1, -1, 2 ** 20, 2 ** 31 - 1, -2 ** 31, 1000000, 131072]], np.int32)
    check(tl, 8, 2, 2, 64, pos=pos, seed=4)
    check(tl, 8, 2, 2, 64, pos=pos, theta=1e7, interleaved=True, seed=4)


def test_given_frequencies(tl):
    check(tl, 20, 2, 1, 64, inv_freq=[1.0 / (1 + i) for i in range(32)], seed=5)
    check(tl, 20, 2, 1, 64, inv_freq=[0.0] * 31 + [100.0], seed=6)


def test_in_place(tl):
    check(tl, 33, 8, 2, 128, in_place=True, seed=7)
    check(tl, 3000, 8, 2, 64, rd=32, in_place=True, interleaved=True, seed=8)


def test_position_zero_without_norm_copies(tl):
    x = torch.randn((5, 4, 64), device="cuda").half()
    x[0, 0, 0], x[1, 1, 63], x[2, 2, 40] = float("inf"), float("nan"), float("-inf")
    out = torch.empty_like(x)
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    tl.Rotary(64, 16).apply(x.data_ptr(), None, out.data_ptr(), None, pos.data_ptr(), 5, 4, 0)
    torch.cuda.synchronize()
    assert torch.equal(out[:, :, 16:].nan_to_num(nan=7.0), x[:, :, 16:].nan_to_num(nan=7.0))  # what is not rotated: as it is
    assert torch.equal(out[0, 1:], x[0, 1:])


def test_zero_rows(tl):
    """A row of zeros stays one, with eps and without (0 / 0 is NaN there, as the formula's)."""
    x = torch.zeros((2, 1, 64), dtype=torch.float16, device="cuda")
    w, pos, out = torch.ones(64, dtype=torch.float16, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda"), torch.ones_like(x)
    tl.Rotary(64).apply(x.data_ptr(), None, out.data_ptr(), None, pos.data_ptr(), 2, 1, 0, w.data_ptr(), eps=1e-6)
    torch.cuda.synchronize()
    assert not out.any()


def test_captured(tl):
    t, hq, hkv, d = 40, 8, 2, 128
    x, pos = torch.randn((t, (hq + hkv) * d), device="cuda").half(), torch.arange(t, dtype=torch.int32, device="cuda")
    outs = [[torch.zeros((t, h, d), dtype=torch.float16, device="cuda") for h in (hq, hkv)] for _ in range(2)]
    r = tl.Rotary(d)

    def call(o, s=0):
        r.apply(x.data_ptr(), x[:, hq * d:].data_ptr(), o[0].data_ptr(), o[1].data_ptr(), pos.data_ptr(), t, hq, hkv, eps=1e-5,
                q_stride=x.stride(0), k_stride=x.stride(0), stream=s)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(outs[0], torch.cuda.current_stream().cuda_stream)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        pos.add_(i)
        call(outs[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and a.any() for a, b in zip(*outs))
