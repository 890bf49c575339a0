"""Sequences in which every token decides an output of its own kind: tokens come in
d classes, a query of one class has the score FAR above all others' with the tokens of its class, and
its output is the mean of their values.  A token that takes part twice, or not at all, moves it by
1 / (tokens of the class); that is far more than the bound on the rounding."""
import numpy as np

FAR = 60.0           # the weight of the other classes: exp(-60) of a token's
ONE = 127.0 / 128.0  # as a group's largest magnitude: its scale is 2^-7, and multiples of it are held as they are


def rows(t0, n, hkv, d, seed):
    """Keys, values [n][hkv][d] fp16 and classes [n][hkv] of the tokens from t0 on, the same whatever
    pieces they come in."""
    t = np.arange(t0, t0 + n)[:, None] + np.zeros((1, hkv), np.int64)
    h = np.arange(hkv)[None, :]
    cls = mix(t * 64 + h, seed) % d
    k = np.zeros((n, hkv, d), np.float16)
    np.put_along_axis(k, cls[..., None].astype(np.int64), np.float16(ONE), axis=2)
    steps = (mix((t * 64 + h)[..., None] * 256 + np.arange(d), seed + 1) % 255).astype(np.int64) - 127
    v = (steps / 128.0).astype(np.float16)
    v[..., 0] = ONE
    return k, v, cls


def mix(x, seed):
    """A 64-bit mixing of whole numbers: multiplications and shifts."""
    x = (np.asarray(x, dtype=np.uint64) + np.uint64(seed + 1)) * np.uint64(0x9E3779B97F4A7C15)
    for s, m in ((30, 0xBF58476D1CE4E5B9), (27, 0x94D049BB133111EB)):
        x = (x ^ (x >> np.uint64(s))) * np.uint64(m)
    return (x ^ (x >> np.uint64(31))) >> np.uint64(1)


def queries(cls, d, scale):
    """cls [...] -> rows [..., d] fp16 whose score with a key of their class is FAR."""
    q = np.zeros(cls.shape + (d,), np.float16)
    np.put_along_axis(q, cls[..., None].astype(np.int64), np.float16(FAR / scale / ONE), axis=-1)
    return q


def expect(v, cls, d, last, qcls):
    """Mean values of the tokens 0 .. last[j] of class qcls[j] of one kv head, and their number."""
    out, count = np.zeros((len(qcls), d)), np.zeros(len(qcls), np.int64)
    for j, (n, c) in enumerate(zip(last, qcls)):
        own = cls[:n + 1] == c
        count[j] = own.sum()
        if count[j]:
            out[j] = v[:n + 1][own].astype(np.float64).mean(0)
    return out, count


def tolerance(out, tokens):
    """Equal scores have equal weights, and equal ones rounded, in the products and in their sums.  What is left:
    a group's product of 64 addends at most (a weight may come in two halves), each group and each
    chunk or wave added (fewer than groups) in fp32, magnitudes up to 1; the 22 bits of a weight, twice; the
    reciprocal of the sum (with its 1e-6, the sum being 2^7 at least) and the last product; the output."""
    rel = (64 + 2 * (tokens / 32 + 1) + 16) * 2.0 ** -24 + 2 * 2.0 ** -22 + 1e-6 / 128 + 4 * 2.0 ** -24
    return 2.0 ** -11 * np.abs(out) + rel + 2.0 ** -25
