"""Plain 64-bit forms of the cache in 8 bits and of attention over it, and the cache
that its GPU tests share."""
import numpy as np
import torch

from retention_ref import dev

GROUP = 32


def held(x):
    """What the cache stands for that was given x [S][hkv][d] (fp16), in 64 bits."""
    out = x.astype(np.float64)
    for g in range(len(x) // GROUP):
        for h in range(x.shape[1]):
            out[g * GROUP:(g + 1) * GROUP, h] = held_group(x[g * GROUP:(g + 1) * GROUP, h])
    return out


def held_group(x):
    if not np.isfinite(x).all():
        return np.full(x.shape, np.nan)
    a = np.abs(x.astype(np.float64)).max()
    if a == 0:
        return np.zeros(x.shape)
    m, e = np.frexp(a / 127.0)
    scale = np.ldexp(np.floor(m * 2048), e - 11)  # 11 significant bits
    return np.rint(x.astype(np.float64) / scale) * scale


class QuantCache:
    """A manager of a cache in 8 bits beside a host copy of what it was given:
    k[layer][i] / v[layer][i] are [tokens][hkv][d] fp16 arrays of sequence i."""

    def __init__(self, tl, lens, hkv, d, block=32, layers=1, seed=0, spare=0, hq=None, room=None, blocks=None):
        self.tl, self.hkv, self.d, self.layers, self.hq = tl, hkv, d, layers, hq or hkv
        self.rng = np.random.default_rng(seed)
        self.room, n = room or max(list(lens) + [1]) + 40, len(lens)
        self.mgr = tl.KVCacheManager(num_layers=layers, num_heads=hkv, head_dim=d, max_seq_len=self.room,
                                     max_batch_size=n + spare, block_tokens=block,
                                     num_blocks=blocks or (n + spare) * -(-self.room // block), quantized=True)
        self.ids = []
        for _ in range(n):
            sid, err = self.mgr.allocateSequence(self.room)
            assert err is None, err
            self.ids.append(sid)
        self.k = [[np.zeros((0, hkv, d), np.float16) for _ in lens] for _ in range(layers)]
        self.v = [[np.zeros((0, hkv, d), np.float16) for _ in lens] for _ in range(layers)]
        self.append(lens)

    def rows(self, n, std=1.0):
        return (self.rng.standard_normal((n, self.hkv, self.d)) * std).astype(np.float16)

    def new_rows(self, counts):
        """Rows for counts[i] tokens of every sequence: [layer] of (k, v) lists."""
        return [([self.rows(c) for c in counts], [self.rows(c) for c in counts]) for _ in range(self.layers)]

    def note(self, new, keep=None):
        for layer, (k, v) in enumerate(new):
            for i in range(len(k)):
                n = len(k[i]) if keep is None else keep
                self.k[layer][i] = np.concatenate([self.k[layer][i], k[i][:n]])
                self.v[layer][i] = np.concatenate([self.v[layer][i], v[i][:n]])

    def append(self, counts, how="prefill", new=None):
        """counts[i] tokens for sequence i, and the step is committed."""
        some = [i for i, c in enumerate(counts) if c]
        new = new or self.new_rows(counts)
        if not some:
            return
        if how == "prefill":
            b = self.tl.PrefillBatch(self.mgr, len(some), self.hq)
            b.prepare([self.ids[i] for i in some], [counts[i] for i in some])
        elif how == "step":
            assert set(counts) <= {0, 1}
            b = self.tl.DecodeBatch(self.mgr, len(some), self.hq)
            b.prepare([self.ids[i] for i in some])
        if how == "step":  # all layers in one call
            k, v = (dev(np.stack([np.concatenate([new[layer][w][i] for i in some]) for layer in range(self.layers)]))
                    for w in (0, 1))
            b.append(0, self.layers, k.data_ptr(), v.data_ptr())
            torch.cuda.synchronize()
        else:
            for layer, (ks, vs) in enumerate(new):
                k, v = dev(np.concatenate([ks[i] for i in some])), dev(np.concatenate([vs[i] for i in some]))
                if how == "prefill":
                    b.append(layer, k.data_ptr(), v.data_ptr())
                else:
                    at = 0
                    for i in some:
                        err = self.mgr.appendKV(self.ids[i], layer, k[at:].data_ptr(), v[at:].data_ptr(), counts[i])
                        assert err is None, err
                        at += counts[i]
                torch.cuda.synchronize()
        if how == "prefill":
            b.commit()
        elif how == "step":
            b.commit(1)
        else:
            for i in some:
                assert self.mgr.advanceSeqLen(self.ids[i], counts[i]) is None
        self.note(new)

    def read(self, layer=0, lens=None, s_max=None, which="kv"):
        """The cache read back: (k, v) [entry][hkv][s_max][d] on the host, with NaN where
        nothing was written."""
        lens = [len(x) for x in self.k[layer]] if lens is None else lens
        s_max = max(lens) if s_max is None else s_max
        out = [torch.full((len(lens) + 1, self.hkv, s_max, self.d), float("nan"), dtype=torch.float16, device="cuda")
               for _ in range(2)]
        b = self.tl.DecodeBatch(self.mgr, len(lens), self.hq)
        b.prepare_lengths(self.ids[:len(lens)], lens)
        b.gather(layer, out[0].data_ptr() if "k" in which else None, out[1].data_ptr() if "v" in which else None, s_max)
        torch.cuda.synchronize()
        assert all(torch.isnan(o[-1]).all() for o in out)  # rows behind the last entry
        return [o[:-1].cpu().numpy() for o in out]

    def expect(self, layer, i, n=None):
        """What the cache stands for after n tokens (None: all) of sequence i."""
        return held(self.k[layer][i][:n]), held(self.v[layer][i][:n])

    def check(self, lens=None):
        """Every layer, bit for bit."""
        for layer in range(self.layers):
            k, v = self.read(layer)
            for i in range(len(self.ids)):
                for got, want in zip((k[i], v[i]), self.expect(layer, i)):
                    n = len(want)
                    with np.errstate(over="ignore"):
                        want = want.astype(np.float16).transpose(1, 0, 2)
                    assert np.array_equal(got[:, :n], want, equal_nan=True), np.argwhere(got[:, :n] != want)[:5]
                    assert not got[:, n:].any()


def attend(q, k, v, scale, last):
    """q [T][hq][d] over the held k, v [S][hkv][d] in 64 bits, query j over the keys 0 ..
    last[j].  Returns (out, sum P |v|, error of a score [T][hq])."""
    t, hq, d = q.shape
    g = hq // k.shape[1]
    out, mass, err = np.zeros((t, hq, d)), np.zeros((t, hq, d)), np.zeros((t, hq))
    for h in range(hq):
        kh, vh, qh = k[:, h // g], v[:, h // g], q[:, h].astype(np.float64)
        s = qh @ kh.T * scale
        s[np.arange(len(k))[None, :] > np.asarray(last)[:, None]] = -np.inf
        # the fp32 sum of d products, its products with the two scales: (d + 6) roundings of the absolute sum
        err[:, h] = (np.abs(qh) @ np.abs(kh).T).max(axis=1) * abs(scale) * (d + 6) * 2.0 ** -24
        e = np.exp(s - s.max(axis=1, keepdims=True))
        p = e / e.sum(axis=1, keepdims=True)
        out[:, h], mass[:, h] = p @ vh, p @ np.abs(vh)
    return out, mass, err


def check_out(got, out, mass, err, terms, most):
    """Each weight is rounded to fp16 once (2^-11 of it; 2^-32 of the largest where it is
    below fp16's normal numbers), in the products and in their sum, and has the relative error
    of its score's (twice: the maximum's too); sums of `terms` fp32 numbers
    lose at most terms * 2^-24, the scaled sums of the groups as much again; the output is
    rounded to fp16 once.  most: the largest |value|."""
    rel = 2 * 2.0 ** -11 + 2 * err + (2 * terms + 8) * 2.0 ** -24
    tol = 2.0 ** -11 * np.abs(out) + rel[..., None] * mass * 1.01 + 1e-6 * np.abs(out) + 2.0 ** -24 + terms * 2.0 ** -32 * most
    bad = ~(np.abs(got.astype(np.float64) - out) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], np.nanmax(np.abs(got - out)), tol.min())
