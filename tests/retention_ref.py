"""Plain 64-bit forms of the cache accounts, the eviction and attention to cached
states, and the buffers that their GPU tests share."""
import numpy as np
import torch


class Cache:
    """A manager of one or more layers beside a host copy of what it holds:
    k[layer][i] / v[layer][i] are [tokens][hkv][d] fp16 arrays of sequence i.  The
    pool starts as NaN, so a read of what was never appended shows."""

    def __init__(self, tl, lens, hkv, d, room=None, block=0, layers=1, seed=0, spare=0, hq=None, blocks=None):
        self.tl, self.hkv, self.d, self.layers, self.hq = tl, hkv, d, layers, hq or hkv
        self.rng = np.random.default_rng(seed)
        room = room or max(lens) + 8
        if block:
            room = -(-room // block) * block
        self.room, n = room, len(lens)
        args = dict(num_layers=layers, num_heads=hkv, head_dim=d, max_seq_len=room, max_batch_size=n + spare)
        if block:
            args.update(block_tokens=block, num_blocks=blocks or (n + spare) * (room // block))
        self.mgr = tl.KVCacheManager(**args)
        total = 2 * self.mgr.getTotalMemory() // 2
        extra = self.mgr.blockBytes() if block else 0
        pool = _Raw(self.mgr, (total + extra) // 2)
        torch.as_tensor(pool, device="cuda").fill_(float("nan"))
        self.ids = []
        for _ in range(n):
            sid, err = self.mgr.allocateSequence(room)
            assert err is None, err
            self.ids.append(sid)
        self.slot = [self.mgr.slot_of(s) for s in self.ids]
        self.k = [[np.zeros((0, hkv, d), np.float16) for _ in lens] for _ in range(layers)]
        self.v = [[np.zeros((0, hkv, d), np.float16) for _ in lens] for _ in range(layers)]
        self.append(lens)

    def rows(self, n, std=1.0):
        return (self.rng.standard_normal((n, self.hkv, self.d)) * std).astype(np.float16)

    def append(self, counts):
        some = [(i, c) for i, c in enumerate(counts) if c]
        if not some:
            return
        p = self.tl.PrefillBatch(self.mgr, len(some), self.hq)
        p.prepare([self.ids[i] for i, _ in some], [c for _, c in some])
        for layer in range(self.layers):
            new = [(self.rows(c), self.rows(c)) for _, c in some]
            for (i, _), (k, v) in zip(some, new):
                self.k[layer][i] = np.concatenate([self.k[layer][i], k])
                self.v[layer][i] = np.concatenate([self.v[layer][i], v])
            dk, dv = dev(np.concatenate([k for k, _ in new])), dev(np.concatenate([v for _, v in new]))
            p.append(layer, dk.data_ptr(), dv.data_ptr())
            torch.cuda.synchronize()
        p.commit()

    def account(self, fill=0.0, dtype=torch.float32):
        n = self.mgr.getConfig().max_batch_size
        return torch.full((n, self.hkv, self.room), fill, dtype=dtype, device="cuda")

    def held(self, layer, i, n):
        """The first n cached K and V rows of sequence i, from the device."""
        out = [torch.full((1, self.hkv, n, self.d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]
        b = self.tl.DecodeBatch(self.mgr, 1, self.hkv)
        b.prepare_lengths([self.ids[i]], [n])
        b.gather(layer, out[0].data_ptr(), out[1].data_ptr(), n)
        torch.cuda.synchronize()
        return [o[0].transpose(0, 1).contiguous().cpu().numpy() for o in out]


class _Raw:
    def __init__(self, mgr, n):
        self.mgr = mgr
        self.__cuda_array_interface__ = dict(shape=(n,), typestr="<f2", data=(mgr.pool(), False), version=2)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def attend(q, k, v, scale, last=None):
    """q [T][hq][d] over k, v [S][hkv][d] in 64 bits; query j attends to the keys
    0 .. last[j] (None: all).  Returns (out [T][hq][d], bound of |out| terms
    [T][hq][d] = sum P |v|, weights [hq][T][S], error of a score [T][hq])."""
    t, hq, d = q.shape
    s_len, hkv, _ = k.shape
    g = hq // hkv
    q64, k64, v64 = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    out, mass = np.zeros((t, hq, d)), np.zeros((t, hq, d))
    w, err = np.zeros((hq, t, s_len)), np.zeros((t, hq))
    for h in range(hq):
        kh, vh = k64[:, h // g], v64[:, h // g]
        s = q64[:, h] @ kh.T * scale
        # |fp32 score - exact| <= (d + 4) roundings of the sum of absolute products
        err[:, h] = (np.abs(q64[:, h]) @ np.abs(kh).T).max(axis=1, initial=0) * abs(scale) * (d + 4) * 2.0 ** -24
        if last is not None:
            s[np.arange(s_len)[None, :] > np.asarray(last)[:, None]] = -np.inf
        if s_len:
            e = np.exp(s - s.max(axis=1, keepdims=True))
            p = e / e.sum(axis=1, keepdims=True)
            w[h] = p
            out[:, h], mass[:, h] = p @ vh, p @ np.abs(vh)
    return out, mass, w, err


def check_out(got, out, mass, err, terms):
    """Each weight is rounded to fp16 once (half a step, 2^-11 of it) and has the
    relative error of its score's (twice: the maximum's too); the sums of `terms`
    fp32 numbers lose at most terms * 2^-24; the output is rounded to fp16 once."""
    rel = 2.0 ** -11 + 2 * err + (terms + 8) * 2.0 ** -23
    tol = 2.0 ** -11 * np.abs(out) + rel[..., None] * mass * 1.01 + 1e-6 * np.abs(out) + 2.0 ** -24
    bad = ~(np.abs(got.astype(np.float64) - out) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - out).max(), tol.min())


def check_account(got, want, w, err, rows, s_len, before=None):
    """got, want [hkv][S]; w [hq][T][S] the added weights.  A weight has the
    relative error of its score (twice), of exp2 and the products (8 roundings) and of its
    row's sum of s_len terms; the account is a sum of `rows` weights."""
    hkv = got.shape[0]
    e = err.T[:, :, None] * w
    added = w.reshape(hkv, rows, s_len).sum(axis=1)
    tol = 2 * e.reshape(hkv, rows, s_len).sum(axis=1) + added * (s_len + rows + 12) * 2.0 ** -23
    if before is not None:
        tol = tol + np.abs(before) * 2.0 ** -23
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol * 1.01 + 1e-30)
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want).max())


def evict(w, pos, keep, newest):
    """One kv head: the source index of each of the first `keep` places."""
    n = len(w)
    rank = sorted(range(n), key=lambda t: (pos[t] < newest, np.isnan(w[t]) if pos[t] < newest else False,
                                           -w[t] if pos[t] < newest and not np.isnan(w[t]) else 0.0, t))
    kept = sorted(rank[:keep])
    movers = [t for t in kept if t >= keep]
    stay = {t for t in kept if t < keep}
    src, m = [], iter(movers)
    for t in range(keep):
        src.append(t if t in stay else next(m))
    return src


def even_tail(tl, n, d, block=0):
    """A cache whose every 64th token has a weight 2^25 times the others', which have
    values of 1000 and it of 0, the query that sees it so (at a scale of 1) and what
    attention gives: most of the output is from weights that one fp16 cannot hold
    beside a largest one of 1."""
    c = Cache(tl, [0], 1, d, room=n, block=block)
    k, v = np.zeros((n, 1, d), np.float16), np.full((n, 1, d), 1000.0, np.float16)
    k[::64, 0, 0], v[::64] = 4.34375, 0.0
    parts = iter([k, v])
    c.rows = lambda m, std=1.0: next(parts)
    c.append([n])
    q = np.zeros(d, np.float16)
    q[0] = 4.0
    heavy = len(k[::64])
    light = (n - heavy) * np.exp(-4.0 * 4.34375)
    want = 1000.0 * light / (heavy + light)
    # A weight's rounding to fp16, where the largest is 2^7 at least: half a step of
    # 2^-24 / 2^7, (n - heavy) / heavy of them per largest one, times 1000; the
    # output's rounding; scores of 17.4 with d + 4 roundings, and sums of n terms.
    tol = 1000.0 * (n - heavy) / heavy * 2.0 ** -32 + want * (2.0 ** -11 + (17.4 * (d + 4) + n) * 2.0 ** -23) + 2.0 ** -25
    return c, q, want, tol
