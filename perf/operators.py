"""Attention that keeps account of a cache's tokens, eviction by that account,
and attention to cached states of another length, as measurable cases.

Every case is the call of one layer through the public binding tinyllm_kv, in
fp16, on a manager's slot pool or block pool.  A program prepares a step once
and makes this call for each of its layers, so the prepared batch belongs to
the state and the call alone is the pass:

  decode   DecodeBatch.decode_weights: append one token per sequence, attend,
           and add every cached token's attention weight (summed over the query
           heads of its kv head) to the running account, in fp32
  prompt   PrefillBatch.weights: the same account after a prompt, by its last
           `window` tokens or by all of them, causal
  evict    EvictBatch.run: keep the `budget` tokens per kv head that the account
           and the newest positions name, the rest of the cache moved into the
           rows that became free
  cross    CrossBatch.attention: the queries of several sequences over cached
           states (an encoder's), every query over all of them; several entries
           may read the same states

A pass leaves lengths and accounts as they were (no commit, separate outputs),
so it can be repeated on the same state and gives the same results.
"""
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tiny-llm_amd")

# Most cached bytes of a drawn case, and most operations: what the largest
# listed ones have.
_MOST_KV_BYTES = 2 << 30
_MOST_FLOPS = 5.5e11


def listed():
    return [
        # The smallest step: four short chats on a small MHA model (8 heads of 64).
        dict(name="decode_small_mha", kind="decode", batch=4, hq=8, hkv=8, d=64, dist="range",
             lo=128, hi=512, len_seed=1, block=0),
        # A full batch at long context on a Llama-3-8B-sized layer (32 / 8 heads of 128).
        dict(name="decode_gqa_b64_ctx8k", kind="decode", batch=64, hq=32, hkv=8, d=128,
             dist="range", lo=8192, hi=8192, len_seed=3, block=0),
        # Continuous batching: lognormal context lengths on a block pool, group 8.
        dict(name="decode_ragged_blocks_g8", kind="decode", batch=96, hq=64, hkv=8, d=128,
             dist="lognormal", lo=2048, hi=16384, len_seed=4, block=16),
        # The account after one long document, by its last 32 tokens.
        dict(name="prompt_window_8192", kind="prompt", seqs=1, hq=32, hkv=8, d=128, lo=8192, hi=8192,
             prefix_hi=0, window=32, len_seed=5, block=0),
        # The account after a burst of prompts, by all of their tokens.
        dict(name="prompt_whole_4x2048", kind="prompt", seqs=4, hq=32, hkv=8, d=128, lo=1700, hi=2048,
             prefix_hi=600, window=0, len_seed=6, block=16),
        # The steady state of a bounded cache: one token came, one goes, on a
        # cache that was evicted from before (32 heads of 128).
        dict(name="evict_one_of_1025", kind="evict", batch=16, hkv=32, d=128, lo=1500, hi=3000,
             budget=1024, recent=512, again=1, len_seed=7),
        # A burst of prompts cut down to a quarter.
        dict(name="evict_8x8192_to_2048", kind="evict", batch=8, hkv=8, d=128, lo=7000, hi=8192,
             budget=2048, recent=256, again=0, len_seed=8),
        # One long document cut down to an eighth.
        dict(name="evict_32768_to_4096", kind="evict", batch=1, hkv=8, d=128, lo=32768, hi=32768,
             budget=4096, recent=512, again=0, len_seed=9),
        # Beam search, five beams on each of four inputs: one token a beam over
        # the input's 1500 states (8 heads of 64).
        dict(name="cross_beams_one_token", kind="cross", entries=20, states=4, hq=8, hkv=8, d=64,
             q_lo=1, q_hi=1, lo=1500, hi=1500, trim=0, len_seed=10, block=0),
        # Decoder prompts of a batch over ragged, padded inputs.
        dict(name="cross_prompts_16x1500", kind="cross", entries=16, states=16, hq=16, hkv=16, d=64,
             q_lo=64, q_hi=448, lo=300, hi=1500, trim=1, len_seed=11, block=0),
        # Eight tokens checked against one very long input on a block pool.
        dict(name="cross_8_over_32768", kind="cross", entries=1, states=1, hq=32, hkv=8, d=128,
             q_lo=8, q_hi=8, lo=32768, hi=32768, trim=0, len_seed=12, block=16),
        # Long targets over long inputs: bound by the matrix rate.
        dict(name="cross_2x2048_over_8192", kind="cross", entries=2, states=2, hq=32, hkv=8, d=128,
             q_lo=2048, q_hi=2048, lo=8192, hi=8192, trim=0, len_seed=13, block=0),
    ]


def _log(rng, lo, hi):
    """An integer from lo..hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["decode"] * 4 + ["prompt"] * 3 + ["evict"] * 4 + ["cross"] * 5)
    while True:
        d = rng.choice([64, 128, 128, 128, 256, 32])
        hkv = rng.choice([1, 2, 4, 8, 8, 8, 32])
        hq = hkv * rng.choice([1, 2, 4, 4, 8] if hkv < 32 else [1, 2])
        c = dict(kind=kind, hkv=hkv, d=d, len_seed=rng.randrange(1 << 30))
        if kind != "evict":
            c.update(hq=hq, block=rng.choice([0, 0, 16, 16, 32, 64]))
        if kind == "decode":
            lo = _log(rng, 1, 16384)
            c.update(batch=_log(rng, 1, 256), dist=rng.choice(["range", "range", "lognormal"]), lo=lo)
            c["hi"] = min(32768, lo + _log(rng, 1, 8192)) if c["dist"] == "range" else 32768
        elif kind == "prompt":
            lo = _log(rng, 1, 8192)
            c.update(seqs=_log(rng, 1, 16), lo=lo, hi=min(8192, lo + _log(rng, 1, 1024)),
                     prefix_hi=rng.choice([0, 0, _log(rng, 16, 6144)]),
                     window=rng.choice([0, 0, 1, _log(rng, 2, 128), 32]))
        elif kind == "evict":
            lo = _log(rng, 8, 32768)
            c.update(batch=_log(rng, 1, 128), lo=lo, hi=min(32768, lo + _log(rng, 1, 4096)))
            c["budget"] = max(1, int(lo * rng.uniform(0.05, 1.1)))
            c["recent"] = rng.choice([0, c["budget"], _log(rng, 1, c["budget"]), c["budget"] // 2])
            c["again"] = rng.choice([0, 0, 1, 1, _log(rng, 1, 1024)])
        else:
            lo, q_lo = _log(rng, 1, 32768), rng.choice([1, _log(rng, 1, 2048)])
            entries = _log(rng, 1, 64)
            c.update(entries=entries, states=max(1, entries // rng.choice([1, 1, 2, 5])), q_lo=q_lo,
                     q_hi=rng.choice([q_lo, min(2048, 2 * q_lo)]), lo=lo,
                     hi=min(32768, lo + _log(rng, 1, 4096)), trim=rng.choice([0, 0, 1]))
        if _held(c) * c["hkv"] * c["d"] * 4 <= _MOST_KV_BYTES and work(c)["flops"] <= _MOST_FLOPS:
            return c


# --------------------------------------------------------------------------
# Shapes: properties of the case, not of the seed
# --------------------------------------------------------------------------
def _lengths(c):
    """Cached tokens of each sequence (prompt: new tokens; cross: states)."""
    n = c.get("batch") or c.get("seqs") or c.get("states")
    rng = np.random.default_rng(c["len_seed"])
    if c.get("dist") == "lognormal":  # median lo, sigma 1, at most hi
        x = np.exp(rng.normal(np.log(c["lo"]), 1.0, size=n))
        return [int(v) for v in np.clip(np.round(x), 1, c["hi"])]
    return [int(v) for v in rng.integers(c["lo"], c["hi"] + 1, size=n)]


def _prefixes(c):
    rng = np.random.default_rng(c["len_seed"] + 1)
    return [int(v) for v in rng.integers(0, c["prefix_hi"] + 1, size=c["seqs"])]


def _queries(c):
    """(queries, states' index, attended states) of each entry of a cross case."""
    rng = np.random.default_rng(c["len_seed"] + 2)
    s = _lengths(c)
    q = [int(v) for v in rng.integers(c["q_lo"], c["q_hi"] + 1, size=c["entries"])]
    src = [i * c["states"] // c["entries"] for i in range(c["entries"])]
    if c["trim"]:  # padded inputs; one that is all padding
        att = [int(rng.integers(max(1, s[j] // 2), s[j] + 1)) for j in src]
        att[-1] = 0
    else:
        att = [s[j] for j in src]
    return q, src, att


def _caps(c):
    """Tokens that each sequence has room for."""
    n = _lengths(c)
    if c["kind"] == "decode":
        return [x + 1 for x in n]
    if c["kind"] == "prompt":
        return [a + b for a, b in zip(n, _prefixes(c))]
    if c["kind"] == "evict":
        return [max(x, min(x, c["budget"]) + c["again"]) for x in n]
    return n


def _held(c):
    caps = _caps(c)
    return sum(caps) if c.get("block") else max(caps) * len(caps)


def _window(c, n):
    return min(n, c["window"]) if c["window"] else n


def work(c):
    kind, row = c["kind"], c["hkv"] * c["d"]
    if kind == "decode":
        s, q = sum(x + 1 for x in _lengths(c)), c["batch"] * c["hq"] * c["d"]
        # K and V, q and out, the new rows read and written, the account read and written
        return dict(bytes=4 * s * row + 4 * q + 8 * c["batch"] * row + 8 * s * c["hkv"], flops=4 * s * c["hq"] * c["d"])
    if kind == "prompt":
        nbytes = flops = 0
        for n, p in zip(_lengths(c), _prefixes(c)):
            w = _window(c, n)
            # K once, the window's queries, the account read where there was one, and written
            nbytes += 2 * (n + p) * row + 2 * w * c["hq"] * c["d"] + 4 * (n + 2 * p) * c["hkv"]
            flops += 2 * (w * (n - w + p) + w * (w + 1) // 2) * c["hq"] * c["d"]
        return dict(bytes=nbytes, flops=flops)
    if kind == "evict":
        nbytes = 0
        for x in _lengths(c):
            keep = min(x, c["budget"])
            n = keep + c["again"] if c["again"] else x
            keep = min(n, c["budget"])
            # the account and the positions, and the rows that have to move: of the
            # kept ones, those behind the budget, in the middle of what it can be
            moved = min(n - keep, keep) * keep // n
            nbytes += c["hkv"] * (8 * n + 8 * keep) + moved * row * 8
        return dict(bytes=nbytes, flops=0)
    q, src, att = _queries(c)
    seen = {j: max(a for i, a in zip(src, att) if i == j) for j in src}
    return dict(bytes=4 * sum(q) * c["hq"] * c["d"] + 4 * sum(seen.values()) * row,
                flops=4 * sum(a * b for a, b in zip(q, att)) * c["hq"] * c["d"])


# --------------------------------------------------------------------------
# Inputs, from the seed alone
# --------------------------------------------------------------------------
def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) * std


def _account(g, shape):
    """Running weights as decoding leaves them: most of the weight on few
    tokens, a long tail, and tokens that were never attended to."""
    u = torch.rand(shape, generator=g, device="cuda")
    return torch.where(u < 0.03, torch.zeros_like(u), 8 * u ** 6)


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    row, kind, lens = c["hkv"] * c["d"], c["kind"], _lengths(c)
    x = {}
    if kind == "decode":
        x["k"], x["v"] = (_normal(g, (sum(lens), row)) for _ in range(2))
        x["nk"], x["nv"] = (_normal(g, (len(lens), row)) for _ in range(2))
        x["q"] = _normal(g, (len(lens), c["hq"], c["d"]))
    elif kind == "prompt":
        new, old = sum(lens), sum(_prefixes(c))
        x["k"], x["v"] = (_normal(g, (old, row)) for _ in range(2))
        x["nk"], x["nv"] = (_normal(g, (new, row)) for _ in range(2))
        x["q"] = _normal(g, (new, c["hq"], c["d"]))
    elif kind == "evict":
        x["k"], x["v"] = (_normal(g, (sum(lens), row)) for _ in range(2))
        x["nk"], x["nv"] = (_normal(g, (len(lens) * c["again"], row)) for _ in range(2))
    else:
        x["k"], x["v"] = (_normal(g, (sum(lens), row)) for _ in range(2))
        x["q"] = _normal(g, (sum(_queries(c)[0]), c["hq"], c["d"]))
    if kind in ("decode", "prompt", "evict"):
        x["w"] = _account(g, (len(lens), c["hkv"], _room(c)))
    if kind == "evict":
        x["nw"] = _account(g, (len(lens), c["hkv"], c["again"]))
    return x


def _room(c):
    """Tokens that a sequence of the case's manager has room for at most."""
    m, b = max(_caps(c)), c.get("block")
    return -(-m // b) * b if b else m


# --------------------------------------------------------------------------
# State
# --------------------------------------------------------------------------
class _PoolArray:
    """A manager's pool as an array.  It holds the manager, and the tensor made
    of it holds it, so the pool lives as long as any tensor over it."""

    def __init__(self, mgr, shape):
        self.mgr = mgr
        self.__cuda_array_interface__ = dict(shape=shape, typestr="<f2", data=(mgr.pool(), False), version=2)


def _tl():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import tinyllm_kv
    return tinyllm_kv


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _append(mgr, ids, counts, hq, k, v):
    some = [(s, n) for s, n in zip(ids, counts) if n]
    if some:
        p = _tl().PrefillBatch(mgr, len(some), hq)
        p.prepare([s for s, _ in some], [n for _, n in some], _stream())
        p.append(0, k.data_ptr(), v.data_ptr(), _stream())
        p.commit()


def _manager(c, hq):
    """A manager with the case's sequences, sequence i in slot i, and its slot
    pool as an array ([slot][K | V][token][row])."""
    caps, room = _caps(c), _room(c)
    args = dict(num_layers=1, num_heads=c["hkv"], head_dim=c["d"], max_batch_size=len(caps), max_seq_len=room)
    if c.get("block"):
        args.update(block_tokens=c["block"], num_blocks=sum(-(-n // c["block"]) for n in caps))
    mgr = _tl().KVCacheManager(**args)
    ids = []
    for n in caps:
        sid, err = mgr.allocateSequence(n)
        assert err is None, err
        ids.append(sid)
    pool = None
    if not c.get("block"):
        shape = (len(caps), 2, room, c["hkv"] * c["d"])
        pool = torch.as_tensor(_PoolArray(mgr, shape), device="cuda")
    return mgr, ids, pool


def _fill(cache, at, counts, k, v):
    """Rows of k, v into the plain cache [sequence][K | V][token][row] from `at` on."""
    o = 0
    for i, (a, n) in enumerate(zip(at, counts)):
        cache[i, 0, a:a + n], cache[i, 1, a:a + n] = k[o:o + n], v[o:o + n]
        o += n


def prepare(c, seed):
    x, kind = _inputs(c, seed), c["kind"]
    hq, lens = c.get("hq", c["hkv"]), _lengths(c)
    zero = [0] * len(lens)
    st = dict(c=c, x=x, kind=kind, own=own)
    if own:
        tl = _tl()
        mgr, ids, st["pool"] = _manager(c, hq)
        st["mgr"] = mgr
    else:
        st["pool"] = torch.zeros((len(lens), 2, _room(c), c["hkv"] * c["d"]), dtype=torch.float16, device="cuda")
    if kind in ("decode", "prompt", "evict"):
        st["w_out"] = torch.zeros_like(x["w"])
    if "q" in x:
        st["out"] = torch.empty_like(x["q"])
    k, v = x.pop("k"), x.pop("v")
    if kind == "decode":
        if own:
            _append(mgr, ids, lens, hq, k, v)
            st["batch"] = tl.DecodeBatch(mgr, len(lens), hq)
            st["batch"].prepare(ids, _stream())
        else:
            _fill(st["pool"], zero, lens, k, v)
    elif kind == "prompt":
        pre = _prefixes(c)
        if own:
            _append(mgr, ids, pre, hq, k, v)
            st["batch"] = tl.PrefillBatch(mgr, len(lens), hq)
            st["batch"].prepare(ids, lens, _stream())
            st["batch"].append(0, x["nk"].data_ptr(), x["nv"].data_ptr(), _stream())
        else:
            _fill(st["pool"], zero, pre, k, v)
            _fill(st["pool"], pre, lens, x["nk"], x["nv"])
    elif kind == "evict":
        st["pos"] = torch.zeros(x["w"].shape, dtype=torch.int32, device="cuda")
        st["pos_out"] = torch.zeros_like(st["pos"])
        kept = [min(n, c["budget"]) for n in lens]
        if own:
            _append(mgr, ids, lens, hq, k, v)
        else:
            _fill(st["pool"], zero, lens, k, v)
            st["len"], st["base"], st["gone"] = list(lens), list(zero), list(zero)
        if c["again"]:  # an earlier eviction, then `again` more tokens
            if own:
                ev = tl.EvictBatch(mgr, len(lens))
                ev.prepare(ids, [c["budget"]] * len(lens), c["recent"], _stream())
                ev.run(0, x["w"].data_ptr(), x["w"].data_ptr(), st["pos"].data_ptr(), st["pos"].data_ptr(), _stream())
                ev.commit()
                _append(mgr, ids, [c["again"]] * len(lens), hq, x["nk"], x["nv"])
            else:
                _evict(st, x["w"], x["w"], st["pos"], st["pos"])
                st["gone"], st["base"] = [n - m for n, m in zip(lens, kept)], list(kept)
                st["len"] = [m + c["again"] for m in kept]
                _fill(st["pool"], kept, [c["again"]] * len(lens), x["nk"], x["nv"])
            for i, m in enumerate(kept):
                x["w"][i, :, m:m + c["again"]] = x["nw"][i]
        if own:
            st["batch"] = tl.EvictBatch(mgr, len(lens))
            st["batch"].prepare(ids, [c["budget"]] * len(lens), c["recent"], _stream())
    else:
        q, src, att = _queries(c)
        if own:
            _append(mgr, ids, lens, hq, k, v)
            st["batch"] = tl.CrossBatch(mgr, len(q), hq)
            st["batch"].prepare([ids[j] for j in src], q, att, _stream())
        else:
            _fill(st["pool"], zero, lens, k, v)
    return st


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(st):
    return _run_own(st) if st["own"] else _run_plain(st)


def _run_own(st):
    c, x, kind, s, b = st["c"], st["x"], st["kind"], _stream(), st["batch"]
    scale = c["d"] ** -0.5
    if kind == "decode":
        b.decode_weights(0, x["q"].data_ptr(), x["nk"].data_ptr(), x["nv"].data_ptr(), st["out"].data_ptr(), scale,
                         x["w"].data_ptr(), st["w_out"].data_ptr(), s)
        return (st["out"], st["w_out"]) + (() if c["block"] else (st["pool"],))
    if kind == "prompt":
        b.weights(0, x["q"].data_ptr(), scale, c["window"], x["w"].data_ptr(), st["w_out"].data_ptr(), s)
        return st["w_out"]
    if kind == "evict":
        b.run(0, x["w"].data_ptr(), st["w_out"].data_ptr(), st["pos"].data_ptr(), st["pos_out"].data_ptr(), s)
        return st["w_out"], st["pos_out"], st["pool"]
    b.attention(0, x["q"].data_ptr(), st["out"].data_ptr(), scale, s)
    return st["out"]


def _heads(c, rows):
    """Cache rows [S][hkv * d] as [hkv][S][d] in 32 bits."""
    return rows.view(rows.shape[0], c["hkv"], c["d"]).transpose(0, 1).float().contiguous()


def _softmax(c, q, k, last=None):
    """Weights of q [T][hq][d] over the cache rows k [S][hkv * d]: [hkv][T * group][S].
    last: the last attended key of each query, or None."""
    t, g = q.shape[0], c["hq"] // c["hkv"]
    qh = q.view(t, c["hkv"], g, c["d"]).transpose(0, 1).reshape(c["hkv"], t * g, c["d"]).float()
    s = torch.bmm(qh, _heads(c, k).transpose(1, 2).contiguous()).mul_(c["d"] ** -0.5)
    if last is not None:
        hidden = torch.arange(k.shape[0], device="cuda")[None, :] > last.repeat_interleave(g)[:, None]
        s.masked_fill_(hidden, float("-inf"))
    e = s.sub_(s.amax(dim=2, keepdim=True)).exp_()
    return e.div_(e.sum(dim=2, keepdim=True))


def _values(c, p, v, t):
    """p [hkv][T * group][S] times the cache rows v, as [T][hq][d]."""
    o = torch.bmm(p, _heads(c, v)).view(c["hkv"], t, -1, c["d"])
    return o.transpose(0, 1).reshape(t, c["hq"], c["d"])


def _run_plain(st):
    c, x, kind, cache = st["c"], st["x"], st["kind"], st["pool"]
    if kind == "decode":
        for i, n in enumerate(_lengths(c)):
            cache[i, 0, n], cache[i, 1, n] = x["nk"][i], x["nv"][i]
            p = _softmax(c, x["q"][i:i + 1], cache[i, 0, :n + 1])
            st["out"][i:i + 1] = _values(c, p, cache[i, 1, :n + 1], 1)
            w = p.sum(dim=1)
            w[:, :n] += x["w"][i, :, :n]
            st["w_out"][i, :, :n + 1] = w
        return (st["out"], st["w_out"]) + (() if c["block"] else (cache,))
    if kind == "prompt":
        at = 0
        for i, (n, p0) in enumerate(zip(_lengths(c), _prefixes(c))):
            w = _window(c, n)
            last = p0 + torch.arange(n - w, n, device="cuda")
            acc = _softmax(c, x["q"][at + n - w:at + n], cache[i, 0, :p0 + n], last).sum(dim=1)
            acc[:, :p0] += x["w"][i, :, :p0]
            st["w_out"][i, :, :p0 + n] = acc
            at += n
        return st["w_out"]
    if kind == "evict":
        _evict(st, x["w"], st["w_out"], st["pos"], st["pos_out"])
        return st["w_out"], st["pos_out"], cache
    at = 0
    for n, j, a in zip(*_queries(c)):
        if a:
            st["out"][at:at + n] = _values(c, _softmax(c, x["q"][at:at + n], cache[j, 0, :a]), cache[j, 1, :a], n)
        else:
            st["out"][at:at + n] = 0
        at += n
    return st["out"]


def _evict(st, w_in, w_out, pos_in, pos_out):
    c, cache = st["c"], st["pool"]
    for i, (n, base, gone) in enumerate(zip(st["len"], st["base"], st["gone"])):
        keep = min(n, c["budget"])
        t = torch.arange(n, device="cuda", dtype=torch.int32)
        pos = torch.where(t < base, pos_in[i, :, :n], t + gone)
        rank = torch.where(pos >= n + gone - c["recent"], torch.full_like(w_in[i, :, :n], float("inf")),
                           w_in[i, :, :n])
        order = rank.sort(dim=1, descending=True, stable=True).indices  # ties: the lower index first
        kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(1, order[:, :keep], True)
        # the i-th row that became free takes the i-th kept row behind the budget
        movers = (~kept[:, keep:]).to(torch.uint8).sort(dim=1, stable=True).indices + keep
        free = (~kept[:, :keep]).cumsum(dim=1) - 1
        src = t[None, :keep].long().expand(c["hkv"], keep)
        if n > keep:
            src = torch.where(kept[:, :keep], src, movers.gather(1, free.clamp(0, n - keep - 1)))
        w, p = w_in[i, :, :n].gather(1, src), pos.gather(1, src)
        w_out[i, :, :keep], pos_out[i, :, :keep] = w, p
        rows = cache[i, :, :n].view(2, n, c["hkv"], c["d"])
        rows[:, :keep] = rows.gather(1, src.t()[None, :, :, None].expand(2, keep, c["hkv"], c["d"]))


# --------------------------------------------------------------------------
# The same in 64 bits
# --------------------------------------------------------------------------
def _attend64(q, k, v, scale, first=None):
    """(weights summed over queries [S], attention [T][d]) of one head's q [T][d]
    over k, v [S][d]; first: query j attends keys 0 .. first + j, None: all."""
    total = torch.zeros(k.shape[0], dtype=torch.float64, device="cuda")
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    kt, vd = k.double().t().contiguous(), v.double() if v is not None else None
    step = max(1, (1 << 27) // max(1, k.shape[0]))
    for a in range(0, q.shape[0], step):
        s = q[a:a + step].double() @ kt * scale
        if first is not None:
            s += torch.full_like(s, float("-inf")).triu(first + a + 1)
        p = torch.softmax(s, dim=1)
        total += p.sum(dim=0)
        if v is not None:
            out[a:a + step] = p @ vd
    return total, out


def _blocks(counts):
    ends = np.cumsum(counts)
    return [slice(int(e - n), int(e)) for e, n in zip(ends, counts)]


def exact(c, seed):
    x, kind = _inputs(c, seed), c["kind"]
    lens, g = _lengths(c), c.get("hq", c["hkv"]) // c["hkv"]
    scale, d = c["d"] ** -0.5, c["d"]
    col = [slice(h * d, h * d + d) for h in range(c["hkv"])]
    pool = None
    if not c.get("block") and kind in ("decode", "evict"):
        pool = torch.zeros((len(lens), 2, _room(c), c["hkv"] * d), dtype=torch.float16, device="cuda")
    if kind == "evict":
        return _exact_evict(c, x, pool)
    if kind == "cross":
        out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
        q, src, att = _queries(c)
        states = _blocks(lens)
        for rows, j, a in zip(_blocks(q), src, att):
            for h in range(c["hq"] if a else 0):
                k, v = (x[n][states[j]][:a, col[h // g]] for n in ("k", "v"))
                out[rows, h] = _attend64(x["q"][rows, h], k, v, scale)[1]
        return out
    w_out = torch.zeros(x["w"].shape, dtype=torch.float64, device="cuda")
    if kind == "decode":
        out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
        for i, (rows, n) in enumerate(zip(_blocks(lens), lens)):
            k, v = (torch.cat([x[m][rows], x["n" + m][i:i + 1]]) for m in ("k", "v"))
            if pool is not None:
                pool[i, 0, :n + 1], pool[i, 1, :n + 1] = k, v
            w_out[i, :, :n] = x["w"][i, :, :n].double()
            for h in range(c["hkv"]):
                hs = slice(h * g, h * g + g)
                w, out[i, hs] = _attend64(x["q"][i, hs], k[:, col[h]], v[:, col[h]], scale)
                w_out[i, h, :n + 1] += w
        return (out, w_out) + (() if pool is None else (pool,))
    pre = _prefixes(c)
    for i, (new, old, n, p0) in enumerate(zip(_blocks(lens), _blocks(pre), lens, pre)):
        k, w = torch.cat([x["k"][old], x["nk"][new]]), _window(c, n)
        w_out[i, :, :p0] = x["w"][i, :, :p0].double()
        for h in range(c["hq"]):
            q = x["q"][new][n - w:, h]
            w_out[i, h // g, :p0 + n] += _attend64(q, k[:, col[h // g]], None, scale, p0 + n - w)[0]
    return w_out


def _exact_evict(c, x, pool):
    """Row by row: the kept tokens by sorting (account, index) pairs on the host."""
    d, lens = c["d"], _lengths(c)
    acc = x["w"].cpu().numpy().astype(np.float64)
    w_out, pos_out = np.zeros_like(acc), np.zeros(acc.shape, dtype=np.int32)
    new = x["nw"].cpu().numpy()
    for i, (rows, n) in enumerate(zip(_blocks(lens), lens)):
        pool[i, 0, :n], pool[i, 1, :n] = x["k"][rows], x["v"][rows]
        rounds = [n, min(n, c["budget"]) + c["again"]] if c["again"] else [n]
        pos = [np.arange(n) for _ in range(c["hkv"])]
        for r, size in enumerate(rounds):
            keep, seen = min(size, c["budget"]), n + (c["again"] if r else 0)
            if r:
                at = size - c["again"]
                pool[i, :, at:size] = torch.stack([x[m][i * c["again"]:(i + 1) * c["again"]] for m in ("nk", "nv")])
                acc[i, :, at:size] = new[i]
            for h in range(c["hkv"]):
                if r:
                    pos[h] = np.concatenate([pos[h], np.arange(n, seen)])
                w = acc[i, h, :size].copy()
                w[pos[h] >= seen - c["recent"]] = np.inf
                best = np.lexsort((np.arange(size), -w))[:keep]
                moved = np.sort(best[best >= keep])
                free = np.setdiff1d(np.arange(keep), best)
                acc[i, h, free], pos[h][free] = acc[i, h, moved], pos[h][moved]
                pos[h] = pos[h][:keep]
                to, frm = torch.from_numpy(free).cuda(), torch.from_numpy(moved).cuda()
                cols = slice(h * d, h * d + d)
                pool[i, :, to, cols] = pool[i, :, frm, cols]
        for h in range(c["hkv"]):
            w_out[i, h, :keep], pos_out[i, h, :keep] = acc[i, h, :keep], pos[h]
    return torch.from_numpy(w_out).cuda(), torch.from_numpy(pos_out).cuda(), pool
