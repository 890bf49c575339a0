"""A cache held in 8 bits, attention over it, and the step that makes queries and
keys ready for it, as measurable cases.

A group of 32 tokens of one kv head has one scale per K and V: the largest
magnitude / 127, cut down to 11 significant bits, and whole numbers of -127..127
by round-half-even of x / scale.  A sequence's last group stays in fp16 until it has
its 32 tokens, so a value is rounded once, from what the program gave.  Every
case is the call of one layer through the public binding tinyllm_kv; a program
prepares a step once and makes the call for each of its layers, so the prepared
batch belongs to the state and the call alone is the pass:

  write    DecodeBatch.append (one token per sequence) or PrefillBatch.append, then
           DecodeBatch.gather: the new tokens into the cache, and all of it read back
           in fp16, [sequence][kv head][token][head_dim]
  decode   DecodeBatch.decode: append one token per sequence and attend
  prefill  PrefillBatch.run: append several tokens per sequence and attend causally
  rotate   Rotary.apply: RMS norm of every query and key head, then the rotation by
           position, along one axis or several

A pass leaves lengths as they were (no commit), so it can be repeated on the same
state and gives the same results.
"""
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tiny-llm_amd")

_GROUP = 32  # tokens that share a scale

# Most cached values of a drawn case, of rotated values, and operations: what the
# largest listed ones have.
_MOST_VALUES = 1.1e9
_MOST_ROTATED = 5e7
_MOST_FLOPS = 5.6e11


def listed():
    return [
        # The smallest step: four young chats on a small MHA model (8 heads of 64).
        dict(name="write_step_young_chats", kind="write", seqs=4, hq=8, hkv=8, d=64, block=32,
             dist="range", lo=20, hi=60, new_lo=1, new_hi=1, len_seed=1),
        # A burst of prompts that continue cached ones.
        dict(name="write_prompts_8x2048", kind="write", seqs=8, hq=32, hkv=8, d=128, block=128,
             dist="range", lo=0, hi=600, new_lo=1500, new_hi=2048, len_seed=2),
        # One long document, cached and lent out again.
        dict(name="write_document_32768", kind="write", seqs=1, hq=32, hkv=8, d=128, block=256,
             dist="range", lo=0, hi=0, new_lo=32768, new_hi=32768, len_seed=3),
        # A small decode step, where latency is what counts.
        dict(name="decode_small_mha", kind="decode", seqs=4, hq=8, hkv=8, d=64, block=64,
             dist="range", lo=128, hi=512, new_lo=1, new_hi=1, len_seed=4),
        # A full batch at long context on a Llama-3-8B-sized layer (32 / 8 heads of 128).
        dict(name="decode_gqa_b64_ctx8k", kind="decode", seqs=64, hq=32, hkv=8, d=128, block=128,
             dist="range", lo=8192, hi=8192, new_lo=1, new_hi=1, len_seed=5),
        # Continuous batching: lognormal context lengths, group 8.
        dict(name="decode_ragged_g8", kind="decode", seqs=96, hq=64, hkv=8, d=128, block=64,
             dist="lognormal", lo=2048, hi=16384, new_lo=1, new_hi=1, len_seed=6),
        # One conversation about a very long document.
        dict(name="decode_one_131072", kind="decode", seqs=1, hq=32, hkv=8, d=128, block=256,
             dist="range", lo=131071, hi=131071, new_lo=1, new_hi=1, len_seed=7),
        # Four drafted tokens per sequence checked in one step.
        dict(name="prefill_4_drafted_b32", kind="prefill", seqs=32, hq=32, hkv=8, d=128, block=128,
             dist="range", lo=1000, hi=6000, new_lo=4, new_hi=4, len_seed=8),
        # A long prompt into an empty cache: bound by the matrix rate.
        dict(name="prefill_prompt_8192", kind="prefill", seqs=1, hq=32, hkv=8, d=128, block=256,
             dist="range", lo=0, hi=0, new_lo=8192, new_hi=8192, len_seed=9),
        # Chunks of long prompts, each behind what is cached of it.
        dict(name="prefill_chunks_4x512", kind="prefill", seqs=4, hq=32, hkv=8, d=128, block=64,
             dist="range", lo=2500, hi=6000, new_lo=400, new_hi=512, len_seed=10),
        # Queries and keys of a decode step, out of the fused projection's rows.
        dict(name="rotate_step_b64", kind="rotate", tokens=64, hq=32, hkv=8, d=128, rd=128, pairs="halves",
             axes=1, norm=1, fused=1, far=100000),
        # A prompt with images: time, height and width.
        dict(name="rotate_images_8000", kind="rotate", tokens=8000, hq=32, hkv=8, d=128, rd=128, pairs="halves",
             axes=3, norm=1, fused=0, far=20000),
    ]


def _log(rng, lo, hi):
    """An integer from lo..hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["write"] * 4 + ["decode"] * 5 + ["prefill"] * 5 + ["rotate"] * 4)
    while True:
        d = rng.choice([64, 128, 128, 128, 256, 32])
        hkv = rng.choice([1, 2, 4, 8, 8, 8, 32])
        hq = hkv * rng.choice([1, 2, 4, 4, 8] if hkv < 32 else [1, 2])
        if kind == "rotate":
            c = dict(kind=kind, tokens=_log(rng, 1, 16384), hq=hq, hkv=hkv, d=d, rd=rng.choice([d, d, d, d // 2]),
                     pairs=rng.choice(["halves", "halves", "neighbours"]), axes=rng.choice([1, 1, 3, 2]),
                     norm=rng.choice([1, 1, 0]), fused=rng.choice([0, 1]), far=_log(rng, 64, 1000000))
            if c["tokens"] * (hq + hkv) * d <= _MOST_ROTATED:
                return c
            continue
        lo = rng.choice([0, _log(rng, 1, 32768), _log(rng, 1, 32768)])
        c = dict(kind=kind, seqs=_log(rng, 1, 128), hq=hq, hkv=hkv, d=d, block=rng.choice([32, 64, 128, 128, 256]),
                 dist="range", lo=lo, hi=lo + _log(rng, 1, 8192), len_seed=rng.randrange(1 << 30))
        if lo and rng.random() < 0.3:
            c.update(dist="lognormal", hi=32768)
        new = 1 if kind == "decode" or kind == "write" and rng.random() < 0.4 else _log(rng, 2, 4096)
        c.update(new_lo=new, new_hi=new if new == 1 else min(4096, new + rng.choice([0, _log(rng, 1, new)])))
        pre, cnt = _lengths(c)
        most = max(a + b for a, b in zip(pre, cnt))
        # (the plain form pads queries and keys to the longest sequence's)
        if (c["seqs"] * most * hkv * d * 2 <= _MOST_VALUES and work(c)["flops"] <= _MOST_FLOPS and
                (kind != "prefill" or c["seqs"] * hq * max(cnt) * most <= 2.2e9)):
            return c


# --------------------------------------------------------------------------
# Shapes: properties of the case, not of the seed
# --------------------------------------------------------------------------
def _lengths(c):
    """(cached tokens, new tokens) of each sequence."""
    rng = np.random.default_rng(c["len_seed"])
    if c["dist"] == "lognormal":  # median lo, sigma 1, at most hi
        pre = np.clip(np.round(np.exp(rng.normal(np.log(c["lo"]), 1.0, size=c["seqs"]))), 1, c["hi"])
    else:
        pre = rng.integers(c["lo"], c["hi"] + 1, size=c["seqs"])
    cnt = rng.integers(c["new_lo"], c["new_hi"] + 1, size=c["seqs"])
    return [int(v) for v in pre], [int(v) for v in cnt]


def _sections(c):
    """Axis of each pair of dimensions: a quarter of them by time, the rest by
    height and width in equal parts (two axes: half and half)."""
    n = c["rd"] // 2
    if c["axes"] == 1:
        return [0] * n
    first = n // 4 if c["axes"] == 3 else n // 2
    second = (n - first) // 2 if c["axes"] == 3 else n - first
    return [0] * first + [1] * second + [2] * (n - first - second)


def _held_bytes(tokens, c):
    """Bytes that `tokens` cached tokens of K and V take."""
    whole = tokens // _GROUP * _GROUP
    row = c["hkv"] * c["d"]
    return 2 * whole * row + whole // _GROUP * c["hkv"] * 8 + 4 * (tokens - whole) * row


def work(c):
    if c["kind"] == "rotate":
        n = c["tokens"] * (c["hq"] + c["hkv"]) * c["d"]
        return dict(bytes=4 * n + 4 * c["axes"] * c["tokens"], flops=(6 if c["norm"] else 3) * n)
    pre, cnt = _lengths(c)
    row = c["hkv"] * c["d"]
    nbytes = flops = 0
    for p, n in zip(pre, cnt):
        nbytes += 4 * n * row  # the new rows, read
        opened = p // _GROUP * _GROUP
        if c["kind"] == "write":
            # all that is cached, read or written, and given out in fp16; the open
            # group's first rows are read where it is closed
            nbytes += _held_bytes(p + n, c) + 4 * (p + n) * row + 4 * (p - opened) * row * (p + n >= opened + _GROUP)
        else:
            nbytes += _held_bytes(p + n, c) + 4 * n * c["hq"] * c["d"]
            flops += 4 * (n * p + n * (n + 1) // 2) * c["hq"] * c["d"]
    return dict(bytes=nbytes, flops=flops)


# --------------------------------------------------------------------------
# Inputs, from the seed alone
# --------------------------------------------------------------------------
def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) * std


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "rotate":
        return _rotate_inputs(c, g)
    pre, cnt = _lengths(c)
    row, x = c["hkv"] * c["d"], {}
    # Keys have channels that are larger than the others, in every token.
    loud = (torch.randn(row, generator=g, device="cuda") * 0.5).exp().half()
    for name, n in (("", sum(pre)), ("n", sum(cnt))):
        x[name + "k"], x[name + "v"] = _normal(g, (n, row)) * loud, _normal(g, (n, row))
    x["q"] = _normal(g, (sum(cnt), c["hq"], c["d"]))
    return x


def _rotate_inputs(c, g):
    t, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
    if c["fused"]:  # rows of the fused projection: queries, keys, values
        rows = _normal(g, (t, (hq + 2 * hkv) * d), 2.0)
        q, k = rows[:, :hq * d], rows[:, hq * d:(hq + hkv) * d]
    else:
        q, k = _normal(g, (t, hq * d), 2.0), _normal(g, (t, hkv * d), 2.0)
    x = dict(q=q, k=k)
    for n in ("qw", "kw"):
        x[n] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).half() if c["norm"] else None
    at = torch.randint(0, c["far"], (max(1, t // 1000 + 1),), generator=g, device="cuda", dtype=torch.int32)
    i = torch.arange(t, device="cuda", dtype=torch.int32)
    if c["axes"] == 1 and t <= 256:  # a step: sequences of any length
        pos = torch.randint(0, c["far"], (1, t), generator=g, device="cuda", dtype=torch.int32)
    elif c["axes"] == 1:
        pos = (at[0] + i)[None]
    else:  # pieces of 1000 tokens, each an image of 25 x 40 at its own time
        when = at[(i // 1000).long()]
        pos = torch.stack([when, when + i % 1000 // 40, when + i % 40])[:c["axes"]]
    x["pos"] = pos.contiguous()
    return x


# --------------------------------------------------------------------------
# State
# --------------------------------------------------------------------------
def _tl():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import tinyllm_kv
    return tinyllm_kv


def _stream():
    return torch.cuda.current_stream().cuda_stream


def prepare(c, seed):
    x = _inputs(c, seed)
    st = dict(c=c, x=x, own=own)
    if c["kind"] == "rotate":
        if own:
            st["rotary"] = _tl().Rotary(c["d"], rotary_dim=c["rd"], theta=10000.0, interleaved=c["pairs"] == "neighbours",
                                        axis_of=_sections(c))
            st["q_out"], st["k_out"] = (torch.empty((c["tokens"], c[h], c["d"]), dtype=torch.float16, device="cuda")
                                        for h in ("hq", "hkv"))
        return st
    pre, cnt = _lengths(c)
    ends = [p + n for p, n in zip(pre, cnt)]
    st["most"] = max(ends)
    k, v = x.pop("k"), x.pop("v")
    if own:
        _prepare_manager(st, pre, cnt, ends, k, v)
    else:
        _prepare_plain(st, pre, cnt, ends, k, v)
    return st


def _prepare_manager(st, pre, cnt, ends, k, v):
    c, x, tl = st["c"], st["x"], _tl()
    mgr = tl.KVCacheManager(num_layers=1, num_heads=c["hkv"], head_dim=c["d"], max_batch_size=len(pre),
                            max_seq_len=max(ends), block_tokens=c["block"],
                            num_blocks=sum(-(-n // c["block"]) for n in ends), quantized=True)
    ids = []
    for n in ends:
        sid, err = mgr.allocateSequence(n)
        assert err is None, err
        ids.append(sid)
    some = [(s, n) for s, n in zip(ids, pre) if n]
    if some:
        p = tl.PrefillBatch(mgr, len(some), c["hq"])
        p.prepare([s for s, _ in some], [n for _, n in some], _stream())
        p.append(0, k.data_ptr(), v.data_ptr(), _stream())
        p.commit()
    st["mgr"] = mgr
    step = c["new_hi"] == 1
    st["batch"] = (tl.DecodeBatch if step else tl.PrefillBatch)(mgr, len(ids), c["hq"])
    if step:
        st["batch"].prepare(ids, _stream())
    else:
        st["batch"].prepare(ids, cnt, _stream())
    if c["kind"] == "write":
        st["out"] = torch.empty((2, len(ids), c["hkv"], st["most"], c["d"]), dtype=torch.float16, device="cuda")
        st["reader"] = st["batch"]
        if not step:  # read what the append has left there, before it is committed
            st["batch"].append(0, x["nk"].data_ptr(), x["nv"].data_ptr(), _stream())
            st["reader"] = tl.DecodeBatch(mgr, len(ids), c["hq"])
            st["reader"].prepare_lengths(ids, ends, _stream())
    else:
        st["out"] = torch.empty_like(x["q"])


def _prepare_plain(st, pre, cnt, ends, k, v):
    """The cache [K | V][sequence][kv head][group][token][head_dim] of whole numbers
    and its scales, the open groups' rows, and the indices of a pass."""
    c = st["c"]
    n, groups = len(pre), -(-st["most"] // _GROUP)
    st["cache"] = torch.zeros((2, n, c["hkv"], groups, _GROUP, c["d"]), dtype=torch.int8, device="cuda")
    st["scale"] = torch.zeros((2, n, c["hkv"], groups), dtype=torch.float32, device="cuda")
    st["open"] = torch.zeros((2, n, _GROUP, c["hkv"], c["d"]), dtype=torch.float16, device="cuda")
    zero = [0] * n
    if sum(pre):
        _append(st, _indices(zero, pre), torch.stack([k, v]))
        st["open"] = st["opened"].permute(1, 0, 3, 2, 4).contiguous()
    st["at"] = _indices(pre, cnt)
    t = torch.arange(groups * _GROUP, device="cuda")
    st["hidden"] = t[None, :] >= torch.tensor(ends, device="cuda")[:, None]
    first, j = torch.tensor(pre, device="cuda"), torch.arange(max(cnt), device="cuda")
    st["causal"] = t[None, None, :] > torch.minimum(first[:, None] + j, torch.tensor(ends, device="cuda")[:, None] - 1)[..., None]
    starts = torch.tensor([0] + list(np.cumsum(cnt)[:-1]), device="cuda")
    real = j[None, :] < torch.tensor(cnt, device="cuda")[:, None]
    st["q_rows"] = torch.where(real, starts[:, None] + j, torch.zeros_like(starts)[:, None])
    st["q_real"] = real


def _indices(pre, cnt):
    """Where the rows of the groups that an append touches come from and go to."""
    n, starts = len(pre), np.cumsum([0] + list(cnt))
    held = [p % _GROUP for p in pre]
    wide = -(-max(h + m for h, m in zip(held, cnt)) // _GROUP)
    w = np.arange(wide * _GROUP)[None, :]
    h, m = np.array(held)[:, None], np.array(cnt)[:, None]
    rows = np.where(w < h, np.arange(n)[:, None] * _GROUP + np.minimum(w, _GROUP - 1), n * _GROUP + starts[:-1, None] + w - h)
    rows = np.where(w < h + m, rows, n * _GROUP + starts[-1])  # behind the end: zeros
    i, f = np.nonzero((np.arange(wide)[None, :] + 1) * _GROUP <= h + m)
    left = np.array([(a + b) % _GROUP > 0 for a, b in zip(pre, cnt)])
    put = lambda a: torch.as_tensor(np.ascontiguousarray(a), device="cuda")  # noqa: E731
    return dict(rows=put(rows), i=put(i), f=put(f), g=put(np.array(pre)[i] // _GROUP + f), wide=wide,
                last=put(np.minimum((h + m)[:, 0] // _GROUP, wide - 1)), all=put(np.arange(n)),
                left=put(np.nonzero(left)[0]), left_g=put(((np.array(pre) + np.array(cnt)) // _GROUP)[left]))


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(st):
    return _run_own(st) if st["own"] else _run_plain(st)


def _run_own(st):
    c, x, s = st["c"], st["x"], _stream()
    if c["kind"] == "rotate":
        st["rotary"].apply(x["q"].data_ptr(), x["k"].data_ptr(), st["q_out"].data_ptr(), st["k_out"].data_ptr(),
                           x["pos"].data_ptr(), c["tokens"], c["hq"], c["hkv"],
                           q_weight=x["qw"].data_ptr() if c["norm"] else None,
                           k_weight=x["kw"].data_ptr() if c["norm"] else None, eps=1e-5,
                           q_stride=x["q"].stride(0), k_stride=x["k"].stride(0), stream=s)
        return st["q_out"], st["k_out"]
    b, out, scale = st["batch"], st["out"], c["d"] ** -0.5
    if c["kind"] == "write":
        if c["new_hi"] == 1:
            b.append(0, 1, x["nk"].data_ptr(), x["nv"].data_ptr(), s)
        else:
            b.append(0, x["nk"].data_ptr(), x["nv"].data_ptr(), s)
        st["reader"].gather(0, out[0].data_ptr(), out[1].data_ptr(), st["most"], s)
        return out
    call = b.decode if c["kind"] == "decode" else b.run
    call(0, x["q"].data_ptr(), x["nk"].data_ptr(), x["nv"].data_ptr(), out.data_ptr(), scale, s)
    return out


def _quantised(x):
    """x [..., 32, d] as whole numbers and one scale per group.  In 64 bits: a
    quotient next to a half decides the number."""
    most = x.float().abs().amax(dim=(-2, -1))
    v = most / torch.full_like(most, 127)  # (by a number, torch multiplies with a rounded 1 / 127)
    scale = (v.view(torch.int32) & -8192).view(torch.float32)  # 11 significant bits
    by = torch.where(scale == 0, torch.ones_like(scale), scale).double()
    return (x.double() / by[..., None, None]).round().to(torch.int8), scale


def _append(st, at, new):
    """The rows new [K | V][token][row] into the cache; what is left of the open groups
    into st["opened"] [sequence][K | V][kv head][token][head_dim]."""
    c = st["c"]
    n, zero = st["open"].shape[1], torch.zeros((2, 1, c["hkv"], c["d"]), dtype=torch.float16, device="cuda")
    rows = torch.cat([st["open"].view(2, n * _GROUP, c["hkv"], c["d"]), new.view(2, -1, c["hkv"], c["d"]), zero], dim=1)
    x = rows[:, at["rows"].view(-1)].view(2, n, at["wide"], _GROUP, c["hkv"], c["d"]).permute(0, 1, 4, 2, 3, 5)
    q, s = _quantised(x)
    st["cache"][:, at["i"], :, at["g"]] = q[:, at["i"], :, at["f"]]
    st["scale"][:, at["i"], :, at["g"]] = s[:, at["i"], :, at["f"]]
    st["opened"] = x[:, at["all"], :, at["last"]]


def _cached(st):
    """What the cache stands for, in 32 bits: [K | V][sequence][kv head][token][head_dim]."""
    x = st["cache"].float() * st["scale"][..., None, None]
    at = st["at"]
    x[:, at["left"], :, at["left_g"]] = st["opened"][at["left"]].float()
    return x.flatten(3, 4)


def _run_plain(st):
    c, x = st["c"], st["x"]
    if c["kind"] == "rotate":
        return _rotate_plain(c, x)
    _append(st, st["at"], torch.stack([x["nk"], x["nv"]]))
    kv = _cached(st)
    if c["kind"] == "write":
        kv = kv.masked_fill_(st["hidden"][None, :, None, :, None], 0.0)
        return kv[:, :, :, :st["most"]].half()
    n, hkv, g, d = c["seqs"], c["hkv"], c["hq"] // c["hkv"], c["d"]
    q = x["q"][st["q_rows"]].float()  # [sequence][token][head][d], padded
    t = q.shape[1]
    q = q.view(n, t, hkv, g, d).transpose(1, 2).reshape(n * hkv, t * g, d)
    keys = kv.shape[3]
    s = torch.bmm(q, kv[0].reshape(n * hkv, keys, d).transpose(1, 2).contiguous()).mul_(d ** -0.5)
    s = s.view(n, hkv, t, g, keys).masked_fill_(st["causal"][:, None, :, None, :], float("-inf"))
    e = s.sub_(s.amax(dim=-1, keepdim=True)).exp_()
    e = e.div_(e.sum(dim=-1, keepdim=True)).view(n * hkv, t * g, keys)
    o = torch.bmm(e, kv[1].reshape(n * hkv, keys, d)).view(n, hkv, t, g, d).transpose(1, 2)
    return o.reshape(n, t, c["hq"], d)[st["q_real"]].half()


def _rotate_plain(c, x):
    n = c["rd"] // 2
    # Angles in 64 bits: a far position times a frequency has no digits left in 32.
    freq = 10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)
    axis = torch.tensor(_sections(c), device="cuda")
    angle = x["pos"].double()[axis].t() * freq  # [token][pair]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    outs = []
    for name, w in (("q", "qw"), ("k", "kw")):
        v = x[name].reshape(c["tokens"], -1, c["d"]).float()
        if c["norm"]:
            v = v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + 1e-5) * x[w].float()
        r = v[..., :c["rd"]]
        a, b = (r[..., :n], r[..., n:]) if c["pairs"] == "halves" else (r[..., 0::2], r[..., 1::2])
        a, b = a * cos - b * sin, a * sin + b * cos
        r = torch.cat([a, b], dim=-1) if c["pairs"] == "halves" else torch.stack([a, b], dim=-1).flatten(-2)
        outs.append(torch.cat([r, v[..., c["rd"]:]], dim=-1).half())
    return tuple(outs)


# --------------------------------------------------------------------------
# The same in 64 bits
# --------------------------------------------------------------------------
def _held64(x, c):
    """What a cache stands for that was given the rows x [token][row]: [token][kv head][d]."""
    x = x.double().view(-1, c["hkv"], c["d"])
    whole = x.shape[0] // _GROUP
    for h in range(c["hkv"] if whole else 0):
        body = x[:whole * _GROUP, h].reshape(whole, -1)
        step = body.abs().max(dim=1).values / torch.tensor([127.0], dtype=torch.float64, device="cuda")
        step = (step.view(torch.int64) >> 42 << 42).view(torch.float64)  # 11 significant bits
        near = torch.round(body / torch.where(step > 0, step, 1.0)[:, None]) * step[:, None]
        x[:whole * _GROUP, h] = near.view(-1, c["d"])
    return x


def _attend64(q, k, v, first, scale):
    """Attention of one head's q [T][d], token j over the keys 0 .. first + j."""
    out, kt, step = torch.zeros_like(q), k.t().contiguous(), max(1, (1 << 27) // k.shape[0])
    for a in range(0, q.shape[0], step):
        s = q[a:a + step] @ kt * scale
        s += torch.full_like(s, float("-inf")).triu(first + a + 1)
        out[a:a + step] = torch.softmax(s, dim=1) @ v
    return out


def exact(c, seed):
    x = _inputs(c, seed)
    if c["kind"] == "rotate":
        return _rotate64(c, x)
    pre, cnt = _lengths(c)
    most, g = max(p + n for p, n in zip(pre, cnt)), c["hq"] // c["hkv"]
    if c["kind"] == "write":
        out = torch.zeros((2, c["seqs"], c["hkv"], most, c["d"]), dtype=torch.float64, device="cuda")
    else:
        out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    p0 = n0 = 0
    for i, (p, n) in enumerate(zip(pre, cnt)):
        k, v = (_held64(torch.cat([x[m][p0:p0 + p], x["n" + m][n0:n0 + n]]), c) for m in ("k", "v"))
        if c["kind"] == "write":
            out[0, i, :, :p + n], out[1, i, :, :p + n] = k.transpose(0, 1), v.transpose(0, 1)
        else:
            for h in range(c["hq"]):
                out[n0:n0 + n, h] = _attend64(x["q"][n0:n0 + n, h].double(), k[:, h // g].contiguous(),
                                              v[:, h // g].contiguous(), p, c["d"] ** -0.5)
        p0, n0 = p0 + p, n0 + n
    return out


def _rotate64(c, x):
    """The rotation as a product of complex numbers."""
    n = c["rd"] // 2
    pos = x["pos"].cpu().numpy().astype(np.float64)
    angle = pos[np.array(_sections(c))].T / 10000.0 ** (np.arange(n) / n)
    turn = torch.from_numpy(np.exp(1j * angle)).cuda()[:, None, :]
    outs = []
    for v, w in ((x["q"], x["qw"]), (x["k"], x["kw"])):
        v = v.double().reshape(c["tokens"], -1, c["d"])
        if w is not None:
            v = v / (v.pow(2).sum(-1, keepdim=True) / c["d"] + 1e-5).sqrt() * w.double()
        first = slice(0, n) if c["pairs"] == "halves" else slice(0, c["rd"], 2)
        second = slice(n, c["rd"]) if c["pairs"] == "halves" else slice(1, c["rd"], 2)
        z = torch.complex(v[..., first], v[..., second]) * turn
        v = v.clone()
        v[..., first], v[..., second] = z.real, z.imag
        outs.append(v)
    return tuple(outs)
