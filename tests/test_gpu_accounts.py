"""GPU: the accounts of attention weights -- DecodeBatch.decode_weights and
PrefillBatch.weights -- against 64-bit attention, elementwise within bounds derived
from the roundings of the path."""
import numpy as np
import pytest
import torch

from retention_ref import Cache, attend, check_account, check_out, dev, even_tail

pytestmark = pytest.mark.gpu


def decode_step(tl, c, lens, G, append=True, given=True, in_place=False, layer=0, attended=None, scale=None):
    """One decode_weights call on the cache, checked."""
    n, hq, d = len(lens), c.hkv * G, c.d
    scale = d ** -0.5 if scale is None else scale
    q = c.rng.standard_normal((n, hq, d)).astype(np.float16)
    nk, nv = c.rows(n), c.rows(n)
    b = tl.DecodeBatch(c.mgr, n, hq)
    if attended is None:
        b.prepare(c.ids)
    else:
        b.prepare_lengths(c.ids, attended)
    w_in, w_out = c.account(), c.account(7.0)
    w_in.copy_(torch.rand(w_in.shape, device="cuda"))
    if in_place:
        w_out = w_in
    start, before = w_in.cpu().numpy(), w_out.cpu().numpy()
    dq, dk, dv = dev(q), dev(nk), dev(nv)
    out = torch.full((n, hq, d), 9.0, dtype=torch.float16, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    if attended is None and not append:
        b.append(0, 1, dk.data_ptr(), dv.data_ptr(), s)
    b.decode_weights(layer, dq.data_ptr(), dk.data_ptr() if append else None, dv.data_ptr() if append else None,
                     out.data_ptr(), scale, w_in.data_ptr() if given else None, w_out.data_ptr(), s)
    torch.cuda.synchronize()
    got, acc = out.cpu().numpy(), w_out.cpu().numpy()
    for i in range(n):
        if attended is None:
            k = np.concatenate([c.k[layer][i], nk[i:i + 1]])
            v = np.concatenate([c.v[layer][i], nv[i:i + 1]])
            old = lens[i]
        else:
            k, v, old = c.k[layer][i][:attended[i]], c.v[layer][i][:attended[i]], attended[i]
        S = len(k)
        o, mass, w, err = attend(q[i:i + 1], k, v, scale)
        check_out(got[i:i + 1], o, mass, err, S)
        want = w.reshape(c.hkv, G, S).sum(axis=1)
        base = start[c.slot[i], :, :S].astype(np.float64) * (np.arange(S) < old) if given else np.zeros((c.hkv, S))
        check_account(acc[c.slot[i], :, :S], want + base, w, err, G, S, base)
        assert np.array_equal(acc[c.slot[i], :, S:], before[c.slot[i], :, S:])
    for slot in set(range(before.shape[0])) - set(c.slot):
        assert np.array_equal(acc[slot], before[slot])
    return got, acc


@pytest.mark.parametrize("d,hkv,G,block,lens", [
    (64, 8, 1, 0, [127, 255, 383, 511]),
    (128, 2, 4, 0, [0, 1, 62, 63, 64, 65, 700]),
    (128, 2, 8, 16, [0, 15, 16, 17, 300, 1023]),
    (256, 1, 2, 32, [31, 33, 200, 640]),
    (32, 4, 1, 64, [5, 64, 129, 513]),
    (32, 3, 8, 0, [1, 2000]),
    (256, 2, 8, 0, [95, 96]),
    (128, 1, 1, 16, [4099]),
])
def test_decode_weights(tl, d, hkv, G, block, lens):
    c = Cache(tl, lens, hkv, d, block=block, seed=d + G, spare=1, hq=hkv * G)
    decode_step(tl, c, lens, G)


@pytest.mark.parametrize("d,hkv,G,block,lens", [
    (32, 8, 1, 0, [3000]),         # little work: pieces of four tiles
    (64, 8, 4, 16, [2500, 40]),
    (128, 8, 8, 16, [1500]),
    (256, 4, 4, 0, [900, 300]),
    (256, 2, 2, 16, [2600]),
    (128, 8, 4, 0, [8300]),        # more: eight waves
    (64, 8, 1, 0, [1024] * 8),
    (64, 8, 1, 0, [1500] * 20),    # whole entries on eight waves
    (64, 2, 2, 0, [300, 767]),
    (32, 8, 1, 16, [(i * 97) % 700 for i in range(40)]),   # many entries
    (64, 8, 2, 0, [50] * 33 + [4000]),                     # ... and a long one among them
])
def test_decode_weights_in_pieces(tl, d, hkv, G, block, lens):
    c = Cache(tl, lens, hkv, d, block=block, seed=d + G + 1, hq=hkv * G)
    decode_step(tl, c, lens, G)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.5])
def test_decode_weights_scales_of_either_sign(tl, scale):
    lens = [70, 900]
    c = Cache(tl, lens, 2, 64, seed=16, hq=4)
    decode_step(tl, c, lens, 2, scale=scale)


@pytest.mark.parametrize("block", [0, 16])
@pytest.mark.parametrize("append,given,in_place", [(False, True, False), (True, False, False), (True, True, True)])
def test_decode_weights_forms(tl, block, append, given, in_place):
    """Without the append (after DecodeBatch.append), from zero, in place."""
    lens = [3, 70, 130]
    c = Cache(tl, lens, 2, 64, block=block, seed=5, hq=4)
    decode_step(tl, c, lens, 2, append, given, in_place)


def test_decode_weights_of_given_lengths(tl):
    """prepare_lengths: no new token, every attended token's account goes on; a
    sequence that attends to nothing gets zeros and keeps its account."""
    lens = [40, 64, 10]
    c = Cache(tl, lens, 2, 128, seed=6, hq=8)
    got, _ = decode_step(tl, c, lens, 4, append=False, attended=[33, 0, 10])
    assert not got[1].any()


def test_decode_weights_more_entries_than_a_launch_takes(tl):
    lens = [(i * 37) % 90 for i in range(150)]
    c = Cache(tl, lens, 1, 32, block=16, seed=7, hq=2)
    decode_step(tl, c, lens, 2)


def test_decode_weights_layers_and_another_stream(tl):
    lens = [100, 333]
    c = Cache(tl, lens, 2, 64, layers=3, seed=8, hq=4)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for layer in (2, 0):
            decode_step(tl, c, lens, 2, layer=layer)


def test_decode_weights_values_at_the_ends_of_their_range(tl):
    """Scores far apart and far from zero, and accounts of very different size."""
    c = Cache(tl, [200], 1, 64, seed=9, hq=2)
    q = np.zeros((1, 2, 64), np.float16)
    q[..., 0] = [[60000.0, -300.0]]
    kn = c.rows(1)
    k = np.concatenate([c.k[0][0], kn])
    b = tl.DecodeBatch(c.mgr, 1, 2)
    b.prepare(c.ids)
    w_out, out = c.account(), torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda")
    dq, dk = dev(q), dev(kn)
    b.decode_weights(0, dq.data_ptr(), dk.data_ptr(), dk.data_ptr(), out.data_ptr(), 0.125, None, w_out.data_ptr())
    torch.cuda.synchronize()
    _, _, w, err = attend(q, k, np.concatenate([c.v[0][0], kn]), 0.125)
    # scores near 20000 cannot be told apart better than their own rounding
    got = w_out.cpu().numpy()[0, :, :201]
    assert np.isfinite(got).all() and abs(got.sum() - 2) < 1e-4
    top = int(w[0, 0].argmax())
    assert w[0, 0, top] > 0.999 and got[0, top] >= 0.999
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("d,block", [(64, 0), (128, 16), (256, 0)])
def test_decode_weights_far_below_the_largest(tl, d, block):
    c, q, want, tol = even_tail(tl, 4096, d, block)
    b = tl.DecodeBatch(c.mgr, 1, 1)
    b.prepare_lengths(c.ids, [4096])
    dq, w = dev(q[None, None]), c.account()
    out = torch.empty_like(dq)
    b.decode_weights(0, dq.data_ptr(), None, None, out.data_ptr(), 1.0, None, w.data_ptr())
    torch.cuda.synchronize()
    assert np.abs(out.cpu().numpy().astype(np.float64) - want).max() <= tol


def test_decode_weights_offsets_beyond_32_bits(tl):
    """A cache of more than 4 GiB of keys per slot."""
    hkv, d, S = 32, 256, 262144 + 300
    mgr = tl.KVCacheManager(num_layers=1, num_heads=hkv, head_dim=d, max_seq_len=S + 1, max_batch_size=1)
    sid, _ = mgr.allocateSequence(S + 1)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((S, hkv, d), generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    assert mgr.appendKV(sid, 0, k.data_ptr(), v.data_ptr(), S) is None
    mgr.advanceSeqLen(sid, S)
    q = torch.randn((1, hkv, d), generator=g, device="cuda", dtype=torch.float16)
    out = torch.empty_like(q)
    acc = torch.zeros((1, hkv, S + 1), device="cuda")
    b = tl.DecodeBatch(mgr, 1, hkv)
    b.prepare_lengths([sid], [S])
    b.decode_weights(0, q.data_ptr(), None, None, out.data_ptr(), d ** -0.5, None, acc.data_ptr())
    torch.cuda.synchronize()
    for h in (0, hkv - 1):
        s = (k[:, h].double() @ q[0, h].double()) * d ** -0.5
        p = torch.softmax(s, dim=0)
        # scores of a few units, 260 roundings each; sums of 2^18 terms in the order of a tree
        assert (acc[0, h, :S].double() - p).abs().max() <= 1e-3 * p.max()
        assert (out[0, h].double() - p @ v[:, h].double()).abs().max() <= 2.0 ** -10 * (p @ v[:, h].double().abs()).max()


def test_decode_weights_captured(tl):
    """A captured call, replayed between eager work of the same batch."""
    lens = [50, 400]
    c = Cache(tl, lens, 2, 128, seed=11, hq=8)
    b = tl.DecodeBatch(c.mgr, 2, 8)
    b.prepare(c.ids)
    q = dev(c.rng.standard_normal((2, 8, 128)).astype(np.float16))
    nk, nv = dev(c.rows(2)), dev(c.rows(2))
    out = torch.zeros((2, 8, 128), dtype=torch.float16, device="cuda")
    w_in, w_out = c.account(0.25), c.account()

    def call():
        b.decode_weights(0, q.data_ptr(), nk.data_ptr(), nv.data_ptr(), out.data_ptr(), 128 ** -0.5, w_in.data_ptr(),
                         w_out.data_ptr(), torch.cuda.current_stream().cuda_stream)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        q.normal_()
        call()
        torch.cuda.synchronize()
        want = out.clone(), w_out.clone()
        out.zero_(), w_out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(w_out, want[1]), i


def test_graphs_of_one_batch_share_its_workspace(tl):
    """Decode and prompt accounts of two layers and windows, each captured into a graph
    of its own, replayed in turn with eager calls between."""
    lens, new = [3000, 40], [33, 150]
    c = Cache(tl, lens, 2, 64, room=3300, layers=2, seed=17, hq=8)
    d, p = tl.DecodeBatch(c.mgr, 2, 8), tl.PrefillBatch(c.mgr, 2, 8)
    d.prepare(c.ids)
    p.prepare(c.ids, new)
    q = dev(c.rng.standard_normal((sum(new), 8, 64)).astype(np.float16))
    k, v = dev(c.rows(sum(new))), dev(c.rows(sum(new)))
    outs = [torch.zeros((2, 8, 64), dtype=torch.float16, device="cuda") for _ in range(2)]
    accs = [c.account() for _ in range(4)]
    for layer in range(2):
        p.append(layer, k.data_ptr(), v.data_ptr())

    def decode(layer):
        d.decode_weights(layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[layer].data_ptr(), 0.125, None,
                         accs[layer].data_ptr(), torch.cuda.current_stream().cuda_stream)

    def prompt(i):  # (decode appends the rows that the prompt begins with)
        p.weights(i, q.data_ptr(), 0.125, [0, 20][i], None, accs[2 + i].data_ptr(), torch.cuda.current_stream().cuda_stream)

    calls = [lambda: decode(0), lambda: decode(1), lambda: prompt(0), lambda: prompt(1)]
    # (the plan of a window is made anew after another one: its launches do not depend on that)
    for call in calls:
        call()
    torch.cuda.synchronize()
    want = [x.clone() for x in outs + accs]
    graphs = []
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call()
    for order in ([0, 1, 2, 3], [3, 1, 0, 2], [2, 0, 3, 1]):
        for x in outs + accs:
            x.zero_()
        for i in order:
            graphs[i].replay()
            calls[order[0]]()
        torch.cuda.synchronize()
        for x, y in zip(outs + accs, want):
            assert torch.equal(x, y), order


def test_a_capture_does_not_grow_the_workspace(tl):
    c = Cache(tl, [300], 1, 64, seed=12)
    b = tl.DecodeBatch(c.mgr, 1, 1)
    b.prepare(c.ids)
    q = dev(c.rng.standard_normal((1, 1, 64)).astype(np.float16))
    k, w = dev(c.rows(1)), c.account()
    out = torch.empty_like(q)
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x.add_(1)  # a capture of something
        with pytest.raises(tl.TinyLLMError, match="captured"):
            b.decode_weights(0, q.data_ptr(), k.data_ptr(), k.data_ptr(), out.data_ptr(), 0.125, None, w.data_ptr(),
                             torch.cuda.current_stream().cuda_stream)


def test_decode_weights_refusals(tl):
    c = Cache(tl, [5, 9], 2, 64, seed=13)
    b = tl.DecodeBatch(c.mgr, 2, 2)
    b.prepare(c.ids)
    q, w = torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda"), c.account()
    p, a = q.data_ptr(), w.data_ptr()
    for args, msg in (((0, None, p, p, p, 1.0, a, a), "q/out"), ((0, p, p, p, None, 1.0, a, a), "q/out"),
                      ((0, p, p, None, p, 1.0, a, a), "new_v"), ((0, p, None, p, p, 1.0, a, a), "new_k"),
                      ((1, p, p, p, p, 1.0, a, a), "layer_idx"), ((-1, p, p, p, p, 1.0, a, a), "layer_idx"),
                      ((0, p + 2, p, p, p, 1.0, a, a), "aligned"), ((0, p, p, p, p + 8, 1.0, a, a), "aligned"),
                      ((0, p, p, p, p, 1.0, a, None), "weights_out"), ((0, p, p, p, p, 1.0, a, a + 2), "aligned"),
                      ((0, p, p, p, p, 1.0, a, a + 4), "overlaps")):
        with pytest.raises(tl.TinyLLMError, match=msg):
            b.decode_weights(*args)
    b.prepare_lengths(c.ids, [1, 2])
    with pytest.raises(tl.TinyLLMError, match="prepare"):
        b.decode_weights(0, p, p, p, p, 1.0, a, a)
    b.prepare([])
    b.decode_weights(0, p, p, p, p, 1.0, a, a)  # nothing to do
    torch.cuda.synchronize()
    assert not w.any()


# ------------------------------------------------------------------- prompts
def prompt_step(tl, c, pre, new, G, window, given=True, in_place=False, layer=0, scale=None):
    n, hq, d = len(new), c.hkv * G, c.d
    scale = d ** -0.5 if scale is None else scale
    t = sum(new)
    q = c.rng.standard_normal((t, hq, d)).astype(np.float16)
    nk, nv = c.rows(t), c.rows(t)
    p = tl.PrefillBatch(c.mgr, n, hq)
    p.prepare(c.ids, new)
    s = torch.cuda.current_stream().cuda_stream
    dk, dv, dq = dev(nk), dev(nv), dev(q)
    p.append(layer, dk.data_ptr(), dv.data_ptr(), s)
    w_in, w_out = c.account(), c.account(7.0)
    w_in.copy_(torch.rand(w_in.shape, device="cuda"))
    if in_place:
        w_out = w_in
    start, before = w_in.cpu().numpy(), w_out.cpu().numpy()
    p.weights(layer, dq.data_ptr(), scale, window, w_in.data_ptr() if given else None, w_out.data_ptr(), s)
    torch.cuda.synchronize()
    acc, at = w_out.cpu().numpy(), 0
    for i in range(n):
        S, w_n = pre[i] + new[i], min(new[i], window or new[i])
        k = np.concatenate([c.k[layer][i], nk[at:at + new[i]]])
        last = pre[i] + np.arange(new[i] - w_n, new[i])
        _, _, w, err = attend(q[at + new[i] - w_n:at + new[i]], k, k, scale, last)
        want = w.reshape(c.hkv, G * w_n, S).sum(axis=1)
        base = start[c.slot[i], :, :S].astype(np.float64) * (np.arange(S) < pre[i]) if given else np.zeros((c.hkv, S))
        check_account(acc[c.slot[i], :, :S], want + base, w, err, G * w_n, S, base)
        assert np.array_equal(acc[c.slot[i], :, S:], before[c.slot[i], :, S:])
        at += new[i]
    for slot in set(range(before.shape[0])) - set(c.slot):
        assert np.array_equal(acc[slot], before[slot])


@pytest.mark.parametrize("d,hkv,G,block,pre,new,window", [
    (64, 2, 1, 0, [0, 0, 0], [1, 64, 333], 0),
    (128, 1, 4, 0, [0, 17, 500], [300, 1, 65], 0),
    (128, 2, 8, 16, [0, 31, 40], [129, 16, 255], 0),
    (128, 1, 4, 16, [0, 700], [900, 3], 32),
    (64, 2, 2, 0, [1000, 0], [40, 40], 1),
    (256, 1, 2, 32, [0, 90], [100, 257], 33),
    (256, 1, 1, 0, [0], [400], 0),
    (32, 3, 8, 64, [5, 0], [70, 128], 7),
    (32, 1, 1, 0, [0], [2], 5),
])
def test_prompt_weights(tl, d, hkv, G, block, pre, new, window):
    c = Cache(tl, pre, hkv, d, room=max(a + b for a, b in zip(pre, new)) + 3, block=block, seed=d + G, spare=1, hq=hkv * G)
    prompt_step(tl, c, pre, new, G, window)


@pytest.mark.parametrize("given,in_place", [(False, False), (True, True)])
def test_prompt_weights_forms(tl, given, in_place):
    c = Cache(tl, [20, 0], 2, 64, room=200, layers=2, seed=3, hq=4)
    prompt_step(tl, c, [20, 0], [100, 150], 2, 0, given, in_place, layer=1)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.5])
def test_prompt_weights_scales_of_either_sign(tl, scale):
    c = Cache(tl, [70, 0], 2, 64, room=400, seed=13, hq=4)
    prompt_step(tl, c, [70, 0], [300, 65], 2, 0, scale=scale)


@pytest.mark.parametrize("d,hkv,G,pre,new,window", [
    (128, 8, 4, [0, 900], [1100, 700], 0),   # rows and keys over several workgroups, the diagonal between them
    (64, 1, 1, [0], [2500], 0),
    (128, 1, 8, [3000], [1500], 1000),
    (128, 1, 8, [8968], [32], 0),            # few rows, many chunks of keys
    (256, 2, 4, [4000], [40], 20),
])
def test_prompt_weights_long(tl, d, hkv, G, pre, new, window):
    c = Cache(tl, pre, hkv, d, room=max(a + b for a, b in zip(pre, new)), seed=14, hq=hkv * G)
    prompt_step(tl, c, pre, new, G, window)


def test_prompt_weights_more_entries_than_a_launch_takes(tl):
    n = 100
    pre, new = [(i * 7) % 40 for i in range(n)], [1 + (i * 11) % 50 for i in range(n)]
    c = Cache(tl, pre, 1, 32, room=96, block=16, seed=4, hq=2)
    prompt_step(tl, c, pre, new, 2, 9)


def test_prompt_weights_of_every_window_in_one_step(tl):
    """The plan follows the window from call to call."""
    c = Cache(tl, [10], 1, 64, room=300, seed=5, hq=2)
    p = tl.PrefillBatch(c.mgr, 1, 2)
    p.prepare(c.ids, [200])
    q = c.rng.standard_normal((200, 2, 64)).astype(np.float16)
    nk, dq = c.rows(200), dev(q)
    dk = dev(nk)
    p.append(0, dk.data_ptr(), dk.data_ptr())
    k = np.concatenate([c.k[0][0], nk])
    for window in (3, 0, 200, 1, 1000):
        w_out = c.account()
        p.weights(0, dq.data_ptr(), 0.125, window, None, w_out.data_ptr())
        torch.cuda.synchronize()
        n = min(200, window or 200)
        _, _, w, err = attend(q[200 - n:], k, k, 0.125, 10 + np.arange(200 - n, 200))
        check_account(w_out.cpu().numpy()[0, :, :210], w.reshape(1, 2 * n, 210).sum(axis=1), w, err, 2 * n, 210)


def test_prompt_weights_refusals(tl):
    c = Cache(tl, [5], 2, 64, room=64, seed=6)
    p = tl.PrefillBatch(c.mgr, 1, 2)
    p.prepare(c.ids, [4])
    q, w = torch.zeros((4, 2, 64), dtype=torch.float16, device="cuda"), c.account()
    x, a = q.data_ptr(), w.data_ptr()
    for args, msg in (((0, None, 1.0, 0, a, a), "q is null"), ((0, x + 4, 1.0, 0, a, a), "aligned"),
                      ((0, x, 1.0, -1, a, a), "window"), ((2, x, 1.0, 0, a, a), "layer_idx"),
                      ((0, x, 1.0, 0, a, None), "weights_out"), ((0, x, 1.0, 0, a, a + 8), "overlaps")):
        with pytest.raises(tl.TinyLLMError, match=msg):
            p.weights(*args)
    p.prepare([], [])
    p.weights(0, x, 1.0, 0, a, a)
    torch.cuda.synchronize()
    assert not w.any()
