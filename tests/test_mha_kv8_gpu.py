"""Decode attention over an 8-bit KV cache, against the definition in 64 bits with a bound from the roundings (kv8_cases)."""
import ctypes
import math

import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

import kv8_cases as C

pytestmark = pytest.mark.gpu
D, BF16 = C.D, C.BF16
FORMATS = [C.E4M3, C.INT8]


def workspace(dev, n_q, msl):
    return torch.full((ops.workspace_bytes(n_q, D, msl) // 4,), math.nan, device=dev)


def decode(dev, q, cache, n_kv, msl, pos, fmt, *, ws="enough", **more):
    n_q = q.shape[0]
    out, tap = torch.full((n_q, D), math.nan, dtype=BF16, device=dev), torch.full((n_q, D), math.nan, device=dev)
    ws = workspace(dev, n_q, msl) if isinstance(ws, str) else ws
    r = ops.mha_decode_kv8(q, cache, out, ws, output_f32=tap, pos=pos, kv_dim=n_kv * D, kv_mul=n_q // n_kv, head_num=n_q, head_dim=D, max_seq_len=msl, kv8_format=fmt, **more)
    assert r is out
    return out.cpu(), tap.cpu()


HEADS = [(1, 1), (16, 8), (32, 8), (64, 8), (16, 1), (33, 3), (5, 5), (40, 8)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("keys", [1, 2, 31, 32, 33, 100, 129, 257, 1000, 4099])
def test_lengths_and_heads(dev, n_q, n_kv, keys, fmt):
    g = torch.Generator().manual_seed(keys * 100 + n_q)
    msl = keys + 70
    cache, k, v = C.filled(2, n_kv, msl, keys, fmt, keys + n_q)
    q = C.rows(g, n_q, outliers=False)
    out, tap = decode(dev, q.to(dev), cache.to(dev), n_kv, msl, keys - 1, fmt, layer_id=1)
    C.close(tap, *C.attention(q, k[1], v[1]), rounded=out)
    assert torch.equal(tap.to(BF16), out)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 16, 64, 65, 200, 256])
def test_splits(dev, splits, fmt):
    g = torch.Generator().manual_seed(splits)
    keys, n_q, n_kv = 33001, 6, 2
    cache, k, v = C.filled(1, n_kv, keys, keys, fmt, splits)
    q = C.rows(g, n_q, outliers=False)
    want = C.attention(q, k[0], v[0])
    out, tap = decode(dev, q.to(dev), cache.to(dev), n_kv, keys, keys - 1, fmt, layer_id=0, num_splits=splits)
    C.close(tap, *want, rounded=out)
    # the same call again, the workspace as the first one left it: the same bits
    ws = workspace(dev, n_q, keys)
    again = [decode(dev, q.to(dev), cache.to(dev), n_kv, keys, keys - 1, fmt, layer_id=0, num_splits=splits, ws=ws) for _ in range(3)]
    assert all(torch.equal(x[1], tap) for x in again)


@pytest.mark.parametrize("n_q,n_kv,keys,splits", [(256, 16, 3000, 0), (144, 9, 2500, 70), (144, 9, 2500, 3), (130, 10, 700, 0), (160, 160, 1100, 0), (300, 300, 800, 20), (192, 12, 9000, 256)])
def test_more_heads_than_are_joined_by_workgroups_of_their_own(dev, n_q, n_kv, keys, splits):
    """Over 128 query heads one workgroup joins all of a KV head's: a wavefront each, or all of them in turn where there are over 64 splits."""
    g = torch.Generator().manual_seed(n_q + splits)
    cache, k, v = C.filled(1, n_kv, keys, keys, C.E4M3, keys)
    q = C.rows(g, n_q, outliers=False)
    want = C.attention(q, k[0], v[0])
    cache, ws = cache.to(dev), torch.full((n_q * 528 * 256 // 4 + 64,), math.nan, device=dev)
    taps = []
    for _ in range(2):
        out, tap = decode(dev, q.to(dev), cache, n_kv, keys, keys - 1, C.E4M3, layer_id=0, num_splits=splits, ws=ws)
        C.close(tap, *want, rounded=out)
        taps.append(tap)
    assert torch.equal(*taps)


def test_offsets_past_32_bits(dev):
    """A layer that starts past 4 GiB of the cache, and one KV head whose records alone pass 4 GiB."""
    n_kv, msl, layers = 8, 131072, 17
    per = ops.kv8_bytes(1, msl, n_kv * D, D)
    assert per * (layers - 1) > 1 << 32
    big = torch.empty(per * layers, dtype=torch.uint8, device=dev)
    g = torch.Generator().manual_seed(1)
    small, k, v = C.filled(1, n_kv, 700, 700, C.INT8, 8)
    last = big[per * (layers - 1):].view(1, n_kv, msl // 32, C.RECORD)
    last[:, :, :small.shape[2]] = small.to(dev)
    q = C.rows(g, 16, outliers=False)
    out, tap = decode(dev, q.to(dev), big, n_kv, msl, 699, C.INT8, layer_id=layers - 1)
    C.close(tap, *C.attention(q, k[0], v[0]), rounded=out)
    del big, last
    # all codes 0 but the rows of one token at the end, whose score outweighs the others': its V row comes out
    msl = (1 << 32) // 260 + 4000
    cache = torch.zeros(ops.kv8_bytes(1, msl, D, D), dtype=torch.uint8, device=dev)
    assert cache.numel() > 1 << 32
    x = torch.randn(3, D, generator=g).to(BF16)
    sin, cos, w = torch.zeros(msl, 64, device=dev), torch.ones(msl, 64, device=dev), torch.full((2 * D,), 3.0, dtype=BF16, device=dev)
    kv = torch.stack([x[0], x[2]]).to(dev)
    ops.mha_decode_append_kv8(kv[0], kv[0], kv[1], w, sin, cos, cache, torch.zeros(D, dtype=BF16, device=dev), workspace(dev, 1, msl), layer_id=0, pos=msl - 1, kv_dim=D, kv_mul=1, head_num=1,
                              head_dim=D, max_seq_len=msl, kv8_format=C.INT8)
    out, tap = decode(dev, (3 * kv[0]).view(1, D), cache, 1, msl, msl - 1, C.INT8, layer_id=0)
    codes, scale = C.quantise(x[2].view(1, D), C.INT8)
    row = C.stands_for(codes, scale, C.INT8)
    # (score 3 x 3 |x|^2 / sqrt(128) = 100 above the others': 16.5 million weights of e^-100)
    assert bool(((tap.double() - row).abs() <= 2.0 ** -15 * row.abs()).all())


def test_two_graphs_that_share_a_workspace(dev):
    """Captured calls of two models (other heads, lengths, codes) with one workspace, replayed in turn with eager calls between."""
    g = torch.Generator().manual_seed(55)
    ws = torch.full((ops.workspace_bytes(32, D, 8192) // 4,), math.nan, device=dev)
    made = []
    for n_q, n_kv, keys, fmt in ((32, 8, 4100, C.E4M3), (24, 2, 1800, C.INT8)):
        cache, k, v = C.filled(1, n_kv, keys, keys, fmt, keys)
        q, cache = C.rows(g, n_q, outliers=False), cache.to(dev)
        q_dev, out, tap = q.to(dev), torch.zeros(n_q, D, dtype=BF16, device=dev), torch.zeros(n_q, D, device=dev)

        def call(q_dev=q_dev, cache=cache, out=out, tap=tap, n_q=n_q, n_kv=n_kv, keys=keys, fmt=fmt):
            ops.mha_decode_kv8(q_dev, cache, out, ws, output_f32=tap, layer_id=0, pos=keys - 1, kv_dim=n_kv * D, kv_mul=n_q // n_kv, head_num=n_q, head_dim=D, max_seq_len=keys,
                               kv8_format=fmt)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        made.append((graph, call, out, tap, C.attention(q, k[0], v[0])))
    for turn in range(6):
        for graph, call, out, tap, want in made:
            out.zero_(), tap.zero_()
            graph.replay() if turn != 3 else call()
            torch.cuda.synchronize()
            C.close(tap.cpu(), *want, rounded=out.cpu())


def test_without_a_workspace_and_with_little(dev):
    g = torch.Generator().manual_seed(3)
    keys, n_q, n_kv = 5000, 8, 2
    cache, k, v = C.filled(1, n_kv, keys, keys, C.E4M3, 9)
    q = C.rows(g, n_q, outliers=False)
    want = C.attention(q, k[0], v[0])
    for room in (None, 4, n_q * 528 * 2 // 4 + 4, n_q * 528 * 5 // 4 + 3):
        ws = None if room is None else torch.full((room + 64,), 5.0, device=dev)
        out, tap = decode(dev, q.to(dev), cache.to(dev), n_kv, keys, keys - 1, C.E4M3, layer_id=0, ws=None if room is None else ws[:room])
        C.close(tap, *want, rounded=out)
        assert room is None or bool((ws[room:] == 5.0).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_position_on_the_device(dev, fmt):
    g = torch.Generator().manual_seed(8)
    msl, n_q, n_kv = 9000, 32, 8
    cache, k, v = C.filled(1, n_kv, msl, msl, fmt, 21)
    q, ws = C.rows(g, n_q, outliers=False).to(dev), workspace(dev, n_q, msl)
    cache = cache.to(dev)
    for at, bound in ((0, 8999), (31, 8999), (32, 500), (127, 8999), (128, 8999), (4098, 8999), (8999, 8999), (9500, 8999), (-3, 8999), (600, 500)):
        word = torch.tensor([at], dtype=torch.int32, device=dev)
        keys = max(0, min(at, bound)) + 1
        out, tap = decode(dev, q, cache, n_kv, msl, bound, fmt, layer_id=0, pos_device=word, ws=ws)
        C.close(tap, *C.attention(q.cpu(), k[0, :, :keys], v[0, :, :keys]), rounded=out)


@pytest.mark.parametrize("n_q,n_kv,msl,fmt", [(8, 1, 30000, C.E4M3), (22, 2, 9000, C.INT8), (48, 8, 2500, C.E4M3)])
def test_one_captured_launch_at_every_length(dev, n_q, n_kv, msl, fmt):
    """A launch captured for the window, replayed at positions all over it: one workgroup's share, slices, splits of every number; the workspace is not cleared between."""
    g = torch.Generator().manual_seed(msl)
    cache, k, v = C.filled(1, n_kv, msl, msl, fmt, n_q)
    q, ws, cache = C.rows(g, n_q, outliers=False), workspace(dev, n_q, msl), cache.to(dev)
    q_dev, word = q.to(dev), torch.zeros(1, dtype=torch.int32, device=dev)
    out, tap = torch.zeros(n_q, D, dtype=BF16, device=dev), torch.zeros(n_q, D, device=dev)

    def call():
        ops.mha_decode_kv8(q_dev, cache, out, ws, output_f32=tap, layer_id=0, pos=msl - 1, pos_device=word, kv_dim=n_kv * D, kv_mul=n_q // n_kv, head_num=n_q, head_dim=D, max_seq_len=msl,
                           kv8_format=fmt)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    edges = [32 * t + x for t in (1, 4, 12, 13, 18, 19, 31, 32, 33, 96, 97) for x in (-1, 0)]
    for pos in [p for p in edges if p < msl] + torch.randint(0, msl, (25,), generator=g).tolist() + [msl - 1]:
        word.fill_(pos)
        out.fill_(math.nan), tap.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        C.close(tap.cpu(), *C.attention(q, k[0, :, :pos + 1], v[0, :, :pos + 1]), rounded=out.cpu())


@pytest.mark.parametrize("fmt", FORMATS)
def test_scores_far_apart(dev, fmt):
    """One position far above the others, anywhere; scales from the smallest to large ones; weights that underflow."""
    g = torch.Generator().manual_seed(2)
    keys, n_q, n_kv = 700, 4, 1
    for peak in (0, 1, 350, 671, 672, 699):
        k, v = C.rows(g, 1, 1, keys), C.rows(g, 1, 1, keys)
        q = C.rows(g, n_q, outliers=False)
        k[0, 0, peak] = (q[0].float() * 40).to(BF16)
        k[0, 0, (peak + 60) % keys] = 0.0
        v[0, 0, (peak + 33) % keys] = (v[0, 0, 5].float() * 2.0 ** 20).to(BF16)
        v[0, 0, (peak + 34) % keys] = (v[0, 0, 5].float() * 2.0 ** -50).to(BF16)
        pad = -keys % 32
        packed, values = [], []
        for x in (k, v):
            c, s = C.quantise(x, fmt)
            values.append(C.stands_for(c, s, fmt))
            packed += [torch.cat([c, torch.full((1, 1, pad, D), 0x7F, dtype=torch.uint8)], 2), torch.cat([s, torch.full((1, 1, pad), math.nan, dtype=BF16)], 2)]
        out, tap = decode(dev, q.to(dev), C.pack(*packed).to(dev), n_kv, keys, keys - 1, fmt, layer_id=0)
        C.close(tap, *C.attention(q, values[0][0], values[1][0]), rounded=out)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("keys,bad", [(1, 0), (40, 39), (40, 3), (3000, 2999), (3000, 1500)])
def test_a_row_of_nan_shows_and_one_behind_the_last_does_not(dev, keys, bad, fmt):
    g = torch.Generator().manual_seed(keys)
    n_q, n_kv, msl = 8, 2, keys + 40
    cache, k, v = C.filled(1, n_kv, msl, keys, fmt, keys)
    q = C.rows(g, n_q, outliers=False)
    ref = C.attention(q, k[0], v[0])
    for which in (1, 3):  # K's scales, V's
        parts = list(C.unpack(cache))
        parts[which][0, 1, bad] = math.nan
        out, tap = decode(dev, q.to(dev), C.pack(*parts).to(dev), n_kv, msl, keys - 1, fmt, layer_id=0)
        C.close(tap[:4], ref[0][:4], ref[1][:4], rounded=out[:4])
        assert bool(torch.isnan(tap[4:]).all()) and bool(torch.isnan(out[4:].float()).all())


def new_token(g, n_q, n_kv):
    x = torch.randn((n_q + 2 * n_kv) * D, generator=g).to(BF16)
    return x.split([n_q * D, n_kv * D, n_kv * D])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("pos", [0, 1, 31, 32, 33, 100, 128, 1000, 4098])
def test_append(dev, n_q, n_kv, pos, fmt):
    """One call against the rows' call and the attention's: the cache's bytes, and the outputs within the bound for the query the rows' call makes."""
    g = torch.Generator().manual_seed(pos * 10 + n_q)
    msl = pos + 45
    cache, _, _ = C.filled(2, n_kv, msl, pos, fmt, pos + n_q)
    q, k, v = (x.to(dev) for x in new_token(g, n_q, n_kv))
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    sin, cos = (x.to(dev) for x in C.tables(msl))
    dims = dict(layer_id=1, pos=pos, kv_dim=n_kv * D, head_num=n_q, head_dim=D, max_seq_len=msl, kv8_format=fmt)
    two, one = cache.to(dev), cache.to(dev)
    normed = torch.zeros(1, n_q * D, dtype=BF16, device=dev)
    ops.qk_norm_rope_append_kv8(normed, k[None], v[None], two, w, sin, cos, row_num=1, query_src=q[None], **dims)
    out, tap = torch.full((n_q, D), math.nan, dtype=BF16, device=dev), torch.full((n_q, D), math.nan, device=dev)
    keep = q.clone()
    r = ops.mha_decode_append_kv8(q, k, v, w, sin, cos, one, out, workspace(dev, n_q, msl), kv_mul=n_q // n_kv, output_f32=tap, **dims)
    assert r is out and torch.equal(q, keep)
    assert torch.equal(one, two)
    kc, ks, vc, vs = C.unpack(two.cpu())
    keys, values = (C.stands_for(c, s, fmt)[1, :, :pos + 1] for c, s in ((kc, ks), (vc, vs)))
    C.close(tap.cpu(), *C.attention(normed.cpu().view(n_q, D), keys, values), rounded=out.cpu())


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_of_a_row_of_nan(dev, fmt):
    g = torch.Generator().manual_seed(6)
    n_q, n_kv, msl, pos = 8, 2, 300, 200
    sin, cos = (x.to(dev) for x in C.tables(msl))
    w = torch.ones(2 * D, dtype=BF16, device=dev)
    for bad in ("k", "v"):
        cache, _, _ = C.filled(1, n_kv, msl, pos, fmt, 2)
        cache = cache.to(dev)
        q, k, v = (x.clone().to(dev) for x in new_token(g, n_q, n_kv))
        (k if bad == "k" else v)[D + 9] = math.inf
        out = torch.zeros(n_q, D, dtype=BF16, device=dev)
        ops.mha_decode_append_kv8(q, k, v, w, sin, cos, cache, out, workspace(dev, n_q, msl), layer_id=0, pos=pos, kv_dim=n_kv * D, kv_mul=4, head_num=n_q, head_dim=D,
                                  max_seq_len=msl, kv8_format=fmt)
        assert bool(torch.isfinite(out[:4].float()).all()) and bool(torch.isnan(out[4:].float()).all())
        parts = C.unpack(cache.cpu())
        assert bool(torch.isnan(parts[1 if bad == "k" else 3][0, 1, pos])) and not bool(parts[0 if bad == "k" else 2][0, 1, pos].any())


@pytest.mark.parametrize("fmt", FORMATS)
def test_steps_of_several_layers_captured_and_replayed(dev, fmt):
    """A decode step of three layers whose position is on the device, captured once, replayed token by token with other work between the
    replays: every replay against the same calls issued one by one. Layers share the workspace."""
    layers, n_q, n_kv, msl, start = 3, 16, 4, 700, 250
    g = torch.Generator().manual_seed(12)
    cache, _, _ = C.filled(layers, n_kv, msl, msl, fmt, 5)  # (the position jumps at the end: what it passes over has been written)
    eager, graphed = cache.to(dev), cache.to(dev)
    sin, cos = (x.to(dev) for x in C.tables(msl))
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    x = torch.zeros((n_q + 2 * n_kv) * D, dtype=BF16, device=dev)
    q, k, v = x.split([n_q * D, n_kv * D, n_kv * D])
    word, ws = torch.tensor([start], dtype=torch.int32, device=dev), workspace(dev, n_q, msl)
    outs = [torch.zeros(layers, n_q * D, dtype=BF16, device=dev) for _ in range(2)]
    dims = dict(kv_dim=n_kv * D, kv_mul=n_q // n_kv, head_num=n_q, head_dim=D, max_seq_len=msl, kv8_format=fmt)

    def step(buffer, out):
        for layer in range(layers):
            ops.mha_decode_append_kv8(q, k, v, w, sin, cos, buffer, out[layer], ws, layer_id=layer, pos=msl - 1, pos_device=word, **dims)

    step(graphed.clone(), outs[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed, outs[1])
    for token in range(40):
        x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        step(eager, outs[0])
        torch.cuda.synchronize()
        ws.view(torch.int32)[:64].add_(0)  # (other work between)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(eager, graphed), token
        word.add_(1 if token < 30 else 20)


def test_streams(dev):
    """Calls on two streams at once, a workspace each."""
    g = torch.Generator().manual_seed(31)
    n_q, n_kv, keys = 32, 8, 3000
    cache, k, v = C.filled(1, n_kv, keys, keys, C.INT8, 1)
    cache = cache.to(dev)
    qs = [C.rows(g, n_q, outliers=False) for _ in range(2)]
    on_dev, streams = [q.to(dev) for q in qs], [torch.cuda.Stream() for _ in range(2)]
    wss, outs = [workspace(dev, n_q, keys) for _ in range(2)], [torch.zeros(n_q, D, dtype=BF16, device=dev) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            ops.mha_decode_kv8(on_dev[i], cache, outs[i], wss[i], layer_id=0, pos=keys - 1, kv_dim=n_kv * D, kv_mul=4, head_num=n_q, head_dim=D, max_seq_len=keys, kv8_format=C.INT8,
                               stream=streams[i])
    torch.cuda.synchronize()
    for q, out in zip(qs, outs):
        ref, off = C.attention(q, k[0], v[0])
        assert bool(((out.cpu().double() - ref).abs() <= off + 2.0 ** -8 * (ref.abs() + off)).all())


def test_a_wait_that_gives_up(dev):
    """No polls at all: NaN for every head, counted, and the next call is as ever."""
    g = torch.Generator().manual_seed(77)
    n_q, n_kv, keys = 8, 2, 4000
    cache, k, v = C.filled(1, n_kv, keys, keys, C.E4M3, 3)
    cache, q, L = cache.to(dev), C.rows(g, n_q, outliers=False), B.lib()
    before, after = ctypes.c_uint64(), ctypes.c_uint64()
    B.check(L.llmi_hip_poll_timeouts(ctypes.byref(before)), "llmi_hip_poll_timeouts")
    old = L.llmi_hip_set_poll_limit(0)
    try:
        ws = workspace(dev, n_q, keys)
        out, tap = decode(dev, q.to(dev), cache, n_kv, keys, keys - 1, C.E4M3, layer_id=0, ws=ws, num_splits=4)
    finally:
        L.llmi_hip_set_poll_limit(old)
    assert bool(torch.isnan(tap).all())
    B.check(L.llmi_hip_poll_timeouts(ctypes.byref(after)), "llmi_hip_poll_timeouts")
    assert after.value - before.value == n_q
    out, tap = decode(dev, q.to(dev), cache, n_kv, keys, keys - 1, C.E4M3, layer_id=0, ws=ws, num_splits=4)
    C.close(tap, *C.attention(q, k[0], v[0]), rounded=out)


def test_a_prompt_stored_then_tokens_then_read_back(dev):
    """As a program uses them together: a prompt prefilled in bf16, quantised, tokens appended one by one, a chunk of rows at once, everything read back
    for the bf16 calls, whose attention over it agrees."""
    g = torch.Generator().manual_seed(40)
    n_q, n_kv, msl, prompt, layers = 16, 8, 400, 130, 2
    dims = dict(kv_dim=n_kv * D, head_dim=D, max_seq_len=msl)
    kb, vb = (C.rows(g, layers, n_kv, msl, outliers=False).to(dev) for _ in range(2))
    cache = C.garbage(layers, n_kv, msl, 1).to(dev)
    sin, cos = (x.to(dev) for x in C.tables(msl))
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    ws, out = workspace(dev, n_q, msl), torch.zeros(n_q, D, dtype=BF16, device=dev)
    ops.kv8_store(kb, vb, cache, layer_num=layers, num_pos=prompt, kv_layout=1, **dims)
    for pos in range(prompt, prompt + 5):
        q, k, v = (x.to(dev) for x in new_token(g, n_q, n_kv))
        for layer in range(layers):
            ops.mha_decode_append_kv8(q, k, v, w, sin, cos, cache, out, ws, layer_id=layer, pos=pos, kv_mul=2, head_num=n_q, **dims)
    chunk = torch.randn(70, (n_q + 2 * n_kv) * D, generator=g).to(BF16).to(dev)
    q, k, v = chunk.split([n_q * D, n_kv * D, n_kv * D], dim=1)
    normed = torch.zeros(70, n_q * D, dtype=BF16, device=dev)
    used = prompt + 5 + 70
    for layer in range(layers):
        ops.qk_norm_rope_append_kv8(normed, k, v, cache, w, sin, cos, row_num=70, layer_id=layer, pos=prompt + 5, head_num=n_q, query_src=q, **dims)
    kb.fill_(math.nan), vb.fill_(math.nan)
    ops.kv8_load(cache, kb, vb, layer_num=layers, num_pos=used, kv_layout=1, **dims)
    query, tap, bf16_out, bf16_tap = normed[-1].view(n_q, D), torch.zeros(n_q, D, device=dev), torch.zeros_like(out), torch.zeros(n_q, D, device=dev)
    for layer in range(layers):
        at = dict(layer_id=layer, pos=used - 1, kv_mul=2, head_num=n_q, **dims)
        ops.mha_decode_kv8(query, cache, out, ws, output_f32=tap, **at)
        ops.mha_decode(query, kb, vb, bf16_out, ws, output_f32=bf16_tap, kv_layout=1, **at)
        kc, ks, vc, vs = C.unpack(cache.cpu())
        keys, values = (C.stands_for(c, s, C.E4M3)[layer, :, :used] for c, s in ((kc, ks), (vc, vs)))
        ref, off = C.attention(query.cpu(), keys, values)
        C.close(tap.cpu(), ref, off, rounded=out.cpu())
        # the read-back rounds K and V to bf16 once, half a step each
        score = (query.cpu().double().view(n_kv, 2, D).abs() @ keys.abs().transpose(1, 2)).amax(-1) / math.sqrt(D)
        more = (2 * 2.0 ** -8 * score.reshape(n_q, 1) + 2.0 ** -8) * C.attention(query.cpu(), keys, values.abs())[0]
        assert bool(((bf16_tap.cpu().double() - ref).abs() <= 2 * off + 1.1 * more).all())
