"""A chosen number of splits at a position on the device: attention over an 8-bit KV cache and the step that files the new token, from the first
position on, against the definition in 64 bits (kv8_cases)."""
import math

import pytest
import torch

from llminfer_amd import ops

import kv8_cases as C

pytestmark = pytest.mark.gpu
D, BF16 = C.D, C.BF16
FORMATS = [C.E4M3, C.INT8]
HEADS = [(8, 2), (9, 1)]
# The launch is sized for positions 0..bound: one record, three, some (one form, or another, by the position), many.
BOUNDS = [20, 95, 1500, 9000]
SPLITS = [0, 1, 2, 3, 4, 70]


def positions(bound):
    """Words in device memory; what is below 0 counts as 0, what is above the bound as the bound."""
    return [p for p in (-3, 0, 1, 31, 32, 33, 95, 96, 97, 320, 352, 1024, 3104) if p <= bound] + [bound, bound + 500]


def unwritten(dev, n_q):
    return torch.full((n_q, D), math.nan, dtype=BF16, device=dev), torch.full((n_q, D), math.nan, device=dev)


def workspaces(dev, n_q, msl, splits):
    """Enough, never cleared; none, where the call may do without."""
    return [torch.full((ops.workspace_bytes(n_q, D, msl) // 4 + n_q * 528 * 70 // 4 + 4,), math.nan, device=dev)] + ([None] if splits < 2 else [])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("bound", BOUNDS)
def test_steps(dev, bound, n_q, n_kv, fmt):
    g = torch.Generator().manual_seed(bound + n_q)
    msl = bound + 1
    sin, cos = (x.to(dev) for x in C.tables(msl))
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    q, k, v = (x.to(dev) for x in torch.randn((n_q + 2 * n_kv) * D, generator=g).to(BF16).split([n_q * D, n_kv * D, n_kv * D]))
    dims = dict(layer_id=0, kv_dim=n_kv * D, head_num=n_q, head_dim=D, max_seq_len=msl, kv8_format=fmt)
    for word in positions(bound):
        at = max(0, min(word, bound))
        cache = C.filled(1, n_kv, msl, at, fmt, at + n_q)[0].to(dev)
        filed, normed = cache.clone(), torch.zeros(1, n_q * D, dtype=BF16, device=dev)
        ops.qk_norm_rope_append_kv8(normed, k[None], v[None], filed, w, sin, cos, row_num=1, query_src=q[None], pos=at, **dims)
        kc, ks, vc, vs = C.unpack(filed.cpu())
        keys, values = (C.stands_for(c, s, fmt)[0, :, :at + 1] for c, s in ((kc, ks), (vc, vs)))
        want = C.attention(normed.cpu().view(n_q, D), keys, values)
        word = torch.tensor([word], dtype=torch.int32, device=dev)
        for splits in SPLITS:
            for ws in workspaces(dev, n_q, msl, splits):
                out, tap = unwritten(dev, n_q)
                mine = cache.clone()
                ops.mha_decode_append_kv8(q, k, v, w, sin, cos, mine, out, ws, output_f32=tap, pos=bound, pos_device=word, kv_mul=n_q // n_kv, num_splits=splits, **dims)
                C.close(tap.cpu(), *want, rounded=out.cpu())
                assert torch.equal(tap.to(BF16), out) and torch.equal(mine, filed), (at, splits)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("bound", BOUNDS)
def test_attention(dev, bound, n_q, n_kv, fmt):
    g = torch.Generator().manual_seed(bound * 3 + n_q)
    msl = bound + 1
    q = C.rows(g, n_q, outliers=False)
    for word in positions(bound):
        at = max(0, min(word, bound))
        cache, k, v = C.filled(1, n_kv, msl, at + 1, fmt, at + n_q)
        cache, want = cache.to(dev), C.attention(q, k[0], v[0])
        word = torch.tensor([word], dtype=torch.int32, device=dev)
        for splits in SPLITS:
            for ws in workspaces(dev, n_q, msl, splits):
                out, tap = unwritten(dev, n_q)
                ops.mha_decode_kv8(q.to(dev), cache, out, ws, output_f32=tap, layer_id=0, pos=bound, pos_device=word, kv_dim=n_kv * D, kv_mul=n_q // n_kv, head_num=n_q, head_dim=D,
                                   max_seq_len=msl, kv8_format=fmt, num_splits=splits)
                C.close(tap.cpu(), *want, rounded=out.cpu())
                assert torch.equal(tap.to(BF16), out), (at, splits)


@pytest.mark.parametrize("splits", [0, 1, 3])
def test_a_captured_step_from_the_first_token_on(dev, splits):
    """A step captured once, replayed from position 0 on with other work between the replays: every replay against the call with the position on the host."""
    n_q, n_kv, msl = 8, 2, 80
    g = torch.Generator().manual_seed(splits)
    cache = C.garbage(1, n_kv, msl, 3)
    eager, graphed = cache.to(dev), cache.to(dev)
    sin, cos = (x.to(dev) for x in C.tables(msl))
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    x = torch.zeros((n_q + 2 * n_kv) * D, dtype=BF16, device=dev)
    q, k, v = x.split([n_q * D, n_kv * D, n_kv * D])
    word, ws = torch.zeros(1, dtype=torch.int32, device=dev), torch.full((n_q * 528 * 4,), math.nan, device=dev)
    dims = dict(layer_id=0, kv_dim=n_kv * D, kv_mul=n_q // n_kv, head_num=n_q, head_dim=D, max_seq_len=msl, num_splits=splits)
    out, tap = unwritten(dev, n_q)

    def step(buffer):
        ops.mha_decode_append_kv8(q, k, v, w, sin, cos, buffer, out, ws, output_f32=tap, pos=msl - 1, pos_device=word, **dims)

    step(graphed.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed)
    for pos in range(msl):
        x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        word.fill_(pos)
        out.fill_(math.nan), tap.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        normed = torch.zeros(1, n_q * D, dtype=BF16, device=dev)
        ops.qk_norm_rope_append_kv8(normed, k[None], v[None], eager, w, sin, cos, row_num=1, query_src=q[None], layer_id=0, pos=pos, kv_dim=n_kv * D, head_num=n_q, head_dim=D, max_seq_len=msl)
        kc, ks, vc, vs = C.unpack(eager.cpu())
        keys, values = (C.stands_for(c, s, C.E4M3)[0, :, :pos + 1] for c, s in ((kc, ks), (vc, vs)))
        C.close(tap.cpu(), *C.attention(normed.cpu().view(n_q, D), keys, values), rounded=out.cpu())
        assert torch.equal(eager, graphed), pos


@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("keys,splits", [(200, 2), (200, 4), (310, 10), (330, 10), (600, 3), (4000, 70), (4000, 256), (9000, 200)])
def test_a_chosen_number_is_the_same_on_both_sides(dev, keys, splits, n_q, n_kv):
    """The position on the device or on the host: a chosen number of splits deals the records alike, so sums of the same order, the same bits."""
    g = torch.Generator().manual_seed(keys + splits)
    cache = C.filled(1, n_kv, keys + 1, keys, C.E4M3, keys)[0].to(dev)
    q = C.rows(g, n_q, outliers=False).to(dev)
    x = torch.randn((n_q + 2 * n_kv) * D, generator=g).to(BF16).to(dev).split([n_q * D, n_kv * D, n_kv * D])
    w, (sin, cos) = torch.ones(2 * D, dtype=BF16, device=dev), (y.to(dev) for y in C.tables(keys + 1))
    ws = torch.full((n_q * 132 * splits + 4,), math.nan, device=dev)
    dims = dict(layer_id=0, kv_dim=n_kv * D, kv_mul=n_q // n_kv, head_num=n_q, head_dim=D, max_seq_len=keys + 1, num_splits=splits)
    taps = []
    for where in (dict(pos=keys - 1), dict(pos=keys - 1, pos_device=torch.tensor([keys - 1], dtype=torch.int32, device=dev))):
        out, tap = unwritten(dev, n_q)
        ops.mha_decode_kv8(q, cache, out, ws, output_f32=tap, **where, **dims)
        out2, tap2 = unwritten(dev, n_q)
        where = {n: y + 1 for n, y in where.items()}
        ops.mha_decode_append_kv8(*x, w, sin, cos, cache.clone(), out2, ws, output_f32=tap2, **where, **dims)
        taps.append((tap, tap2))
    assert bool(torch.isfinite(taps[0][0]).all()) and bool(torch.isfinite(taps[0][1]).all())
    assert torch.equal(taps[0][0], taps[1][0]) and torch.equal(taps[0][1], taps[1][1])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n_q,n_kv", [(64, 64), (130, 65), (130, 130)])
def test_many_kv_heads(dev, n_q, n_kv, fmt):
    """More KV heads than a chip has workgroups for four each: one workgroup where fewer heads have slices. Steps with the position on the host and on the device."""
    g = torch.Generator().manual_seed(n_q)
    bound = 1300
    msl = bound + 1
    sin, cos = (x.to(dev) for x in C.tables(msl))
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    q, k, v = (x.to(dev) for x in torch.randn((n_q + 2 * n_kv) * D, generator=g).to(BF16).split([n_q * D, n_kv * D, n_kv * D]))
    ws = torch.full((ops.workspace_bytes(n_q, D, msl) // 4,), math.nan, device=dev)
    dims = dict(layer_id=0, kv_dim=n_kv * D, head_num=n_q, head_dim=D, max_seq_len=msl, kv8_format=fmt)
    full = C.filled(1, n_kv, msl, bound, fmt, n_q)[0].to(dev)
    for at in (0, 1, 40, 384, 385, 576, 577, bound):
        filed, normed = full.clone(), torch.zeros(1, n_q * D, dtype=BF16, device=dev)
        ops.qk_norm_rope_append_kv8(normed, k[None], v[None], filed, w, sin, cos, row_num=1, query_src=q[None], pos=at, **dims)
        kc, ks, vc, vs = C.unpack(filed.cpu())
        keys, values = (C.stands_for(c, s, fmt)[0, :, :at + 1] for c, s in ((kc, ks), (vc, vs)))
        want = C.attention(normed.cpu().view(n_q, D), keys, values)
        for where in (dict(pos=at), dict(pos=bound, pos_device=torch.tensor([at], dtype=torch.int32, device=dev))):
            out, tap = unwritten(dev, n_q)
            mine = full.clone()
            ops.mha_decode_append_kv8(q, k, v, w, sin, cos, mine, out, ws, output_f32=tap, kv_mul=n_q // n_kv, **where, **dims)
            C.close(tap.cpu(), *want, rounded=out.cpu())
            assert torch.equal(mine, filed)
            out, tap = unwritten(dev, n_q)
            ops.mha_decode_kv8(normed.view(-1), filed, out, ws, output_f32=tap, kv_mul=n_q // n_kv, **where, **dims)
            C.close(tap.cpu(), *want, rounded=out.cpu())
