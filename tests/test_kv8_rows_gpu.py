"""What fills an 8-bit KV cache and reads it back, against the definition in 64 bits (kv8_cases)."""
import math

import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

import kv8_cases as C

pytestmark = pytest.mark.gpu
D, BF16 = C.D, C.BF16
FORMATS = [C.E4M3, C.INT8]
LAYOUTS = [B.KV_LAYOUT_POS_MAJOR, B.KV_LAYOUT_HEAD_MAJOR]


def laid_out(x, layout):
    """[layers][KV heads][positions][128] as the cache of that layout has it."""
    return (x.transpose(1, 2) if layout == B.KV_LAYOUT_POS_MAJOR else x).contiguous()


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def special_rows(gen, *shape):
    """Rows as they come, and among them rows of zeros, of one value, with infinities or NaN, of the smallest and the largest numbers."""
    x = C.rows(gen, *shape)
    flat = x.view(-1, D)
    n = flat.shape[0]
    odd = [torch.zeros(D), torch.full((D,), -0.0), torch.full((D,), 3.5), torch.full((D,), 1e-40), torch.full((D,), 2.0 ** -60), torch.full((D,), 3.3e38), torch.randn(D) * 1e-19,
           torch.where(torch.arange(D) == 77, math.inf, 1.0), torch.where(torch.arange(D) == 0, -math.inf, 1.0), torch.where(torch.arange(D) == 127, math.nan, 1.0),
           torch.where(torch.arange(D) == 5, 1.0, 1e-30), torch.arange(D) - 63.5, 2.0 ** (torch.arange(D) / 8.0 - 8.0)]
    for i, row in enumerate(odd):
        flat[(i * 7919 + 3) % n] = row.to(BF16)
    return x


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layers,heads,msl,first,count", [
    (1, 1, 1, 0, 1), (1, 1, 32, 0, 32), (2, 3, 40, 0, 40), (2, 3, 70, 5, 20), (1, 8, 200, 31, 2), (3, 2, 100, 32, 33), (1, 5, 129, 64, 65), (2, 1, 97, 96, 1), (1, 2, 300, 17, 280),
])
def test_store_and_load(dev, layers, heads, msl, first, count, fmt, layout):
    g = torch.Generator().manual_seed(msl + 7 * first + count)
    k, v = special_rows(g, layers, heads, msl), special_rows(g, layers, heads, msl)
    cache = C.garbage(layers, heads, msl, 5)
    kc, ks, vc, vs = C.unpack(cache)
    end = first + count
    for rows, codes, scale in ((k, kc, ks), (v, vc, vs)):
        codes[:, :, first:end], scale[:, :, first:end] = C.quantise(rows[:, :, first:end], fmt)
    want = C.pack(kc, ks, vc, vs)
    dims = dict(layer_num=layers, first_pos=first, num_pos=count, kv_dim=heads * D, head_dim=D, max_seq_len=msl, kv_layout=layout, kv8_format=fmt)
    got = cache.to(dev)
    assert ops.kv8_bytes(layers, msl, heads * D, D) == got.numel()
    k_dev, v_dev = laid_out(k, layout).to(dev), laid_out(v, layout).to(dev)
    assert ops.kv8_store(k_dev, v_dev, got, **dims) is got
    assert same_bits(k_dev.cpu(), laid_out(k, layout)) and same_bits(v_dev.cpu(), laid_out(v, layout))
    for a, b, what in zip(C.unpack(got.cpu()), (kc, ks, vc, vs), ("K codes", "K scales", "V codes", "V scales")):
        if "scales" in what:
            a, b = torch.where(torch.isnan(a), 0x7FC0, a.view(torch.int16)), torch.where(torch.isnan(b), 0x7FC0, b.view(torch.int16))
            # (of the places that are not written the bits themselves)
            assert torch.equal(a, b), what
        else:
            assert torch.equal(a, b), what
    outside = torch.ones(got.shape[2] * 32, dtype=torch.bool)
    outside[first:end] = False
    for a, b in zip(C.unpack(got.cpu()), C.unpack(cache)):
        assert same_bits(a[:, :, outside], b[:, :, outside])
    # ... and back, into caches that hold something else
    back = [torch.full_like(x, 7.0) for x in (k_dev, v_dev)]
    stored = want.to(dev)
    assert ops.kv8_load(stored, back[0], back[1], **dims) is None
    assert same_bits(stored.cpu(), want)
    for x, codes, scale in ((back[0], kc, ks), (back[1], vc, vs)):
        ref = torch.full((layers, heads, msl, D), 7.0, dtype=BF16)
        ref[:, :, first:end] = C.stands_for(codes, scale, fmt)[:, :, first:end].float().to(BF16)  # (eight bits times eight: fp32 holds them)
        assert torch.equal(torch.nan_to_num(x.cpu().float(), nan=1e30), torch.nan_to_num(laid_out(ref, layout).float(), nan=1e30))


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_code(dev, fmt):
    """All 256 codes, those that the store never makes too, with scales of 1 and of 0.75."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(16).view(1, 1, 32, D)
    scale = torch.where(torch.arange(32) % 2 == 0, 1.0, 0.75).to(BF16).view(1, 1, 32)
    cache = C.pack(codes, scale, codes, scale).to(dev)
    k, v = torch.zeros(1, 1, 32, D, dtype=BF16, device=dev), torch.zeros(1, 1, 32, D, dtype=BF16, device=dev)
    ops.kv8_load(cache, k, v, layer_num=1, num_pos=32, kv_dim=D, head_dim=D, max_seq_len=32, kv_layout=1, kv8_format=fmt)
    ref = torch.nan_to_num(C.stands_for(codes, scale, fmt).to(BF16).float(), nan=1e30)
    for x in (k, v):
        assert torch.equal(torch.nan_to_num(x.cpu().float(), nan=1e30), ref)


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_quotient(dev, fmt):
    """Every significand over every scale: rows whose largest value fixes the scale, with all 128 significands at each of several magnitudes below it."""
    significand = (128 + torch.arange(128)).float() / 128
    lines = []
    for top in range(128):
        for shift in range(0, 18):
            x = significand * 2.0 ** -shift
            x[0] = (128 + top) / 128 * 2.0
            lines.append(x)
    rows = torch.stack(lines).to(BF16)
    n = rows.shape[0]
    k = rows.view(1, 1, n, D)
    cache = torch.zeros(1, 1, C.records(n), C.RECORD, dtype=torch.uint8, device=dev)
    ops.kv8_store(k.to(dev), (-k).to(dev), cache, layer_num=1, num_pos=n, kv_dim=D, head_dim=D, max_seq_len=n, kv_layout=1, kv8_format=fmt)
    kc, ks, vc, vs = C.unpack(cache.cpu())
    for codes, scale, x in ((kc, ks, k), (vc, vs, -k)):
        want = C.quantise(x, fmt)
        assert torch.equal(codes[:, :, :n], want[0]) and torch.equal(scale[:, :, :n], want[1])


def appended(dev, n_q, n_kv, msl, pos, n, fmt, *, seed=1, inplace=False, device_pos=None, layers=2, layer=1, wide=False):
    """A call's inputs and results, with the oracle's."""
    g = torch.Generator().manual_seed(seed)
    packed = torch.randn(n, (n_q + 2 * n_kv) * D + (40 if wide else 0), generator=g).to(BF16).to(dev)
    q, k, v = packed[:, :n_q * D], packed[:, n_q * D:(n_q + n_kv) * D], packed[:, (n_q + n_kv) * D:(n_q + 2 * n_kv) * D]
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16)
    sin, cos = C.tables(msl)
    before = C.garbage(layers, n_kv, msl, seed + 1)
    cache = before.to(dev)
    at = pos if device_pos is None else max(0, min(device_pos, pos))
    src = q.clone()
    out = q if inplace else torch.zeros(n, n_q * D, dtype=BF16, device=dev)
    word = None if device_pos is None else torch.tensor([device_pos], dtype=torch.int32, device=dev)
    r = ops.qk_norm_rope_append_kv8(out, k, v, cache, w.to(dev), sin.to(dev), cos.to(dev), row_num=n, layer_id=layer, pos=pos, kv_dim=n_kv * D, head_num=n_q, head_dim=D,
                                    max_seq_len=msl, kv8_format=fmt, query_src=None if inplace else q, pos_device=word)
    assert r is None
    s, c = sin[at:at + n], cos[at:at + n]
    ref = dict(q=C.normed(src.cpu().reshape(n, n_q, D), w[:D], s, c), k=C.normed(k.cpu().reshape(n, n_kv, D), w[D:], s, c), v=v.cpu().reshape(n, n_kv, D))
    return out.cpu().reshape(n, n_q, D), cache.cpu(), before, at, ref


CASES = [(1, 1, 1, 0, 1), (16, 8, 64, 5, 1), (32, 8, 300, 31, 2), (64, 8, 100, 33, 64), (5, 5, 130, 0, 130), (40, 8, 90, 60, 30), (33, 3, 70, 69, 1), (4, 2, 2000, 3, 1900)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n_q,n_kv,msl,pos,n", CASES)
def test_rows_of_new_tokens(dev, n_q, n_kv, msl, pos, n, fmt):
    out, cache, before, at, ref = appended(dev, n_q, n_kv, msl, pos, n, fmt, seed=n_q + n)
    # fp32 arithmetic of some thirty roundings in front of bf16's
    assert bool(((out.double() - ref["q"]).abs() <= 2.0 ** -8 * ref["q"].abs() + 1e-5).all())
    kc, ks, vc, vs = C.unpack(cache)
    # V is quantised as it came: the bits. K: its bf16 value may be the neighbouring one where fp32 decides; then codes and scales follow
    codes, scale = C.quantise(ref["v"].transpose(0, 1), fmt)
    assert torch.equal(vc[1, :, at:at + n], codes) and torch.equal(vs[1, :, at:at + n], scale)
    got = C.stands_for(kc[1, :, at:at + n], ks[1, :, at:at + n], fmt)
    want = ref["k"].transpose(0, 1)
    top = want.abs().amax(-1, keepdim=True)
    half = top / 127 * 0.5 if fmt == C.INT8 else torch.maximum(want.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10)
    # half a step of the code (the scale, rounded up, is 2^-7 larger at most), half a step of bf16, fp32's
    assert bool(((got - want).abs() <= half * (1 + 2.0 ** -6) + (2.0 ** -8 + 2.0 ** -12) * want.abs() + 1e-5).all())
    for a, b in zip(C.unpack(cache), C.unpack(before)):
        keep = torch.ones(a.shape[:3], dtype=torch.bool)
        keep[1, :, at:at + n] = False
        assert same_bits(a[keep], b[keep])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads", [(32, 8), (10, 2), (16, 1)])
def test_k_rows_are_the_bf16_cache_s_quantised(dev, heads, fmt):
    """The same bits as a bf16 append by mha_decode_append whose row is stored in 8 bits afterwards."""
    n_q, n_kv = heads
    g = torch.Generator().manual_seed(n_q)
    msl = 80
    sin, cos = (x.to(dev) for x in C.tables(msl))
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    kc, vc = torch.zeros(1, n_kv, msl, D, dtype=BF16, device=dev), torch.zeros(1, n_kv, msl, D, dtype=BF16, device=dev)
    two, one = (torch.zeros(1, n_kv, C.records(msl), C.RECORD, dtype=torch.uint8, device=dev) for _ in range(2))
    ws, out, q_out = torch.zeros(1 << 20, device=dev), torch.zeros(n_q * D, dtype=BF16, device=dev), torch.zeros(1, n_q * D, dtype=BF16, device=dev)
    dims = dict(kv_dim=n_kv * D, head_dim=D, max_seq_len=msl)
    for pos in range(40):
        x = torch.randn((n_q + 2 * n_kv) * D, generator=g).to(BF16).to(dev)
        q, k, v = x.split([n_q * D, n_kv * D, n_kv * D])
        ops.mha_decode_append(q, k, v, w, sin, cos, kc, vc, out, ws, layer_id=0, pos=pos, kv_mul=n_q // n_kv, head_num=n_q, kv_layout=1, **dims)
        ops.qk_norm_rope_append_kv8(q_out, k[None], v[None], one, w, sin, cos, row_num=1, layer_id=0, pos=pos, head_num=n_q, query_src=q[None], kv8_format=fmt, **dims)
    ops.kv8_store(kc, vc, two, layer_num=1, num_pos=40, kv_layout=1, kv8_format=fmt, **dims)
    assert torch.equal(one.cpu(), two.cpu())


@pytest.mark.parametrize("how", [dict(inplace=True), dict(wide=True), dict(device_pos=3), dict(device_pos=-4), dict(device_pos=1000), dict(inplace=True, wide=True, device_pos=20)])
def test_rows_in_place_from_slices_and_at_a_position_on_the_device(dev, how):
    out, cache, before, at, ref = appended(dev, 16, 8, 90, 40, 33, C.E4M3, **how)
    assert bool(((out.double() - ref["q"]).abs() <= 2.0 ** -8 * ref["q"].abs() + 1e-5).all())
    kc, ks, vc, vs = C.unpack(cache)
    codes, scale = C.quantise(ref["v"].transpose(0, 1), C.E4M3)
    assert torch.equal(vc[1, :, at:at + 33], codes) and torch.equal(vs[1, :, at:at + 33], scale)
    keep = torch.ones(2, 8, kc.shape[2], dtype=torch.bool)
    keep[1, :, at:at + 33] = False
    for a, b in zip(C.unpack(cache), C.unpack(before)):
        assert same_bits(a[keep], b[keep])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("pos,n,how", [
    (0, 384, {}), (17, 500, dict(inplace=True)), (100, 449, dict(wide=True)), (64, 1001, dict(device_pos=31)), (64, 385, dict(device_pos=64)), (90, 416, dict(device_pos=-7)),
    (31, 386, dict(device_pos=500)), (1, 383, {}), (5, 383, dict(device_pos=2)),
])
def test_rows_of_many_tokens(dev, pos, n, how, fmt):
    """From some hundred tokens on records are put together by workgroups: the same bits as token by token, whole and at the edges."""
    n_q, n_kv, msl = 12, 3, pos + n + 3
    out, cache, before, at, ref = appended(dev, n_q, n_kv, msl, pos, n, fmt, seed=n, **how)
    assert bool(((out.double() - ref["q"]).abs() <= 2.0 ** -8 * ref["q"].abs() + 1e-5).all())
    kc, ks, vc, vs = C.unpack(cache)
    codes, scale = C.quantise(ref["v"].transpose(0, 1), fmt)
    assert torch.equal(vc[1, :, at:at + n], codes) and torch.equal(vs[1, :, at:at + n], scale)
    keep = torch.ones(2, n_kv, kc.shape[2], dtype=torch.bool)
    keep[1, :, at:at + n] = False
    for a, b in zip(C.unpack(cache), C.unpack(before)):
        assert same_bits(a[keep], b[keep])
    # the same tokens in calls of a few
    g = torch.Generator().manual_seed(n)
    packed = torch.randn(n, (n_q + 2 * n_kv) * D + (40 if how.get("wide") else 0), generator=g).to(BF16).to(dev)
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    sin, cos = (x.to(dev) for x in C.tables(msl))
    few, q_few = before.to(dev), torch.zeros(n, n_q * D, dtype=BF16, device=dev)
    for i in range(0, n, 100):
        rows = packed[i:i + 100]
        q, k, v = rows[:, :n_q * D], rows[:, n_q * D:(n_q + n_kv) * D], rows[:, (n_q + n_kv) * D:(n_q + 2 * n_kv) * D]
        ops.qk_norm_rope_append_kv8(q_few[i:i + 100], k, v, few, w, sin, cos, row_num=rows.shape[0], layer_id=1, pos=at + i, kv_dim=n_kv * D, head_num=n_q, head_dim=D,
                                    max_seq_len=msl, kv8_format=fmt, query_src=q)
    assert torch.equal(few.cpu(), cache) and torch.equal(q_few.cpu().view(n, n_q, D), out)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n", [5, 400])
def test_captured_on_a_side_stream(dev, n, fmt):
    """A range stored, rows filed behind it at a position on the device, both read back: one graph, replayed with other inputs and positions, other work between."""
    n_q, n_kv, msl = 6, 3, 900
    g = torch.Generator().manual_seed(n)
    dims = dict(kv_dim=n_kv * D, head_dim=D, max_seq_len=msl, kv8_format=fmt)
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16).to(dev)
    sin, cos = (x.to(dev) for x in C.tables(msl))
    kc, vc = (torch.zeros(2, msl, n_kv * D, dtype=BF16, device=dev) for _ in range(2))
    packed, word = torch.zeros(n, (n_q + 2 * n_kv) * D, dtype=BF16, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)

    def buffers():
        cache = torch.zeros(ops.kv8_bytes(2, msl, n_kv * D, D), dtype=torch.uint8, device=dev)
        return cache, torch.zeros(n, n_q * D, dtype=BF16, device=dev), torch.zeros_like(kc), torch.zeros_like(vc)

    def call(cache, q, k_back, v_back, bound, at):
        rows = packed.split([n_q * D, n_kv * D, n_kv * D], dim=1)
        ops.kv8_store(kc, vc, cache, layer_num=2, num_pos=77, **dims)
        ops.qk_norm_rope_append_kv8(q, rows[1], rows[2], cache, w, sin, cos, row_num=n, layer_id=1, pos=bound, head_num=n_q, query_src=rows[0], pos_device=at, **dims)
        ops.kv8_load(cache, k_back, v_back, layer_num=2, num_pos=msl, **dims)

    mine = buffers()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call(*mine, msl - n, word)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(*mine, msl - n, word)
    for at in (77, 0, 31, 450, msl - n):
        for x in (kc, vc, packed):
            x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        word.fill_(at)
        for x in mine:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = buffers()
        call(*want, at, None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(mine, want)), at


def test_what_the_front_end_refuses(dev):
    u8 = torch.zeros(2 * 8320, dtype=torch.uint8, device=dev)
    x = torch.zeros(64, D, dtype=BF16, device=dev)
    tab = torch.zeros(64, 64, device=dev)
    dims = dict(kv_dim=D, head_dim=D, max_seq_len=64)
    copy = dict(layer_num=1, num_pos=4, **dims)
    ops.kv8_store(x, x, u8, **copy)
    for args, message in (((x, x, u8[:-1]), "cache8 has 16639 elements"), ((x[:63], x, u8), "key_cache has 8064"), ((x, x.float(), u8), "value_cache has dtype"),
                          ((x, x, u8.view(torch.int8)), "cache8 has dtype"), ((x, x, u8.cpu()), "cache8 must be a device tensor")):
        with pytest.raises(ValueError, match=message):
            ops.kv8_store(*args, **copy)
        with pytest.raises(ValueError, match=message):
            ops.kv8_load(args[2], args[0], args[1], **copy)
    with pytest.raises(B.LlmiError, match="pos"):
        ops.kv8_store(x, x, u8, **dict(copy, first_pos=61))
    for layers, msl in (((1 << 31) - 1, (1 << 31) - 1), ((1 << 31) - 1, 1 << 26)):
        with pytest.raises(ValueError, match="has .* elements"):
            ops.kv8_load(u8, x, x, **dict(copy, layer_num=layers, max_seq_len=msl))
    rows = dict(row_num=2, layer_id=0, pos=0, head_num=1, **dims)
    with pytest.raises(ValueError, match="cache8 has"):
        ops.qk_norm_rope_append_kv8(x, x, x, u8, x, tab, tab, **dict(rows, layer_id=1))
    with pytest.raises(ValueError, match="sin_cache has"):
        ops.qk_norm_rope_append_kv8(x, x, x, u8, x, tab[:3], tab, **rows)
    with pytest.raises(ValueError, match=r"key_new must be \[70\]\[128\]"):
        ops.qk_norm_rope_append_kv8(x.repeat(2, 1), x, x, u8, x, tab, tab, **dict(rows, row_num=70))
    with pytest.raises(TypeError, match="missing required argument: 'row_num'"):
        ops.qk_norm_rope_append_kv8(x, x, x, u8, x, tab, tab, layer_id=0, pos=0, head_num=1, **dims)
    decode = dict(layer_id=0, pos=3, kv_mul=1, head_num=1, **dims)
    with pytest.raises(ValueError, match="output has 100 elements"):
        ops.mha_decode_kv8(x, u8, x.view(-1)[:100], None, **decode)
    with pytest.raises(ValueError, match="cache8 has"):
        ops.mha_decode_kv8(x, u8, x, None, **dict(decode, layer_id=1))
    with pytest.raises(ValueError, match="key_new has 64"):
        ops.mha_decode_append_kv8(x, x.view(-1)[:64], x, x, tab, tab, u8, x, None, **decode)
