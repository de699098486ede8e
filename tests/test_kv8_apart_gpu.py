"""Buffers that lie side by side, cut out of one: the calls for an 8-bit KV cache take them, and write nothing beside what is theirs."""
import pytest
import torch

from llminfer_amd import ops

import kv8_cases as C

pytestmark = pytest.mark.gpu
D, BF16 = C.D, C.BF16


class Slab:
    """One allocation, handed out piece by piece with nothing between."""

    def __init__(self, dev, size):
        self.bytes, self.used = torch.full((size,), 0x5A, dtype=torch.uint8, device=dev), 0

    def take(self, shape, dtype, like=None):
        n = torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()
        assert n % 16 == 0 and self.used + n <= self.bytes.numel()
        x = self.bytes[self.used:self.used + n].view(dtype).view(shape)
        self.used += n
        return x if like is None else x.copy_(like)

    def check(self):
        assert bool((self.bytes[self.used:] == 0x5A).all())


@pytest.mark.parametrize("keys", [70, 3000])
@pytest.mark.parametrize("order", [1, -1])
def test_attention(dev, keys, order):
    n_q, n_kv, msl, splits = 8, 2, keys + 30, 5 if keys > 2000 else 0
    g = torch.Generator().manual_seed(keys)
    cache, k, v = C.filled(2, n_kv, msl, keys, C.E4M3, keys)
    q = C.rows(g, n_q, outliers=False)
    new = torch.randn((n_q + 2 * n_kv) * D, generator=g).to(BF16)
    w = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16)
    sin, cos = C.tables(msl)
    slab = Slab(dev, cache.numel() + n_q * 528 * max(splits, 1) + 4 * msl * D + (1 << 16))
    made = {}
    pieces = [("out", (n_q, D), BF16, None), ("q", (n_q, D), BF16, q), ("tap", (n_q, D), torch.float32, None), ("ws", (n_q * 132 * max(splits, 1),), torch.float32, None),
              ("cache", cache.shape, torch.uint8, cache), ("new", new.shape, BF16, new), ("word", (4,), torch.int32, torch.tensor([keys - 1, 0, 0, 0], dtype=torch.int32)),
              ("out2", (n_q, D), BF16, None), ("w", w.shape, BF16, w), ("sin", sin.shape, torch.float32, sin), ("cos", cos.shape, torch.float32, cos), ("pad", (4,), torch.float32, None)]
    for name, shape, dtype, like in pieces[::order]:
        made[name] = slab.take(shape, dtype, like)
    # (a workspace has 16 bytes more than its partial results take: here they are its neighbour's)
    ws = torch.as_strided(made["ws"], (made["ws"].numel() + 4,), (1,)) if splits else None
    dims = dict(layer_id=1, kv_dim=n_kv * D, kv_mul=n_q // n_kv, head_num=n_q, head_dim=D, max_seq_len=msl, num_splits=splits)
    want = C.attention(q, k[1], v[1])
    for at in (dict(pos=keys - 1), dict(pos=msl - 1, pos_device=made["word"][:1])):
        made["out"].zero_(), made["tap"].zero_()
        ops.mha_decode_kv8(made["q"], made["cache"], made["out"], ws, output_f32=made["tap"], **at, **dims)
        C.close(made["tap"].cpu(), *want, rounded=made["out"].cpu())
    made["word"].fill_(keys)
    parts = made["new"].split([n_q * D, n_kv * D, n_kv * D])
    alone = [x.clone() for x in (*parts, made["w"], made["sin"], made["cos"], made["cache"])]
    out, enough = torch.zeros(n_q, D, dtype=BF16, device=dev), torch.zeros(1 << 18, device=dev)
    ops.mha_decode_append_kv8(*alone, out, enough, pos=keys, **dims)
    for at in (dict(pos=keys), dict(pos=msl - 1, pos_device=made["word"][:1])):
        made["out2"].zero_()
        ops.mha_decode_append_kv8(*parts, made["w"], made["sin"], made["cos"], made["cache"], made["out2"], ws, **at, **dims)
        assert torch.equal(made["cache"], alone[-1])
        if "pos_device" not in at:
            assert torch.equal(made["out2"], out)
    assert torch.equal(made["q"].cpu(), q) and torch.equal(made["new"].cpu(), new) and torch.equal(made["w"].cpu(), w)
    assert torch.equal(made["sin"].cpu(), sin) and torch.equal(made["cos"].cpu(), cos)
    slab.check()


@pytest.mark.parametrize("n", [1, 3, 400])
@pytest.mark.parametrize("how", ["behind", "in place", "named in place", "dense"])
def test_rows(dev, how, n):
    """Query rows in the packed buffer: behind a token's value, in the raw rows' place (told or not), or dense right behind the buffer."""
    n_q, n_kv, msl = 6, 3, n + 50
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, (2 * n_q + 2 * n_kv) * D, generator=g).to(BF16)
    w, (sin, cos) = (1 + 0.1 * torch.randn(2 * D, generator=g)).to(BF16), C.tables(msl)
    cache = C.garbage(2, n_kv, msl, n)
    dims = dict(row_num=n, layer_id=1, pos=20, kv_dim=n_kv * D, head_num=n_q, head_dim=D, max_seq_len=msl)
    alone = [y.to(dev) for y in (x[:, :n_q * D].contiguous(), x[:, n_q * D:(n_q + n_kv) * D].contiguous(), x[:, (n_q + n_kv) * D:(n_q + 2 * n_kv) * D].contiguous(), cache, w, sin, cos)]
    want = torch.zeros(n, n_q * D, dtype=BF16, device=dev)
    ops.qk_norm_rope_append_kv8(want, *alone[1:], query_src=alone[0], **dims)
    slab = Slab(dev, cache.numel() + x.numel() * 4 + 4 * msl * D + (1 << 14))
    cache8, packed = slab.take(cache.shape, torch.uint8, cache), slab.take(x.shape, BF16, x)
    out = slab.take((n, n_q * D), BF16)
    word = slab.take((4,), torch.int32, torch.tensor([20, 0, 0, 0], dtype=torch.int32))
    tables = slab.take(w.shape, BF16, w), slab.take(sin.shape, torch.float32, sin), slab.take(cos.shape, torch.float32, cos)
    raw, k, v, behind = packed.split([n_q * D, n_kv * D, n_kv * D, n_q * D], dim=1)
    query, src = {"behind": (behind, raw), "in place": (raw, None), "named in place": (raw, raw), "dense": (out, raw)}[how]
    ops.qk_norm_rope_append_kv8(query, k, v, cache8, *tables, query_src=src, pos_device=word[:1], **dims)
    assert torch.equal(query, want) and torch.equal(cache8, alone[3])
    kept = x.to(dev)
    assert torch.equal(k, kept[:, n_q * D:(n_q + n_kv) * D]) and torch.equal(v, kept[:, (n_q + n_kv) * D:(n_q + 2 * n_kv) * D])
    if how in ("behind", "dense"):
        assert torch.equal(raw, kept[:, :n_q * D])
    slab.check()


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("order", [1, -1])
def test_copies(dev, order, layout):
    layers, heads, msl = 2, 3, 48
    g = torch.Generator().manual_seed(4)
    k, v = (C.rows(g, layers, heads, msl) for _ in range(2))
    laid = [(x if layout else x.transpose(1, 2)).contiguous() for x in (k, v)]
    slab = Slab(dev, 4 * k.numel() + C.records(msl) * C.RECORD * layers * heads + 64)
    pieces = [("k", laid[0].shape, BF16, laid[0]), ("cache", (layers, heads, C.records(msl), C.RECORD), torch.uint8, C.garbage(layers, heads, msl, 2)), ("v", laid[1].shape, BF16, laid[1])]
    made = {n: slab.take(shape, dtype, like) for n, shape, dtype, like in pieces[::order]}
    dims = dict(layer_num=layers, num_pos=msl, kv_dim=heads * D, head_dim=D, max_seq_len=msl, kv_layout=layout)
    ops.kv8_store(made["k"], made["v"], made["cache"], **dims)
    assert torch.equal(made["k"].cpu(), laid[0]) and torch.equal(made["v"].cpu(), laid[1])
    kc, ks, vc, vs = C.unpack(made["cache"].cpu())
    for codes, scale, rows in ((kc, ks, k), (vc, vs, v)):
        q, s = C.quantise(rows, C.E4M3)
        assert torch.equal(codes[:, :, :msl], q) and torch.equal(scale[:, :, :msl], s)
    keep = made["cache"].clone()
    made["k"].zero_(), made["v"].zero_()
    ops.kv8_load(made["cache"], made["k"], made["v"], **dims)
    assert torch.equal(made["cache"], keep)
    for got, codes, scale in ((made["k"], kc, ks), (made["v"], vc, vs)):
        ref = C.stands_for(codes, scale, C.E4M3)[:, :, :msl].float().to(BF16)
        assert torch.equal(got.cpu(), (ref if layout else ref.transpose(1, 2)).contiguous())
    slab.check()
    # (what is read may be one cache)
    ops.kv8_store(made["k"], made["k"], made["cache"], **dims)
    kc, ks, vc, vs = C.unpack(made["cache"].cpu())
    assert torch.equal(kc[:, :, :msl], vc[:, :, :msl]) and torch.equal(ks[:, :, :msl], vs[:, :, :msl])
