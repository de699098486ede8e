"""llmi_hip_qk_norm_rope_append_tree and llmi_hip_kv_commit_tree on the device: the first against llmi_hip_qk_norm_rope_append row by row
(same bits) and against the formula in 64 bits, the second as the copy it is."""
import ctypes

import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

from tree_cases import D, depths_of, parents_of, rows

pytestmark = pytest.mark.gpu

HEAD, POS = B.KV_LAYOUT_HEAD_MAJOR, B.KV_LAYOUT_POS_MAJOR


def cache(dev, layers, msl, n_kv, layout, seed):
    return rows(seed, *((layers, msl, n_kv, D) if layout == POS else (layers, n_kv, msl, D)), dev=dev)


def slots(c, layout):
    """[layers][position][KV head][128], a view."""
    return c if layout == POS else c.transpose(1, 2)


@pytest.mark.parametrize("layout", [POS, HEAD])
@pytest.mark.parametrize("n,n_q,n_kv,pos,kind", [(1, 16, 8, 0, "chain"), (5, 32, 8, 100, "chain"), (26, 32, 8, 37, "tree"), (64, 64, 8, 300, "tree"),
                                                 (64, 8, 1, 1, "star"), (7, 40, 8, 250, "tree"), (3, 24, 3, 9, "tree")])
def test_append(dev, layout, n, n_q, n_kv, pos, kind):
    msl, dim, kv_dim = pos + n + 2, n_q * D, n_kv * D
    depth = depths_of(parents_of(n, n, kind))
    packed = rows(1, n + 1, dim + 2 * kv_dim, dev=dev, unit=False)  # a node's query, key and value behind one another
    q, k, v = packed.split([dim, kv_dim, kv_dim], dim=1)
    w = (1 + 0.1 * torch.randn(2 * D, device=dev)).to(torch.bfloat16)
    sin, cos = ops.sincos_table(D, msl, dev)
    kc, vc = cache(dev, 2, msl, n_kv, layout, 2), cache(dev, 2, msl, n_kv, layout, 3)
    common = dict(layer_id=1, kv_dim=kv_dim, head_num=n_q, head_dim=D, max_seq_len=msl, kv_layout=layout)
    # row by row: a cache of its own for each, its slot the position the node is rotated for
    want_q, want_k, want_v = torch.zeros(n, dim, dtype=torch.bfloat16, device=dev), kc.clone(), vc.clone()
    for i in range(n):
        k1, v1, row = kc.clone(), vc.clone(), torch.zeros(dim, dtype=torch.bfloat16, device=dev)
        ops.qk_norm_rope_append(row, k[i].contiguous(), v[i].contiguous(), k1, v1, w, sin, cos, pos=pos + depth[i], query_src=q[i].contiguous(), **common)
        want_q[i] = row
        slots(want_k, layout)[1, pos + i] = slots(k1, layout)[1, pos + depth[i]]
        slots(want_v, layout)[1, pos + i] = v[i].view(n_kv, D)
    depth_t = torch.tensor(depth, dtype=torch.int32, device=dev)
    got_k, got_v = kc.clone(), vc.clone()
    out = torch.full((n + 1, dim + 8), 7.0, dtype=torch.bfloat16, device=dev)
    ops.qk_norm_rope_append_tree(out[:n, :dim], k[:n], v[:n], got_k, got_v, w, sin, cos, node_num=n, depth=depth_t, pos=pos, query_src=q[:n], **common)
    torch.cuda.synchronize()
    assert torch.equal(out[:n, :dim], want_q) and torch.equal(got_k, want_k) and torch.equal(got_v, want_v)
    assert bool((out[n] == 7).all()) and bool((out[:, dim:] == 7).all())
    # against the formula: the arithmetic's few fp32 steps (under 16 roundings of 2^-24 on |a| + |b|) and half a bf16 step
    at = torch.tensor([pos + d for d in depth], device=dev)
    for got, raw, weight in ((out[:n, :dim], q[:n], w[:D]), (slots(got_k, layout)[1, pos:pos + n], k[:n], w[D:])):
        x = raw.reshape(n, -1, D).double()
        y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
        a, b, s, c = y[..., :64], y[..., 64:], sin[at].double()[:, None], cos[at].double()[:, None]
        want = torch.cat([a * c - b * s, a * s + b * c], -1)
        size = torch.cat([a.abs() + b.abs()] * 2, -1)
        off = (got.reshape(n, -1, D).double() - want).abs()
        assert bool((off <= 2.0 ** -8 * want.abs() + 16 * 2.0 ** -24 * size).all())
    # in place, chain by default, position on the device
    if kind == "chain":
        k2, v2, q2 = kc.clone(), vc.clone(), q[:n].contiguous()
        word = torch.full((1,), pos, dtype=torch.int32, device=dev)
        ops.qk_norm_rope_append_tree(q2, k[:n], v[:n], k2, v2, w, sin, cos, node_num=n, pos=msl - n, pos_device=word, **common)
        torch.cuda.synchronize()
        assert torch.equal(q2, want_q) and torch.equal(k2, want_k) and torch.equal(v2, want_v)


def test_append_in_place(dev):
    """key_new and value_new in the slots themselves: what the projection of the reference's layer loop leaves there."""
    n, n_kv, pos, msl = 6, 8, 30, 40
    kc, vc = cache(dev, 1, msl, n_kv, POS, 5), cache(dev, 1, msl, n_kv, POS, 6)
    q, w = rows(7, n, 16 * D, dev=dev), rows(8, 2 * D, dev=dev)
    sin, cos = ops.sincos_table(D, msl, dev)
    kw = dict(node_num=n, layer_id=0, pos=pos, kv_dim=n_kv * D, head_num=16, head_dim=D, max_seq_len=msl, kv_layout=POS)
    k1, v1, q1 = kc.clone(), vc.clone(), q.clone()
    ops.qk_norm_rope_append_tree(q1, kc[0, pos:pos + n].reshape(n, -1).clone(), vc[0, pos:pos + n].reshape(n, -1).clone(), k1, v1, w, sin, cos, **kw)
    k2, v2, q2 = kc.clone(), vc.clone(), q.clone()
    ops.qk_norm_rope_append_tree(q2, k2[0, pos:pos + n].view(n, -1), v2[0, pos:pos + n].view(n, -1), k2, v2, w, sin, cos, **kw)
    torch.cuda.synchronize()
    assert torch.equal(k1, k2) and torch.equal(v1, v2) and torch.equal(q1, q2)
    assert not torch.equal(k1, kc)


@pytest.mark.parametrize("depth", [-5, 10000, (1 << 31) - 1, -(1 << 31)])
def test_depths_outside_the_tables(dev, depth):
    """Held within them: nothing else is read."""
    n, msl, pos = 2, 64, 40
    q, k, w = rows(1, n, 8 * D, dev=dev), rows(2, n, 8 * D, dev=dev), rows(3, 2 * D, dev=dev)
    tables = [torch.full((3 * msl, 64), float("nan"), device=dev) for _ in range(2)]
    sin, cos = (t[msl:2 * msl] for t in tables)
    sin.copy_(ops.sincos_table(D, msl, dev)[0])
    cos.copy_(ops.sincos_table(D, msl, dev)[1])
    got = []
    for d in (depth, -pos + min(max(pos + depth, 0), msl - 1)):
        kc, vc, out = cache(dev, 1, msl, 8, HEAD, 5), cache(dev, 1, msl, 8, HEAD, 6), q.clone()
        ops.qk_norm_rope_append_tree(out, k, k, kc, vc, w, sin, cos, node_num=n, depth=torch.full((n,), d, dtype=torch.int32, device=dev), layer_id=0,
                                     pos=pos, kv_dim=8 * D, head_num=8, head_dim=D, max_seq_len=msl, kv_layout=HEAD)
        got.append((out, kc))
    torch.cuda.synchronize()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and bool(torch.isfinite(got[0][0]).all())


def commit(c, path, count, n, layout, pos, **over):
    dev = c[0].device
    p = torch.tensor(path + [-1] * (n - len(path)), dtype=torch.int32, device=dev)
    msl = slots(c[0], layout).shape[1]
    n_kv = slots(c[0], layout).shape[2]
    ops.kv_commit_tree(c[0], c[1], p, torch.tensor([count, 5], dtype=torch.int32, device=dev), **dict(dict(
        node_num=n, layer_num=c[0].shape[0], pos=pos, kv_dim=n_kv * D, head_dim=D, max_seq_len=msl, kv_layout=layout), **over))
    torch.cuda.synchronize()


@pytest.mark.parametrize("layout", [POS, HEAD])
@pytest.mark.parametrize("n,path", [(1, [0]), (2, [0, 1]), (8, [0]), (8, [0, 2, 3, 7]), (26, [0, 1, 5, 6, 25]), (64, [0, 63]), (64, list(range(0, 64, 2))),
                                    (64, list(range(64))), (64, [0] + list(range(2, 64))), (40, [0, 3, 4, 9, 10, 11, 17, 30, 31, 39])])
@pytest.mark.parametrize("n_kv,layers,pos", [(8, 3, 21), (1, 2, 0), (3, 1, 5)])
def test_commit(dev, layout, n, path, n_kv, layers, pos):
    msl = pos + n + 3
    c = [cache(dev, layers, msl, n_kv, layout, 30 + i) for i in range(2)]
    want = [x.clone() for x in c]
    for old, new in zip(c, want):
        slots(new, layout)[:, pos:pos + len(path)] = slots(old, layout)[:, [pos + i for i in path]]
    mine = [x.clone() for x in c]
    commit(mine, path, len(path), n, layout, pos)
    assert all(torch.equal(a, b) for a, b in zip(mine, want))
    again = [x.clone() for x in c]  # the position on the device
    commit(again, path, len(path), n, layout, msl - n, pos_device=torch.full((1,), pos, dtype=torch.int32, device=dev))
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_commit_leaves_alone_what_it_cannot_place(dev):
    """Counts and entries out of range move nothing, and nothing beyond the nodes' slots is touched."""
    c = [cache(dev, 2, 40, 8, HEAD, 50 + i) for i in range(2)]
    for path, count in (([0, 3, 5], 0), ([0, 3, 5], -7), ([0, -1, 0, 10, 64, 1 << 30, -(1 << 31)], 7), ([0, 0, 1, 2], 4), ([7, 1, 2, 3], 4)):
        mine = [x.clone() for x in c]
        commit(mine, path, count, 10, HEAD, 20)
        assert all(torch.equal(a, b) for a, b in zip(mine, c)), (path, count)
    want = [x.clone() for x in c]
    for x, old in zip(want, c):
        x[:, :, 21:30] = old[:, :, [20 + i for i in [1] * 1 + [4] + list(range(3, 10))]]
    mine = [x.clone() for x in c]
    commit(mine, [0, 1, 4, 3], 1000, 10, HEAD, 20)  # (a count beyond the nodes stops at them)
    assert all(torch.equal(a, b) for a, b in zip(mine, want))


def test_commit_past_32_bits(dev):
    layers, msl, n_kv, pos = 17, 131072, 8, 131000
    c = [torch.zeros(layers, msl, n_kv, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    block = rows(1, 2, layers, 64, n_kv, D, dev=dev)
    for i in range(2):
        c[i][:, pos:pos + 64] = block[i]
    commit(c, [0, 7, 63], 3, 64, POS, pos)
    want = block.clone()
    want[:, :, 1:3] = block[:, :, [7, 63]]
    for i in range(2):
        assert torch.equal(c[i][:, pos:pos + 64], want[i]) and not bool(c[i][:, pos - 8:pos].any()) and not bool(c[i][:, pos + 64:].any())


def test_the_front_end_refuses(dev):
    kc, vc = cache(dev, 1, 64, 8, HEAD, 1), cache(dev, 1, 64, 8, HEAD, 2)
    q, k, w = rows(1, 4, 16 * D, dev=dev), rows(2, 4, 8 * D, dev=dev), rows(3, 2 * D, dev=dev)
    sin, cos = ops.sincos_table(D, 64, dev)
    kw = dict(node_num=4, layer_id=0, pos=10, kv_dim=8 * D, head_num=16, head_dim=D, max_seq_len=64, kv_layout=HEAD)
    args = dict(query=q, key_new=k, value_new=k, key_cache=kc, value_cache=vc, norm_weight=w, sin_cache=sin, cos_cache=cos)
    for change, error, text in [
            (dict(query=q[:3]), ValueError, "query must be"), (dict(key_new=k[:, :512]), ValueError, "key_new must be"),
            (dict(value_new=k.t()), ValueError, "value_new must be"), (dict(key_cache=kc[:, :4]), ValueError, "key_cache"),
            (dict(value_cache=vc[:, :, :63].contiguous()), ValueError, "value_cache has"), (dict(norm_weight=w[:D]), ValueError, "norm_weight has"),
            (dict(sin_cache=sin[:60]), ValueError, "sin_cache has"), (dict(depth=torch.zeros(3, dtype=torch.int32, device=dev)), ValueError, "depth has"),
            (dict(layer_id=1), ValueError, "key_cache has"), (dict(value_new=None), B.LlmiError, "NULL"), (dict(pos=61), B.LlmiError, "pos out of range"),
            (dict(node_num=0), B.LlmiError, "out of range"), (dict(node_num=65), ValueError, "query must be"),
            (dict(pos_device=torch.zeros(1, dtype=torch.int64, device=dev)), ValueError, "pos_device has dtype")]:
        with pytest.raises(error, match=text):
            ops.qk_norm_rope_append_tree(**dict(dict(args, **kw), **change))
    path, result = torch.zeros(4, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    ckw = dict(node_num=4, layer_num=1, pos=10, kv_dim=8 * D, head_dim=D, max_seq_len=64, kv_layout=HEAD)
    for change, error, text in [
            (dict(path=path[:3]), ValueError, "path has 3"), (dict(layer_num=2), ValueError, "key_cache has"), (dict(result=path.float()), ValueError, "result has dtype"),
            (dict(key_cache=None), B.LlmiError, "NULL"), (dict(pos=61), B.LlmiError, "pos out of range")]:
        with pytest.raises(error, match=text):
            ops.kv_commit_tree(**dict(dict(key_cache=kc, value_cache=vc, path=path, result=result, **ckw), **change))
    ws, out = torch.empty(1 << 20, device=dev), torch.empty_like(q)
    akw = dict(kw, kv_mul=2)
    for change, error, text in [
            (dict(query=q[:3]), ValueError, "query has"), (dict(output=out[:, :100].contiguous()), ValueError, "output has"),
            (dict(tree_mask=torch.zeros(3, dtype=torch.int64, device=dev)), ValueError, "tree_mask has 3"),
            (dict(tree_mask=torch.zeros(4, dtype=torch.int32, device=dev)), ValueError, "tree_mask has dtype"),
            (dict(layer_id=1), ValueError, "key_cache has"), (dict(pos=61), B.LlmiError, "pos out of range"), (dict(kv_mul=3), B.LlmiError, "head_num"),
            (dict(force_path=1), TypeError, "unexpected keyword"), (dict(output_f32=torch.zeros(5, device=dev)), ValueError, "output_f32 has")]:
        with pytest.raises(error, match=text):
            ops.mha_decode_tree(**dict(dict(query=q, key_cache=kc, value_cache=vc, output=out, workspace=ws, **akw), **change))
