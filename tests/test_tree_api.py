"""The C ABI's calls for drafted tokens without a GPU: struct layout, what is refused, the tree attention's plan."""
import ctypes
import os
import subprocess

import pytest

from llminfer_amd import _binding as B
from llminfer_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_the_c_compiler(tmp_path):
    names = [("llmi_mha_tree_args", B.MhaTreeArgs), ("llmi_qk_norm_rope_tree_args", B.QkNormRopeTreeArgs), ("llmi_verify_tree_args", B.VerifyTreeArgs),
             ("llmi_kv_commit_tree_args", B.KvCommitTreeArgs)]
    lines = []
    want = []
    for c_name, cls in names:
        lines.append('printf("%%zu\\n", sizeof(%s));' % c_name)
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (c_name, field))
            want.append(getattr(cls, field).offset)
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"llmi_hip.h\"\nint main(void) {\n%s\nreturn 0;\n}\n" % "\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    assert [int(x) for x in subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()] == want
    assert B.TREE_MAX_NODES == 64


def tree_args(**over):
    t = B.MhaTreeArgs()
    a = t.mha
    a.query = a.key_cache = a.value_cache = a.output = 0x1000
    a.workspace, a.workspace_bytes = 0x2000, 512 << 20
    a.layer_id, a.pos, a.kv_dim, a.kv_mul, a.head_num, a.head_dim, a.max_seq_len = 0, 4000, 1024, 4, 32, 128, 4096
    t.node_num = 16
    for k, v in over.items():
        setattr(t if k in ("node_num", "tree_mask") else a, k, v)
    return t


def plan(t):
    p = B.MhaPlan()
    return B.lib().llmi_hip_mha_tree_plan(ctypes.byref(t), ctypes.byref(p)), p


@pytest.mark.parametrize("over,status", [
    (dict(), "OK"), (dict(pos=4080), "OK"), (dict(pos=4081), "POS_RANGE"), (dict(pos=-1), "POS_RANGE"), (dict(node_num=0), "INVALID_ARG"),
    (dict(node_num=65), "INVALID_ARG"), (dict(node_num=-3), "INVALID_ARG"), (dict(force_path=1), "INVALID_ARG"), (dict(waves_per_group=4), "INVALID_ARG"),
    (dict(tree_mask=0x1004), "ALIGNMENT"), (dict(query=0), "NULL_POINTER"), (dict(query=0x1008), "ALIGNMENT"), (dict(head_dim=64), "HEAD_DIM"),
    (dict(kv_dim=1000), "KV_DIM"), (dict(head_num=31), "HEAD_GROUP"), (dict(kv_mul=17, head_num=136), "HEAD_GROUP"), (dict(kv_layout=2), "LAYOUT"),
    (dict(num_splits=257), "INVALID_ARG"), (dict(workspace=0x2008), "ALIGNMENT"), (dict(pos_device=0x1002), "ALIGNMENT"),
    (dict(max_seq_len=0), "INVALID_ARG"), (dict(max_seq_len=10, pos=0), "POS_RANGE"),
])
def test_attention_status_codes(over, status):
    assert plan(tree_args(**over))[0] == B.STATUS[status]
    if status != "OK":
        assert B.lib().llmi_hip_mha_decode_tree(ctypes.byref(tree_args(**over))) == B.STATUS[status]


def test_null_arguments():
    L, none = B.lib(), B.STATUS["NULL_POINTER"]
    for call in (L.llmi_hip_mha_decode_tree, L.llmi_hip_qk_norm_rope_append_tree, L.llmi_hip_verify_tree, L.llmi_hip_kv_commit_tree):
        assert call(None) == none
    assert L.llmi_hip_mha_tree_plan(ctypes.byref(tree_args()), None) == none
    assert L.llmi_hip_mha_tree_plan(None, ctypes.byref(B.MhaPlan())) == none


def filled(cls, scalars, over):
    x = cls()
    for name, kind in cls._fields_:
        if kind is ctypes.c_void_p and name not in ("parents", "draft_logits", "pos_device", "stream", "depth"):
            setattr(x, name, 0x1000)
    for k, v in dict(scalars, **over).items():
        setattr(x, k, v)
    return x


@pytest.mark.parametrize("over,status", [
    (dict(target_logits=0), "NULL_POINTER"), (dict(tokens=0), "NULL_POINTER"), (dict(uniform=0), "NULL_POINTER"), (dict(path=0), "NULL_POINTER"),
    (dict(result=0), "NULL_POINTER"), (dict(workspace=0), "NULL_POINTER"), (dict(node_num=0), "INVALID_ARG"), (dict(node_num=65), "INVALID_ARG"),
    (dict(vocab=0), "INVALID_ARG"), (dict(logits_type=2), "INVALID_ARG"), (dict(temperature=-1.0), "INVALID_ARG"),
    (dict(temperature=float("nan")), "INVALID_ARG"), (dict(temperature=float("inf")), "INVALID_ARG"), (dict(temperature=9e-6), "INVALID_ARG"),
    (dict(draft_logits=0x1000, parents=0x1000), "INVALID_ARG"), (dict(draft_logits=0x1000, temperature=0.0), "INVALID_ARG"),
    (dict(target_stride=99), "INVALID_ARG"), (dict(draft_stride=99), "INVALID_ARG"), (dict(target_stride=-100), "INVALID_ARG"),
    (dict(target_logits=0x1002), "ALIGNMENT"), (dict(target_logits=0x1001, logits_type=1), "ALIGNMENT"), (dict(workspace=0x1008), "ALIGNMENT"),
    (dict(tokens=0x1002), "ALIGNMENT"), (dict(parents=0x1002), "ALIGNMENT"), (dict(workspace_bytes=16), "WORKSPACE"),
])
def test_verify_status_codes(over, status):
    scalars = dict(node_num=8, vocab=100, temperature=1.0, workspace_bytes=1 << 20)
    assert B.lib().llmi_hip_verify_tree(ctypes.byref(filled(B.VerifyTreeArgs, scalars, over))) == B.STATUS[status]


@pytest.mark.parametrize("over,status", [
    (dict(key_cache=0), "NULL_POINTER"), (dict(path=0), "NULL_POINTER"), (dict(result=0), "NULL_POINTER"), (dict(head_dim=64), "HEAD_DIM"),
    (dict(kv_dim=100), "KV_DIM"), (dict(layer_num=0), "INVALID_ARG"), (dict(node_num=65), "INVALID_ARG"), (dict(pos=93), "POS_RANGE"),
    (dict(pos=-1), "POS_RANGE"), (dict(kv_layout=3), "LAYOUT"), (dict(key_cache=0x1008), "ALIGNMENT"), (dict(pos_device=0x1001), "ALIGNMENT"),
])
def test_commit_status_codes(over, status):
    scalars = dict(layer_num=2, pos=50, node_num=8, kv_dim=256, head_dim=128, max_seq_len=100, kv_layout=1)
    assert B.lib().llmi_hip_kv_commit_tree(ctypes.byref(filled(B.KvCommitTreeArgs, scalars, over))) == B.STATUS[status]


@pytest.mark.parametrize("over,row,status", [
    ({}, dict(query=0), "NULL_POINTER"), ({}, dict(value_new=0), "NULL_POINTER"), ({}, dict(value_cache=0), "NULL_POINTER"),
    ({}, dict(cos_cache=0), "NULL_POINTER"), ({}, dict(head_dim=64), "HEAD_DIM"), ({}, dict(kv_dim=100), "KV_DIM"), ({}, dict(head_num=0), "INVALID_ARG"),
    (dict(node_num=0), {}, "INVALID_ARG"), (dict(node_num=65), {}, "INVALID_ARG"), ({}, dict(pos=93), "POS_RANGE"), ({}, dict(kv_layout=3), "LAYOUT"),
    ({}, dict(query=0x1008), "ALIGNMENT"), ({}, dict(key_new=0x1008), "ALIGNMENT"), ({}, dict(sin_cache=0x1004), "ALIGNMENT"),
    (dict(key_new_stride=260), {}, "ALIGNMENT"), (dict(key_new_stride=128), {}, "INVALID_ARG"), (dict(query_stride=-2048), {}, "INVALID_ARG"),
    (dict(depth=0x1002), {}, "ALIGNMENT"), ({}, dict(eps=-1.0), "INVALID_ARG"), ({}, dict(eps=float("nan")), "INVALID_ARG"),
])
def test_append_status_codes(over, row, status):
    t = filled(B.QkNormRopeTreeArgs, dict(node_num=8), over)
    scalars = dict(layer_id=0, pos=50, kv_dim=256, head_num=8, head_dim=128, max_seq_len=100, kv_layout=1, eps=1e-6)
    t.row = filled(B.QkNormRopeArgs, scalars, row)
    assert B.lib().llmi_hip_qk_norm_rope_append_tree(ctypes.byref(t)) == B.STATUS[status]


@pytest.mark.parametrize("n,n_q,n_kv,pos,rows,splits", [
    (5, 16, 8, 57, 16, 1), (5, 16, 8, 250, 16, 1), (5, 16, 8, 252, 16, 2), (8, 32, 8, 500, 16, 4), (8, 32, 8, 4099, 16, 16), (8, 32, 8, 9000, 32, 32),
    (16, 32, 8, 6000, 64, 32), (26, 32, 8, 500, 16, 4), (26, 32, 8, 6007, 128, 32), (61, 32, 8, 6000, 128, 16), (61, 32, 8, 32768, 128, 32),
    (64, 64, 8, 131000, 128, 16), (64, 64, 8, 100, 16, 1), (1, 8, 1, 131000, 16, 255),
])
def test_plan_by_size(n, n_q, n_kv, pos, rows, splits):
    rc, p = plan(tree_args(node_num=n, head_num=n_q, kv_dim=128 * n_kv, kv_mul=n_q // n_kv, pos=pos, max_seq_len=pos + n))
    assert rc == 0 and (p.group_pad, p.num_splits) == (rows, splits)
    assert p.path == (B.PATH_SINGLE_PASS if splits == 1 else B.PATH_SPLIT) and p.waves_per_group == 4


def test_plan_invariants_over_random_arguments():
    import random
    rng = random.Random(12)
    for _ in range(3000):
        n, group, n_kv = rng.randint(1, 64), rng.randint(1, 16), rng.choice([1, 2, 3, 4, 8, 16, 40])
        pos = int(2 ** (rng.random() * 18)) - 1
        forced = rng.choice([0, 0, 0, 1, 2, 17, 256])
        t = tree_args(node_num=n, head_num=group * n_kv, kv_dim=128 * n_kv, kv_mul=group, pos=pos, max_seq_len=pos + n + rng.randint(0, 9), num_splits=forced)
        t.mha.workspace_bytes = 1 << 40
        rc, p = plan(t)
        tiles = -(-(pos + n) // 32)
        rows = group * n
        assert rc == 0 and 1 <= p.num_splits <= min(256, tiles) and p.rows_per_split * p.num_splits >= pos + n
        assert p.group_pad in (16, 32, 64, 128) and (rows > 16 or p.group_pad == 16)
        assert (p.num_splits == 1) == (p.workspace_needed == 0)
        if forced:
            assert p.num_splits == min(forced, tiles)
            if p.num_splits > 1:
                t.mha.workspace_bytes = p.workspace_needed - 1
                assert plan(t)[0] == B.STATUS["WORKSPACE"]
                t.mha.workspace_bytes += 1
                assert plan(t)[0] == 0
                t.mha.workspace = None
                assert plan(t)[0] == B.STATUS["WORKSPACE"]
        else:
            # what workspace_bytes says is enough, whatever the length; less of it means fewer splits; none at all, one
            assert p.workspace_needed <= ops.tree_workspace_bytes(group * n_kv, 128, n)
            t.mha.workspace_bytes = p.workspace_needed // 2
            rc, q = plan(t)
            assert rc == 0 and q.num_splits <= max(1, p.num_splits // 2) and q.workspace_needed <= t.mha.workspace_bytes
            t.mha.workspace = None
            rc, q = plan(t)
            assert rc == 0 and q.num_splits == 1 and q.path == B.PATH_SINGLE_PASS


def test_workspace_sizes():
    assert ops.tree_workspace_bytes(32, 128, 8) > 0 and ops.tree_workspace_bytes(0, 128, 8) == 0 and ops.tree_workspace_bytes(32, 128, 0) == 0
    assert ops.verify_workspace_bytes(8, 1000) > 0 and ops.verify_workspace_bytes(0, 5) == 0 and ops.verify_workspace_bytes(3, 0) == 0
    assert ops.verify_workspace_bytes(64, (1 << 31) - 1) > 1 << 20


def test_front_end_refuses_before_the_device_is_reached():
    import torch
    t, i32 = torch.zeros(8, dtype=torch.bfloat16), torch.zeros(8, dtype=torch.int32)
    kw = dict(layer_id=0, pos=5, kv_dim=1024, head_num=32, head_dim=128, max_seq_len=64)
    with pytest.raises(ValueError, match="query must be a device tensor"):
        ops.mha_decode_tree(t, t, t, t, t, node_num=2, kv_mul=4, **kw)
    with pytest.raises(TypeError, match="node_num"):
        ops.mha_decode_tree(t, t, t, t, t, kv_mul=4, **kw)
    with pytest.raises(TypeError, match="workspace_side"):
        ops.mha_decode_tree(t, t, t, t, t, node_num=2, kv_mul=4, workspace_side=1, **kw)
    with pytest.raises(ValueError, match="query must be a device tensor"):
        ops.qk_norm_rope_append_tree(t, t, t, t, t, t, t, t, node_num=2, **kw)
    with pytest.raises(ValueError, match="target_logits must be a .nodes..vocab. tensor"):
        ops.verify_tree(t, i32, t, i32, i32, t)
    with pytest.raises(ValueError, match="1 to 64 rows"):
        ops.verify_tree(torch.zeros(65, 4), i32, t, i32, i32, t)
    with pytest.raises(ValueError, match="target_logits must be a device tensor"):
        ops.verify_tree(torch.zeros(2, 4), i32, t, i32, i32, t)
    with pytest.raises(ValueError, match="key_cache must be a device tensor"):
        ops.kv_commit_tree(t, t, i32, i32, node_num=2, layer_num=1, pos=0, kv_dim=1024, head_dim=128, max_seq_len=64)
