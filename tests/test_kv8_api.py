"""The C ABI's calls for an 8-bit KV cache without a GPU: struct layout, what is refused, sizes, the attention's plan."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

import kv8_cases as C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_the_c_compiler(tmp_path):
    names = [("llmi_kv8_copy_args", B.Kv8CopyArgs), ("llmi_qk_norm_rope_kv8_args", B.QkNormRopeKv8Args), ("llmi_mha_kv8_args", B.MhaKv8Args),
             ("llmi_mha_kv8_append_args", B.MhaKv8AppendArgs)]
    lines, want = [], []
    for c_name, cls in names:
        lines.append('printf("%%zu\\n", sizeof(%s));' % c_name)
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (c_name, field))
            want.append(getattr(cls, field).offset)
    lines.append('printf("%d\\n%d\\n%d\\n%d\\n", LLMI_KV8_E4M3, LLMI_KV8_INT8, LLMI_KV8_RECORD_POSITIONS, LLMI_KV8_RECORD_BYTES);')
    want += [B.KV8_E4M3, B.KV8_INT8, B.KV8_RECORD_POSITIONS, B.KV8_RECORD_BYTES]
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"llmi_hip.h\"\nint main(void) {\n%s\nreturn 0;\n}\n" % "\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    assert [int(x) for x in subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()] == want
    assert (C.RECORD, C.PLACES) == (B.KV8_RECORD_BYTES, B.KV8_RECORD_POSITIONS)


@pytest.mark.parametrize("layers,msl,kv_dim,head_dim,want", [
    (1, 1, 128, 128, 8320), (1, 32, 128, 128, 8320), (1, 33, 128, 128, 2 * 8320), (36, 4096, 1024, 128, 36 * 8 * 128 * 8320),
    (0, 32, 128, 128, 0), (1, 0, 128, 128, 0), (1, 32, 100, 128, 0), (1, 32, 128, 64, 0), (-1, 32, 128, 128, 0),
    (1, (1 << 31) - 1, 128, 128, (1 << 26) * 8320), ((1 << 31) - 1, (1 << 31) - 1, 1 << 30, 128, 0),
])
def test_sizes(layers, msl, kv_dim, head_dim, want):
    assert ops.kv8_bytes(layers, msl, kv_dim, head_dim) == want


def mha(**over):
    a = B.MhaKv8Args()
    a.query, a.cache8, a.output = 0x10000, 0x1000, 1 << 40
    a.workspace, a.workspace_bytes = 0x2000, 512 << 20
    a.layer_id, a.pos, a.kv_dim, a.kv_mul, a.head_num, a.head_dim, a.max_seq_len = 0, 4000, 1024, 4, 32, 128, 4096
    for k, v in over.items():
        setattr(a, k, v)
    return a


def plan(a):
    p = B.MhaPlan()
    return B.lib().llmi_hip_mha_kv8_plan(ctypes.byref(a), ctypes.byref(p)), p


MHA_REFUSED = [
    (dict(pos=4096), "POS_RANGE"), (dict(pos=-1), "POS_RANGE"), (dict(query=0), "NULL_POINTER"), (dict(cache8=0), "NULL_POINTER"), (dict(output=0), "NULL_POINTER"),
    (dict(query=0x10008), "ALIGNMENT"), (dict(cache8=0x1008), "ALIGNMENT"), (dict(output=0x20004), "ALIGNMENT"), (dict(workspace=0x2008), "ALIGNMENT"),
    (dict(output_f32=0x1002), "ALIGNMENT"), (dict(pos_device=0x1002), "ALIGNMENT"), (dict(head_dim=64), "HEAD_DIM"), (dict(kv_dim=1000), "KV_DIM"),
    (dict(kv_dim=0), "KV_DIM"), (dict(kv_dim=-128), "KV_DIM"), (dict(head_num=31), "HEAD_GROUP"), (dict(kv_mul=17, head_num=136), "HEAD_GROUP"), (dict(kv_mul=0, head_num=0), "HEAD_GROUP"),
    (dict(num_splits=257), "INVALID_ARG"), (dict(num_splits=-1), "INVALID_ARG"), (dict(max_seq_len=0), "INVALID_ARG"), (dict(layer_id=-1), "INVALID_ARG"),
    (dict(format=2), "INVALID_ARG"), (dict(format=-1), "INVALID_ARG"), (dict(kv_dim=128 * 65536, kv_mul=1, head_num=65536), "INVALID_ARG"),
    (dict(num_splits=16, workspace_bytes=16 * 32 * 528 + 15), "WORKSPACE"), (dict(num_splits=2, workspace=0), "WORKSPACE"),
    (dict(output=0x10000), "INVALID_ARG"), (dict(output=0x10000 + 32 * 256 - 16), "INVALID_ARG"), (dict(output=0x10000 - 16), "INVALID_ARG"),
    (dict(output_f32=0x10000 - 4), "INVALID_ARG"), (dict(output_f32=0x10000 + 32 * 256 - 4), "INVALID_ARG"),
]


@pytest.mark.parametrize("over,status", MHA_REFUSED)
def test_attention_status_codes(over, status):
    want, L = B.STATUS[status], B.lib()
    assert plan(mha(**over))[0] == want
    assert L.llmi_hip_mha_decode_kv8(ctypes.byref(mha(**over))) == want
    t = B.MhaKv8AppendArgs(mha=mha(**over), key_new=0x1000, value_new=0x1000, norm_weight=0x1000, sin_cache=0x1000, cos_cache=0x1000, eps=1e-6)
    assert L.llmi_hip_mha_decode_append_kv8(ctypes.byref(t)) == want


@pytest.mark.parametrize("over,status", [
    (dict(key_new=0), "NULL_POINTER"), (dict(value_new=0), "NULL_POINTER"), (dict(norm_weight=0), "NULL_POINTER"), (dict(sin_cache=0), "NULL_POINTER"),
    (dict(cos_cache=0), "NULL_POINTER"), (dict(key_new=0x1008), "ALIGNMENT"), (dict(cos_cache=0x1004), "ALIGNMENT"), (dict(eps=-1.0), "INVALID_ARG"),
    (dict(eps=float("nan")), "INVALID_ARG"), (dict(key_new=1 << 40), "INVALID_ARG"), (dict(value_new=(1 << 40) + 32 * 256 - 16), "INVALID_ARG"),
])
def test_append_status_codes(over, status):
    t = B.MhaKv8AppendArgs(mha=mha(), key_new=0x1000, value_new=0x1000, norm_weight=0x1000, sin_cache=0x1000, cos_cache=0x1000, eps=1e-6)
    for k, v in over.items():
        setattr(t, k, v)
    assert B.lib().llmi_hip_mha_decode_append_kv8(ctypes.byref(t)) == B.STATUS[status]


@pytest.mark.parametrize("over,status", [
    (dict(query=0), "NULL_POINTER"), (dict(cache8=0), "NULL_POINTER"), (dict(sin_cache=0), "NULL_POINTER"), (dict(row_num=0), "INVALID_ARG"), (dict(row_num=-5), "INVALID_ARG"),
    (dict(head_num=0), "INVALID_ARG"), (dict(head_num=1 << 30), "INVALID_ARG"), (dict(format=7), "INVALID_ARG"), (dict(pos=4090, row_num=7), "POS_RANGE"), (dict(pos=-1), "POS_RANGE"),
    (dict(pos=0, row_num=4097), "POS_RANGE"), (dict(pos=(1 << 31) - 1, row_num=(1 << 31) - 1), "POS_RANGE"), (dict(query_stride=4092), "ALIGNMENT"),
    (dict(query_stride=4088, row_num=2), "INVALID_ARG"), (dict(key_new_stride=1016, row_num=2), "INVALID_ARG"), (dict(value_new_stride=-1024, row_num=2), "INVALID_ARG"),
    (dict(cache8=0x1008), "ALIGNMENT"), (dict(query_src=0x1008), "ALIGNMENT"), (dict(pos_device=0x1001), "ALIGNMENT"), (dict(head_dim=256), "HEAD_DIM"), (dict(kv_dim=192), "KV_DIM"),
    (dict(eps=float("nan")), "INVALID_ARG"), (dict(layer_id=-2), "INVALID_ARG"),
])
def test_rows_status_codes(over, status):
    a = B.QkNormRopeKv8Args()
    for name in ("query", "key_new", "value_new", "cache8", "norm_weight", "sin_cache", "cos_cache"):
        setattr(a, name, 0x1000)
    a.pos, a.row_num, a.kv_dim, a.head_num, a.head_dim, a.max_seq_len, a.eps = 5, 1, 1024, 32, 128, 4096, 1e-6
    for k, v in over.items():
        setattr(a, k, v)
    assert B.lib().llmi_hip_qk_norm_rope_append_kv8(ctypes.byref(a)) == B.STATUS[status]


@pytest.mark.parametrize("over,status", [
    (dict(key_cache=0), "NULL_POINTER"), (dict(cache8=0), "NULL_POINTER"), (dict(value_cache=0x1008), "ALIGNMENT"), (dict(layer_num=-1), "INVALID_ARG"), (dict(first_pos=-1), "POS_RANGE"),
    (dict(num_pos=-1), "POS_RANGE"), (dict(first_pos=4000, num_pos=97), "POS_RANGE"), (dict(first_pos=(1 << 31) - 1, num_pos=(1 << 31) - 1), "POS_RANGE"), (dict(kv_layout=2), "LAYOUT"),
    (dict(format=2), "INVALID_ARG"), (dict(head_dim=64), "HEAD_DIM"), (dict(kv_dim=64), "KV_DIM"), (dict(max_seq_len=-4), "INVALID_ARG"),
    (dict(max_seq_len=(1 << 31) - 1), "INVALID_ARG"),
])
def test_copy_status_codes(over, status):
    a = B.Kv8CopyArgs()
    a.key_cache = a.value_cache = a.cache8 = 0x1000
    a.layer_num, a.first_pos, a.num_pos, a.kv_dim, a.head_dim, a.max_seq_len, a.kv_layout = 2, 0, 10, 1024, 128, 4096, 1
    for k, v in over.items():
        setattr(a, k, v)
    assert B.lib().llmi_hip_kv8_store(ctypes.byref(a)) == B.STATUS[status]
    assert B.lib().llmi_hip_kv8_load(ctypes.byref(a)) == B.STATUS[status]


def test_neighbours_do_not_overlap():
    """Output right behind or in front of an input (the plan makes no HIP call)."""
    for out in (0x10000 + 32 * 256, 0x10000 - 32 * 256):
        assert plan(mha(output=out))[0] == 0
    assert plan(mha(output_f32=0x10000 - 32 * 512))[0] == 0


def test_null_arguments():
    L, none = B.lib(), B.STATUS["NULL_POINTER"]
    for call in (L.llmi_hip_mha_decode_kv8, L.llmi_hip_mha_decode_append_kv8, L.llmi_hip_qk_norm_rope_append_kv8, L.llmi_hip_kv8_store, L.llmi_hip_kv8_load):
        assert call(None) == none
    assert L.llmi_hip_mha_kv8_plan(ctypes.byref(mha()), None) == none
    assert L.llmi_hip_mha_kv8_plan(None, ctypes.byref(B.MhaPlan())) == none


def test_nothing_to_copy_is_no_launch():
    a = B.Kv8CopyArgs()
    a.key_cache = a.value_cache = a.cache8 = 0x1000
    a.kv_dim, a.head_dim, a.max_seq_len = 1024, 128, 4096
    for layers, count, first in ((0, 7, 0), (3, 0, 0), (3, 0, 4096)):
        a.layer_num, a.num_pos, a.first_pos = layers, count, first
        assert B.lib().llmi_hip_kv8_store(ctypes.byref(a)) == 0 and B.lib().llmi_hip_kv8_load(ctypes.byref(a)) == 0


def test_plan_over_random_arguments():
    rng = random.Random(11)
    for _ in range(3000):
        n_kv, group = rng.choice([1, 2, 3, 8, 16, 40, 512, 65535]), rng.randint(1, 16)
        msl = rng.choice([1, 31, 33, 4096, 131072, (1 << 31) - 1])
        pos = rng.randrange(msl)
        enough = ops.workspace_bytes(n_kv * group, 128, msl)
        room = rng.choice([0, 16, 5000, 1 << 20, enough])
        splits = rng.choice([0, 0, 0, 1, 2, 17, 256])
        rc, p = plan(mha(pos=pos, kv_dim=128 * n_kv, kv_mul=group, head_num=n_kv * group, max_seq_len=msl, workspace_bytes=room, num_splits=splits))
        tiles = pos // 32 + 1
        if rc != 0:
            assert rc == B.STATUS["WORKSPACE"] and splits > 1
            continue
        assert p.workspace_needed <= max(room, 16) and p.workspace_needed < 1 << 31 and 1 <= p.num_splits <= 256
        assert p.num_splits <= tiles and (splits == 0 or p.num_splits <= splits) and p.waves_per_group in (4, 8)
        assert min(p.rows_per_split, 1 << 30) * p.num_splits >= min(pos + 1, 1 << 30)
        assert (p.path == B.PATH_SINGLE_PASS) == (p.num_splits == 1)


@pytest.mark.parametrize("fmt", [C.E4M3, C.INT8])
def test_the_oracle_s_codes(fmt):
    """Nearest codes: no other code's value is nearer, ties go to the even one; and the layout's two directions undo one another."""
    g = torch.Generator().manual_seed(4)
    x = C.rows(g, 3, 2, 64)
    codes, scale = C.quantise(x, fmt)
    every = torch.arange(256, dtype=torch.uint8).view(torch.int8 if fmt else torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every) & (every.abs() <= C.TOP[fmt])]
    off = (x.double() - C.stands_for(codes, scale, fmt)).abs()
    best = (x.double()[..., None] / scale.double()[..., None, None] - every).abs().amin(-1) * scale.double()[..., None]
    assert bool((off <= best * (1 + 1e-12)).all())
    top = x.double().abs().amax(-1)
    s = scale.double()
    below = torch.frexp(s)
    below = torch.ldexp(torch.floor(below[0] * 256) - 1, below[1] - 8)
    assert bool((s * C.TOP[fmt] >= top).all()) and bool((below * C.TOP[fmt] < top).all())
    kc, ks, vc, vs = (codes, scale, codes.flip(2).contiguous(), scale.flip(2).contiguous())
    back = C.unpack(C.pack(kc, ks, vc, vs))
    assert all(torch.equal(a, b) for a, b in zip(back, (kc, ks, vc, vs)))
