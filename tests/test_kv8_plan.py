"""The plan of the attention over an 8-bit KV cache at the lengths where its form changes, without a GPU."""
import ctypes

import pytest

from llminfer_amd import _binding as B
from llminfer_amd import ops


def plan(keys, fmt=0, device=False, **over):
    a = B.MhaKv8Args(query=1 << 33, cache8=1 << 34, output=1 << 35, workspace=1 << 36, workspace_bytes=256 << 20, pos=keys - 1, kv_dim=1024, kv_mul=4, head_num=32, head_dim=128,
                     max_seq_len=1 << 20, format=fmt, pos_device=(1 << 37) if device else 0)
    for k, v in over.items():
        setattr(a, k, v)
    p = B.MhaPlan()
    assert B.lib().llmi_hip_mha_kv8_plan(ctypes.byref(a), ctypes.byref(p)) == 0
    assert p.group_pad == 16 and p.rows_per_split % 32 == 0 and p.rows_per_split * p.num_splits >= keys
    return p.path, p.num_splits, p.waves_per_group, p.workspace_needed


@pytest.mark.parametrize("device", [False, True])
@pytest.mark.parametrize("fmt,most", [(B.KV8_E4M3, 18), (B.KV8_INT8, 12)])
def test_short_contexts_are_single_pass_and_need_no_workspace(fmt, most, device):
    for keys in (1, 32, 128, 129, 300, 32 * most):
        assert plan(keys, fmt, device) == (B.PATH_SINGLE_PASS, 1, 4 if keys <= 128 else 8, 0)
        assert plan(keys, fmt, device, workspace=0, workspace_bytes=0) == (B.PATH_SINGLE_PASS, 1, 4 if keys <= 128 else 8, 0)


@pytest.mark.parametrize("device", [False, True])
def test_splits_by_length(device):
    fused = B.PATH_SPLIT_FUSED
    for keys, splits in ((32 * 18 + 1, 19), (1024, 32), (2500, 32), (3168, 32), (4096, 32)):  # (256 workgroups: 32 for each of 8 KV heads)
        assert plan(keys, device=device)[:2] == (fused, splits) and plan(keys, device=device)[3] == 32 * 528 * splits + 16
    for keys, splits in ((1024, 32), (32 * 96, 32), (32 * 102, 34), (32 * 300, 100), (1 << 20, 256)):
        assert plan(keys, device=device, kv_dim=128, kv_mul=8, head_num=8)[:2] == (fused, splits)
    assert plan(9000, device=device, workspace=0, workspace_bytes=0) == (B.PATH_SINGLE_PASS, 1, 8, 0)
    assert plan(9000, device=device, workspace_bytes=32 * 528 * 5 + 31)[1] == 5


@pytest.mark.parametrize("device", [False, True])
def test_chosen_splits(device):
    for keys, chosen, splits in ((20, 4, 1), (200, 4, 4), (200, 256, 7), (4000, 256, 125), (9000, 3, 3)):
        assert plan(keys, device=device, num_splits=chosen)[1] == splits


def test_what_the_workspace_call_gives_is_enough():
    for heads, group in ((1, 1), (8, 4), (1, 16), (40, 5)):
        for keys in (1, 577, 1024, 5000, 100000):
            assert plan(keys, kv_dim=128 * heads, kv_mul=group, head_num=heads * group)[3] <= ops.workspace_bytes(heads * group, 128, keys)
