"""What the calls for drafted tokens refuse before anything is launched: arguments at the ends of their ranges."""
import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

from tree_cases import D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layer,msl", [((1 << 31) - 1, 1 << 26), ((1 << 30) - 1, 1 << 27), ((1 << 31) - 1, (1 << 31) - 1)])
def test_sizes_past_64_bits(dev, layer, msl):
    """layers * max_seq_len * kv_dim is 2^64 (and more) elements: no tensor holds them, though the product's low 64 bits are 0."""
    x = torch.zeros(4, D, dtype=torch.bfloat16, device=dev)
    ws, i32 = torch.zeros(64, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    cache = dict(kv_dim=D, head_dim=D, max_seq_len=msl, pos=1, node_num=1)
    with pytest.raises(ValueError, match="key_cache has 512 elements"):
        ops.mha_decode_tree(x, x, x, torch.zeros_like(x), ws, layer_id=layer, kv_mul=1, head_num=1, **cache)
    with pytest.raises(ValueError, match="key_cache has 512 elements"):
        ops.qk_norm_rope_append_tree(x, x, x, x, x, x, ws, ws, layer_id=layer, head_num=1, **cache)
    with pytest.raises(ValueError, match="key_cache has 512 elements"):
        ops.kv_commit_tree(x, x, i32, i32, layer_num=layer, **cache)


@pytest.mark.parametrize("temperature", [1e-6, 1e-40, 1e-46, 1e-300, 5e-324, -1e-46, -1e-300])
def test_temperatures_that_fp32_does_not_have(dev, temperature):
    """Too small for a sampled call, and not 0: refused as any other below the least one, not taken for greedy."""
    x, i32 = torch.zeros(4, 100, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    ws = torch.empty(ops.verify_workspace_bytes(4, 100) // 4, device=dev)
    path, result = torch.full_like(i32, 77), torch.full_like(i32, 77)
    with pytest.raises(B.LlmiError, match="out of range"):
        ops.verify_tree(x, i32, torch.zeros(4, device=dev), path, result, ws, temperature=temperature)
    torch.cuda.synchronize()
    assert bool((path == 77).all()) and bool((result == 77).all())


def test_a_temperature_of_zero_is_greedy(dev):
    x, i32 = torch.zeros(4, 100, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    x[:, 60] = 1.0
    ws = torch.empty(ops.verify_workspace_bytes(4, 100) // 4, device=dev)
    for temperature in (0, 0.0, -0.0):
        path, result = torch.full_like(i32, 77), torch.full_like(i32, 77)
        ops.verify_tree(x, i32, None, path, result, ws, temperature=temperature)
        assert path.tolist() == [0, -1, -1, -1] and result.tolist()[:2] == [1, 60]
