"""Attention over an 8-bit KV cache with values near the largest that its sums hold, against the definition in 64 bits (kv8_cases)."""
import math

import pytest
import torch

from llminfer_amd import ops

import kv8_cases as C

pytestmark = pytest.mark.gpu
D, BF16 = C.D, C.BF16
LARGEST = 1e36  # over the positions: what the contract promises


def grown(keys, first, fmt, largest):
    """One KV head whose first `first` positions have scores of 0 and all others of some 7.5 in powers of two, just not enough for a running maximum that is followed from
    8 on to be raised; V rows of +-largest. Query, cache, K and V as they stand there."""
    g = torch.Generator().manual_seed(keys)
    q = C.rows(g, 1, outliers=False)
    k = torch.zeros(1, 1, keys, D, dtype=BF16)
    k[0, 0, first:] = (q[0].double() * (7.5 * math.log(2.0) * math.sqrt(D) / float(q.double().square().sum()))).to(BF16)
    v = (torch.where(torch.rand(1, 1, keys, D, generator=g) < 0.9, 1.0, -1.0) * largest).to(BF16)
    pad, packed, values = -keys % 32, [], []
    for x in (k, v):
        c, s = C.quantise(x, fmt)
        values.append(C.stands_for(c, s, fmt))
        packed += [torch.cat([c, torch.full((1, 1, pad, D), 0x7F, dtype=torch.uint8)], 2), torch.cat([s, torch.full((1, 1, pad), math.nan, dtype=BF16)], 2)]
    score = (values[0][0, 0] @ q[0].double()) / math.sqrt(D) / math.log(2.0)
    assert bool((score[:first] == 0).all()) and bool(((score[first:] > 7.0) & (score[first:] < 8.0)).all())
    return q, C.pack(*packed), values[0][0], values[1][0]


@pytest.mark.parametrize("fmt", [C.E4M3, C.INT8])
@pytest.mark.parametrize("keys,splits", [(384, 0), (384, 1), (576, 0), (3000, 1), (3000, 3), (20000, 1), (20000, 0)])
def test_large_values_beside_a_maximum_that_lags(dev, keys, splits, fmt):
    """Eight wavefronts (and splits) whose first records have the small scores: every weight that follows is some 2^7.5, nowhere is a sum out of range."""
    first = 256 if splits < 2 else 32
    q, cache, k, v = grown(keys, first, fmt, LARGEST / keys)
    out, tap = torch.full((1, D), math.nan, dtype=BF16, device=dev), torch.full((1, D), math.nan, device=dev)
    ops.mha_decode_kv8(q.to(dev), cache.to(dev), out, torch.full((132 * 256 + 4,), math.nan, device=dev), output_f32=tap, layer_id=0, pos=keys - 1, kv_dim=D, kv_mul=1, head_num=1, head_dim=D,
                       max_seq_len=keys, kv8_format=fmt, num_splits=splits)
    C.close(tap.cpu(), *C.attention(q, k, v), rounded=out.cpu())
