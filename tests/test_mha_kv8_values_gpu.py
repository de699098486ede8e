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


@pytest.mark.parametrize("fmt", [C.E4M3, C.INT8])
@pytest.mark.parametrize("splits", [0, 1])
def test_weights_keep_the_bits_of_fp32(dev, splits, fmt):
    """V rows that are all alike: the output is that row whatever the weights, as long as the sum over V has the weights that the sum of weights has.

    257 positions on eight wavefronts. The first one's first 32 positions have a score of 0, a weight of 1; its last position a score between 7 and 8 in powers of two, a weight of as many bits as there
    are, which decides the output; the other wavefronts' scores lie 2^-40 and more below. Sixteen query heads, each with another last score.
    What rounds in fp32: 32 equal products of a weight of 1, V's scale of eight bits and a code: nothing. The last weight times V's scale (2^-24), its products with the code, added one by one where it is a sum of
    up to three numbers (2^-23 each, whichever way the matrix unit rounds), the sum of weights (2^-24), the quotient and its product (2^-24 each); the other wavefronts less than 2^-30. 3 * 2^-23 + 4 * 2^-24 and that:
    6 * 2^-23 of the output. (A weight that is cut to sixteen bits is 2^-17 off.)"""
    g = torch.Generator().manual_seed(5)
    keys, n_q = 257, 16
    for seed in range(8):
        direction = C.rows(g, 1, outliers=False)[0].double()
        direction /= direction.square().sum().sqrt()
        q = (direction * torch.linspace(0.88, 0.99, n_q, dtype=torch.float64)[:, None] * 8.0).to(BF16)
        k = torch.zeros(1, 1, keys, D, dtype=BF16)
        unit = math.log(2.0) * math.sqrt(D) / 8.0  # a score of 1 in powers of two for a query of 8 along the direction
        k[0, 0, 32:256] = (direction * (-60.0 * unit)).to(BF16)
        k[0, 0, 256] = (direction * ((7.98 - 0.01 * seed) * unit)).to(BF16)
        packed, values = [], []
        for x in (k, torch.ones(1, 1, keys, D, dtype=BF16)):
            c, s = C.quantise(x, fmt)
            values.append(C.stands_for(c, s, fmt))
            packed += [torch.cat([c, torch.full((1, 1, 31, D), 0x7F, dtype=torch.uint8)], 2), torch.cat([s, torch.full((1, 1, 31), math.nan, dtype=BF16)], 2)]
        score = (q.double() @ values[0][0, 0].t()) / math.sqrt(D) / math.log(2.0)
        assert bool((score[:, :32] == 0).all()) and bool((score[:, 32:256] < -40.0).all()) and bool(((score[:, 256] > 6.5) & (score[:, 256] < 7.99)).all())
        out, tap = torch.full((n_q, D), math.nan, dtype=BF16, device=dev), torch.full((n_q, D), math.nan, device=dev)
        ops.mha_decode_kv8(q.to(dev), C.pack(*packed).to(dev), out, None, output_f32=tap, layer_id=0, pos=keys - 1, kv_dim=D, kv_mul=n_q, head_num=n_q, head_dim=D, max_seq_len=keys,
                           kv8_format=fmt, num_splits=splits)
        row = values[1][0, 0, 0, 0]
        off = (tap.cpu().double() / row - 1.0).abs().max()
        assert float(off) <= 6 * 2.0 ** -23, float(off)
