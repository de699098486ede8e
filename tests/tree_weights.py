"""Inputs of the tree attention in which few keys have a weight, so that what a weight is rounded to shows in the outputs, and what an output may
then be off by."""
import math

import torch

from tree_cases import D, rows

SCORE = 0.25 * 1.05 * math.sqrt(D)  # the largest sum of |q k| / sqrt(128) over the keys that count


def few_keys(seed, n, n_q, n_kv, ctx, dev, every):
    """q [n][n_q][128] with a first value of 1, k and v [ctx + n][n_kv][128]. Cached positions 0, every, 2 every, ... and the nodes have scores around 0,
    all others lie 226 below (2560 / sqrt(128); 326 in log2: their weights are 0 in fp32, and add nothing)."""
    q, k, v = rows(seed, n, n_q, D, dev=dev), 0.25 * rows(seed + 1, ctx + n, n_kv, D, dev=dev), rows(seed + 2, ctx + n, n_kv, D, dev=dev, unit=False)
    q[:, :, 0] = 1.0
    counts = torch.zeros(ctx + n, dtype=torch.bool, device=dev)
    counts[:ctx:every] = True
    counts[ctx:] = True
    k[:, :, 0] = torch.where(counts, 0.0, -2560.0).to(torch.bfloat16)[:, None]
    return q, k, v


def weight_bound(size, keys):
    """`size`: weighted mean of |V|; `keys`: how many have a weight. A weight is the sum of two bf16 numbers: the second, at most 2^-8 of the weight, is
    rounded to 2^-8 of itself. Its exponent is a sum of 128 products scaled once, a step of which loses at most one last place (2^-23: the matrix
    cores' sums may be cut off); the exponentials of the weight, of the rescaling and of the joins over wavefronts and splits are good to 2^-20 each, their
    arguments' roundings included; sums of `keys` terms and up to 300 parts lose a last place a term. Exponent, exponentials and sums enter
    numerator and denominator."""
    return (2.0 ** -16 + 2 * (130 * 2.0 ** -23 * SCORE + 4 * 2.0 ** -20 + (keys + 300) * 2.0 ** -23)) * size + 1e-30


def rounded_attention(q, k, v, ctx, words, parts):
    """The formula in 64 bits but for the weights of the sum over V, each the sum of `parts` bf16 numbers; the sum of weights stays as it is."""
    n, n_q, _ = q.shape
    group = n_q // k.shape[0]
    out = torch.zeros(n, n_q, D, dtype=torch.float64, device=q.device)
    for i in range(n):
        at = torch.tensor(list(range(ctx)) + [ctx + t for t in range(n) if words[i] >> t & 1], device=q.device)
        for h in range(n_q):
            s = (k[h // group, at].double() * q[i, h].double()).sum(-1) / math.sqrt(D)
            w = torch.exp(s - s.max())
            kept, rest = torch.zeros_like(w), w
            for _ in range(parts):
                kept, rest = kept + rest.to(torch.bfloat16).double(), rest - rest.to(torch.bfloat16).double()
            out[i, h] = (kept[:, None] * v[h // group, at].double()).sum(0) / w.sum()
    return out
