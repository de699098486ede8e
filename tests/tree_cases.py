"""Drafted trees for the tests: parents, words, depths, and the operators' definitions in 64 bits."""
import math
import random

import numpy as np
import torch

D = 128


def parents_of(seed, n, kind="tree"):
    rng = random.Random(seed)
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)]


def words_of(parents):
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return seen


def depths_of(parents):
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return depth


def words_tensor(words, dev):
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device=dev)


def rows(seed, *shape, dev, unit=True):
    """Seeded bf16 rows; unit: root mean square 1 over the last dimension, as QK-Norm leaves them."""
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    x = torch.randn(shape, generator=gen, device=dev)
    if unit:
        x = x / x.square().mean(-1, keepdim=True).sqrt()
    return x.to(torch.bfloat16)


def by_head(cache, layout):
    """One layer's cache as [KV head][position][128], a view."""
    return cache.transpose(0, 1) if layout == 0 else cache


def attention64(q, k, v, ctx, words):
    """q [n][n_q][128]; k, v [n_kv][>= ctx + n][128]. Returns (output, weighted mean of |V|), both [n][n_q][128] in 64 bits. Rows a node
    does not see do not enter."""
    n, n_q, _ = q.shape
    n_kv = k.shape[0]
    group = n_q // n_kv
    out = torch.zeros(n, n_q, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for i in range(n):
        at = list(range(ctx)) + [ctx + t for t in range(n) if words[i] >> t & 1]
        if not at:
            continue
        idx = torch.tensor(at, device=q.device)
        ks, vs = k[:, idx].double(), v[:, idx].double()
        qs = q[i].double().view(n_kv, group, D)
        w = torch.softmax((qs[:, :, None, :] * ks[:, None]).sum(-1) / math.sqrt(D), -1) if len(at) <= 400 else torch.softmax(
            torch.matmul(qs, ks.transpose(1, 2).contiguous()) / math.sqrt(D), -1)
        out[i] = torch.matmul(w, vs).reshape(n_q, D)
        size[i] = torch.matmul(w, vs.abs()).reshape(n_q, D)
    return out, size


def attention_bound(size, keys, score_size):
    """What the fp32 result may be off by, from the definition. `size`: weighted mean of |V|. A weight enters the sum over V rounded to bf16
    at worst (2^-8); its exponent is a sum of 128 products scaled once, each step rounded to fp32 (130 * 2^-24 * score_size, score_size the
    largest sum of |q k| / sqrt(128)), the exponential and the factors that join parts are good to 2^-21 together, and sums of `keys` terms in
    fp32 to keys * 2^-24; exponent and sum enter numerator and denominator."""
    return (2.0 ** -8 + 2 * (130 * 2.0 ** -24 * score_size + 2.0 ** -21 + keys * 2.0 ** -24)) * size + 1e-30


def verify_oracle(target, tokens, parents, uniform, heat, draft=None):
    """Node by node, as the definition goes, in 64 bits on the host. target, draft: float32 numpy [n][vocab]. Returns (path, token)."""
    n, vocab = target.shape
    big = np.finfo(np.float32).max

    def clean(row):
        row = row.astype(np.float64)
        row[np.isnan(row)] = -np.inf
        return np.minimum(row, big)

    def chances(row):
        row = clean(row)
        if not np.isfinite(row.max()):
            return np.zeros(vocab)
        with np.errstate(over="ignore"):
            w = np.exp((row - row.max()) / heat)
        return w / w.sum()

    def likeliest(row):
        row = clean(row)
        return int(np.argmax(row)) if np.isfinite(row.max()) else -1

    path = [0]
    while True:
        at = path[-1]
        left = None if heat == 0 else chances(target[at])
        refused, follow, mass = set(), None, 1.0
        for c in range(1, n):
            if parents[c] != at or not 0 <= tokens[c] < vocab:
                continue
            x = int(tokens[c])
            if heat == 0:
                yes = x == likeliest(target[at])
            elif draft is None:
                yes = x not in refused and left[x] > 0 and float(uniform[c]) * mass < left[x]
                if not yes and x not in refused:
                    refused.add(x)
                    mass -= left[x]
            else:
                yes = left[x] > 0 and float(uniform[c]) * chances(draft[at])[x] < left[x]
            if yes:
                follow = c
                break
        if follow is None:
            break
        path.append(follow)
    if heat == 0 or likeliest(target[at]) < 0:
        return path, likeliest(target[at])
    if draft is not None and at < n - 1:
        left = np.maximum(left - chances(draft[at]), 0.0)
    for x in refused:
        left[x] = 0.0
    sums = np.cumsum(left)
    if sums[-1] <= 0:
        return path, likeliest(target[at])
    token = int(np.searchsorted(sums, float(uniform[0]) * sums[-1], side="right"))
    return path, min(token, int(np.nonzero(left)[0][-1]))
