"""llmi_hip_verify_tree with draft logits where the chain is shorter than the call's rows: the nodes behind it carry tokens outside the
vocabulary and their draft rows hold whatever was there. Nothing was tried behind the last real node, so what follows it is drawn from the
target's own distribution."""
import math

import numpy as np
import pytest
import torch

from llminfer_amd import ops

pytestmark = pytest.mark.gpu

PADS = [-1, "vocab", (1 << 31) - 1, -(1 << 31)]


def chances(row, heat):
    w = np.exp((row.astype(np.float64) - row.max()) / heat)
    return w / w.sum()


def padded_oracle(target, draft, tokens, uniform, heat):
    """Sampling with refusal, node by node in 64 bits: the draft's distribution is taken away where a token of its was refused, and only there."""
    n, vocab = target.shape
    at = 0
    while True:
        left = chances(target[at], heat)
        if at + 1 == n or not 0 <= tokens[at + 1] < vocab:
            break
        q = chances(draft[at], heat)
        x = tokens[at + 1]
        if left[x] > 0 and float(uniform[at + 1]) * q[x] < left[x]:
            at += 1
            continue
        left = np.maximum(left - q, 0.0)
        break
    sums = np.cumsum(left)
    if sums[-1] <= 0:
        return at + 1, int(np.argmax(target[at]))
    return at + 1, min(int(np.searchsorted(sums, float(uniform[0]) * sums[-1], side="right")), int(np.nonzero(left)[0][-1]))


def run(dev, target, draft, tokens, uniform, heat, dtype):
    n, vocab = target.shape
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)
    path, result = torch.full((n,), 77, dtype=torch.int32, device=dev), torch.full((2,), 77, dtype=torch.int32, device=dev)
    ws = torch.full((ops.verify_workspace_bytes(n, vocab) // 4,), math.nan, device=dev)
    ops.verify_tree(up(target).to(dtype), up(tokens), up(uniform), path, result, ws, draft_logits=up(draft).to(dtype), temperature=heat)
    count, token = result.tolist()
    assert path.tolist() == list(range(count)) + [-1] * (n - count)
    return count, token


def make(seed, n, vocab, real, pad, same, dtype):
    """A chain of `real` nodes in `n` rows, its tokens the draft's likely ones; `same`: the draft's rows are the target's."""
    rng = np.random.RandomState(seed)
    target = (1.5 * rng.standard_normal((n, vocab))).astype(np.float32)
    draft = target.copy() if same else (target + rng.standard_normal((n, vocab))).astype(np.float32)
    if dtype == torch.bfloat16:
        target, draft = (torch.from_numpy(x).to(dtype).float().numpy() for x in (target, draft))
    tokens = np.full(n, vocab if pad == "vocab" else pad, np.int32)
    tokens[0] = 0
    for i in range(1, real):
        tokens[i] = np.argsort(-draft[i - 1])[rng.randint(0, min(3, vocab))]
    return target, draft, tokens, rng.random_sample(n).astype(np.float32)


@pytest.mark.parametrize("pad", PADS)
@pytest.mark.parametrize("n,real,vocab", [(2, 1, 6), (2, 1, 5000), (6, 1, 32000), (6, 3, 32000), (6, 5, 900), (64, 40, 4097), (64, 2, 50)])
def test_the_token_behind_a_padded_chain(dev, n, real, vocab, pad):
    for seed in range(6):
        dtype = torch.bfloat16 if seed % 2 else torch.float32
        for same in (False, True):
            target, draft, tokens, u = make(seed, n, vocab, real, pad, same, dtype)
            if seed % 3 == 0:
                u[1:] = 0.0  # (all real nodes are accepted)
            heat = (1.0, 0.7)[seed // 2 % 2]
            want = padded_oracle(target, draft, tokens, u, heat)
            if seed % 3 == 0 or same:
                assert want[0] == real
            assert run(dev, target, draft, tokens, u, heat, dtype) == want, (seed, same)


@pytest.mark.parametrize("garbage", [math.nan, math.inf, -math.inf, 0.0, 3.0e38])
def test_draft_rows_behind_the_chain_are_not_used(dev, garbage):
    target, draft, tokens, u = make(5, 5, 3000, 3, -1, False, torch.float32)
    u[1:] = 0.0
    want = padded_oracle(target, draft, tokens, u, 1.0)
    draft[2:] = garbage
    assert run(dev, target, draft, tokens, u, 1.0, torch.float32) == want == (3, want[1])


@pytest.mark.parametrize("same", [False, True])
def test_every_token_comes_as_often_as_the_target_says(dev, same):
    """All of a root's tokens over evenly spread random numbers: token t falls on the numbers of its own stretch of the running sum, within one
    number at either end."""
    vocab, steps = 6, 500
    target, draft, tokens, _ = make(17, 2, vocab, 1, -1, same, torch.float32)
    seen = np.zeros(vocab)
    for k in range(steps):
        count, token = run(dev, target, draft, tokens, np.full(2, (k + 0.5) / steps, np.float32), 1.0, torch.float32)
        assert count == 1
        seen[token] += 1
    assert np.all(np.abs(seen - steps * chances(target[0], 1.0)) <= 1.0), seen / steps


def test_a_refused_token_still_takes_the_draft_away(dev):
    """A real node that is refused, padding behind it: what is left is max(p - q, 0), as in a chain without padding."""
    for seed in range(20):
        target, draft, tokens, u = make(100 + seed, 4, 700, 2, -1, False, torch.float32)
        u[1] = 0.999
        assert run(dev, target, draft, tokens, u, 1.0, torch.float32) == padded_oracle(target, draft, tokens, u, 1.0), seed
