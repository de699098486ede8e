"""llmi_hip_verify_tree on the device against its definition, node by node in 64 bits on the host. Whole numbers: equal."""
import math

import numpy as np
import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

from tree_cases import parents_of, verify_oracle

pytestmark = pytest.mark.gpu

INF = float("inf")


def make(seed, n, vocab, kind="tree", scale=2.0, bf16=False, likely=0.7):
    """Logits, tokens (mostly likely ones), parents, random numbers, as numpy."""
    rng = np.random.RandomState(seed)
    target = (scale * rng.standard_normal((n, vocab))).astype(np.float32)
    draft = (target + 0.5 * scale * rng.standard_normal((n, vocab))).astype(np.float32)
    if bf16:
        target, draft = (torch.from_numpy(x).to(torch.bfloat16).float().numpy() for x in (target, draft))
    parents = parents_of(seed, n, kind)
    tokens = np.zeros(n, np.int32)
    for i in range(1, n):
        order = np.argsort(-draft[parents[i]])
        tokens[i] = order[min(rng.randint(0, 3), vocab - 1)] if rng.rand() < likely else rng.randint(0, vocab)
    return target, draft, tokens, parents, rng.random_sample(n).astype(np.float32)


def run(dev, target, tokens, parents, uniform, heat, draft=None, dtype=torch.float32, pad=0):
    """Through the front end; `pad`: columns of NaN behind each row's tokens (rows that are slices of wider ones)."""
    n, vocab = target.shape

    def up(x):
        if x is None:
            return None
        wide = torch.full((n, vocab + pad), float("nan"), dtype=dtype, device=dev)
        wide[:, :vocab] = torch.from_numpy(x).to(dtype)
        return wide[:, :vocab]

    chain = parents == [i - 1 for i in range(n)]
    ws = torch.full((ops.verify_workspace_bytes(n, vocab) // 4,), float("nan"), device=dev)
    path = torch.full((n + 1,), 77, dtype=torch.int32, device=dev)
    result = torch.full((3,), 77, dtype=torch.int32, device=dev)
    for given in ([None, parents] if chain and draft is None else [None if chain else parents]):
        path.fill_(77)
        result.fill_(77)
        p = None if given is None else torch.tensor(given, dtype=torch.int32, device=dev)
        ops.verify_tree(up(target), torch.from_numpy(tokens).to(dev), torch.from_numpy(uniform).to(dev), path[:n], result[:2], ws, parents=p,
                        draft_logits=up(draft), temperature=heat)
        torch.cuda.synchronize()
        got = path.tolist()
        assert got[n] == 77 and result[2].item() == 77
        count = result[0].item()
        assert 1 <= count <= n and got[count:n] == [-1] * (n - count)
    return got[:count], result[1].item()


@pytest.mark.parametrize("heat", [0.0, 0.3, 1.0, 2.0])
@pytest.mark.parametrize("n,vocab", [(1, 1), (1, 50), (2, 2), (3, 4095), (5, 4096), (8, 4097), (16, 1000), (33, 8193), (64, 152), (64, 32001),
                                     (26, 151936)])
def test_trees(dev, n, vocab, heat):
    for seed in range(6 if vocab < 40000 else 2):
        for kind in ("tree", "chain", "star"):
            bf16 = seed % 2 == 1
            target, _, tokens, parents, u = make(seed, n, vocab, kind, bf16=bf16)
            want = verify_oracle(target, tokens, parents, u, heat)
            got = run(dev, target, tokens, parents, u, heat, dtype=torch.bfloat16 if bf16 else torch.float32, pad=seed)
            assert got == want, (seed, kind)


@pytest.mark.parametrize("heat", [0.5, 1.0])
@pytest.mark.parametrize("n,vocab", [(1, 7), (2, 50), (5, 1000), (6, 32000), (9, 151936), (64, 4500)])
def test_chains_with_draft_logits(dev, n, vocab, heat):
    for seed in range(8 if vocab < 100000 else 3):
        target, draft, tokens, parents, u = make(seed, n, vocab, "chain", likely=1.0, bf16=seed % 2 == 1)
        if seed % 3 == 0:  # (long paths: the draft is nearly the target)
            draft = target + 0.01 * (draft - target)
            draft = torch.from_numpy(draft).to(torch.bfloat16).float().numpy() if seed % 2 else draft
        want = verify_oracle(target, tokens, parents, u, heat, draft)
        got = run(dev, target, tokens, parents, u, heat, draft, torch.bfloat16 if seed % 2 else torch.float32, pad=3 * (seed % 2))
        assert got == want, seed


def test_ties_go_to_the_lowest_index(dev):
    for vocab in (3, 300, 5000, 20000):
        target = np.zeros((3, vocab), np.float32)
        target[1, [vocab // 3, vocab - 1]] = 4.0
        target[2, vocab - 2:] = 1.0
        tokens = np.array([0, 0, vocab // 3], np.int32)
        assert run(dev, target, tokens, [-1, 0, 1], np.zeros(3, np.float32), 0.0) == ([0, 1, 2], vocab - 2)
        tokens[2] = vocab - 1
        assert run(dev, target, tokens, [-1, 0, 1], np.zeros(3, np.float32), 0.0)[0] == ([0, 1] if vocab > 3 else [0, 1])


@pytest.mark.parametrize("heat", [0.0, 1.0])
def test_filtered_and_broken_logits(dev, heat):
    """-inf and NaN have no weight, +inf has all of it, a row without a weight accepts nothing and draws -1."""
    for seed in range(8):
        target, draft, tokens, parents, u = make(seed, 24, 6000)
        rng = np.random.RandomState(100 + seed)
        for r in range(24):
            target[r, rng.permutation(6000)[:5990 if r % 2 else 3000]] = [-INF, np.nan, -3.4028235e38][r % 3]
        if seed % 2:
            target[2, 4321] = INF
            target[5, [17, 5000]] = INF
        assert run(dev, target, tokens, parents, u, heat) == verify_oracle(target, tokens, parents, u, heat), seed
    for value in (-INF, np.nan):
        target = np.full((2, 5000), value, np.float32)
        assert run(dev, target, np.zeros(2, np.int32), [-1, 0], np.zeros(2, np.float32), heat) == ([0], -1)
        target[0, 4100] = -7.0
        assert run(dev, target, np.full(2, 4100, np.int32), [-1, 0], np.zeros(2, np.float32), heat) == ([0, 1], -1)
    lowest = np.full((1, 5000), -3.4028235e38, np.float32)  # (all at the type's lowest value: all alike)
    assert run(dev, lowest, np.zeros(1, np.int32), [-1], np.array([0.5], np.float32), 1.0) == ([0], 2500)


def test_siblings_with_the_same_token(dev):
    """A token that has been refused is not accepted from a later sibling, and its mass is taken away once."""
    target = np.log(np.array([[0.5, 0.3, 0.2]] * 5)).astype(np.float32)
    parents, tokens = [-1, 0, 0, 0, 0], np.array([0, 1, 1, 1, 2], np.int32)
    # token 1 (0.3) refused at 0.9; twice more not tried, whatever their numbers; then token 2: u * 0.7 < 0.2
    for u4, want in ((0.28, ([0, 4], None)), (0.29, ([0], 0))):
        u = np.array([0.4, 0.9, 0.0, 0.0, u4], np.float32)
        path, token = run(dev, target, tokens, parents, u, 1.0)
        assert path == want[0] and (want[1] is None or token == want[1])
        assert (path, token) == verify_oracle(target, tokens, parents, u, 1.0)


def test_nodes_out_of_range(dev):
    """A parent that does not come before its node, or a token outside the vocabulary: not accepted, nor what hangs below."""
    target = np.zeros((6, 40), np.float32)
    target[:, 5] = 20.0
    u = np.zeros(6, np.float32)
    tokens = np.full(6, 5, np.int32)
    for heat in (0.0, 1.0):
        assert run(dev, target, tokens, [-1, 0, 1, 2, 3, 4], u, heat)[0] == [0, 1, 2, 3, 4, 5]
        for bad in (2, 3, 64, 1 << 30, -1, -(1 << 31)):
            assert run(dev, target, tokens, [-1, 0, bad, 2, 3, 4], u, heat)[0] == [0, 1]
        for bad in (-1, 40, (1 << 31) - 1, -(1 << 31)):
            t = tokens.copy()
            t[3] = bad
            assert run(dev, target, t, [-1, 0, 1, 2, 3, 4], u, heat)[0] == [0, 1, 2]


def test_edges_of_the_random_numbers(dev):
    """0 accepts whatever has a weight and draws the first token with one; just below 1 the last; numbers outside [0, 1) stay in range."""
    target = np.full((2, 9000), -INF, np.float32)
    target[:, [100, 4200, 8999]] = [1.0, 2.0, 0.0]
    last = np.float32(1) - np.float32(2) ** -24
    for token in (100, 4200, 8999):
        assert run(dev, target, np.array([0, token], np.int32), [-1, 0], np.zeros(2, np.float32), 1.0) == ([0, 1], 100)
    assert run(dev, target, np.array([0, 101], np.int32), [-1, 0], np.zeros(2, np.float32), 1.0) == ([0], 100)
    assert run(dev, target, np.array([0, 101], np.int32), [-1, 0], np.full(2, last), 1.0) == ([0], 8999)
    for odd in (1.0, 7.5, INF, np.nan, -3.0, -INF):
        path, token = run(dev, target, np.array([0, 4200], np.int32), [-1, 0], np.full(2, odd, np.float32), 1.0)
        assert token in (100, 4200, 8999) and path in ([0], [0, 1])


def test_nothing_left(dev):
    """All of a row's mass on refused tokens: the likeliest one. (A number of 1 or more refuses what a proper one could not.)"""
    target = np.full((2, 5000), -INF, np.float32)
    target[:, 4444] = 0.0
    assert run(dev, target, np.array([0, 4444], np.int32), [-1, 0], np.full(2, 1.5, np.float32), 1.0) == ([0], 4444)
    draft = target.copy()
    assert run(dev, target, np.array([0, 4444], np.int32), [-1, 0], np.full(2, 1.5, np.float32), 1.0, draft) == ([0], 4444)


def test_a_draft_row_without_weight(dev):
    """It cannot have given the token: refused, and the following one is the target's own."""
    # (4096 equal weights: every sum is exact)
    target = np.zeros((3, 4096), np.float32)
    target[0, 4000] = 40.0
    for empty in (-INF, math.nan):
        draft = target.copy()
        draft[0] = empty
        assert run(dev, target, np.array([0, 4000, 7], np.int32), [-1, 0, 1], np.full(3, 0.5, np.float32), 1.0, draft) == ([0], 4000)
        # (the second row is one: its node is not reached past)
        draft = target.copy()
        draft[1] = empty
        assert run(dev, target, np.array([0, 4000, 7], np.int32), [-1, 0, 1], np.array([0.5, 0.5, 0.0], np.float32), 1.0, draft) == ([0, 1], 2048)


def test_greedy_takes_no_random_numbers(dev):
    target, _, tokens, parents, _ = make(11, 20, 9000)
    ws = torch.empty(ops.verify_workspace_bytes(20, 9000) // 4, device=dev)
    path, result = torch.zeros(20, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    ops.verify_tree(torch.from_numpy(target).to(dev), torch.from_numpy(tokens).to(dev), None, path, result, ws,
                    parents=torch.tensor(parents, dtype=torch.int32, device=dev), temperature=0.0)
    count, token = result.tolist()
    assert (path.tolist()[:count], token) == verify_oracle(target, tokens, parents, None, 0.0)


@pytest.mark.parametrize("with_draft", [False, True])
def test_the_target_is_what_is_sampled(dev, with_draft):
    """The first token behind the root over many random numbers, against the target's distribution: frequencies within five
    standard deviations, sqrt(p (1 - p) / runs)."""
    runs, vocab = 4000, 6
    rng = np.random.RandomState(9)
    target, draft = (rng.standard_normal((3, vocab)).astype(np.float32) for _ in range(2))
    p, q = (np.exp(x[0]) / np.exp(x[0]).sum() for x in (target, draft))
    heads = torch.from_numpy(target).to(dev), torch.from_numpy(draft).to(dev)
    u = torch.from_numpy(rng.random_sample((runs, 3)).astype(np.float32)).to(dev)
    first = rng.choice(vocab, size=runs, p=q / q.sum()) if with_draft else np.full(runs, 2)
    tokens = np.stack([np.zeros(runs), first, np.full(runs, 4)], 1).astype(np.int32)
    t = torch.from_numpy(tokens).to(dev)
    path, result = torch.zeros((runs, 3), dtype=torch.int32, device=dev), torch.zeros((runs, 2), dtype=torch.int32, device=dev)
    star = torch.tensor([-1, 0, 0], dtype=torch.int32, device=dev)
    ws = torch.empty(ops.verify_workspace_bytes(3, vocab) // 4, device=dev)
    for i in range(runs):
        if with_draft:
            ops.verify_tree(heads[0], t[i], u[i], path[i], result[i], ws, draft_logits=heads[1])
        else:
            ops.verify_tree(heads[0], t[i], u[i], path[i], result[i], ws, parents=star)
    torch.cuda.synchronize()
    path, result = path.cpu().numpy(), result.cpu().numpy()
    got = np.where(result[:, 0] > 1, tokens[np.arange(runs), np.maximum(path[:, 1], 0)], result[:, 1])
    share = np.bincount(got, minlength=vocab) / runs
    assert np.all(np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / runs)), (share, p)
    assert (result[:, 0] > 1).any() and (result[:, 0] == 1).any()


def test_captured(dev):
    """One graph, replayed with other logits, tokens and numbers, the program's own work between the replays; two graphs on one workspace."""
    n, vocab = 20, 9001
    cases = [make(40 + i, n, vocab) for i in range(6)]
    target = torch.zeros(n, vocab, device=dev)
    tokens, parents = (torch.zeros(n, dtype=torch.int32, device=dev) for _ in range(2))
    u = torch.zeros(n, device=dev)
    path, result = torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    ws = torch.full((ops.verify_workspace_bytes(n, vocab) // 4,), float("nan"), device=dev)
    graphs = {}
    for heat in (1.0, 0.0):
        ops.verify_tree(target, tokens, u, path, result, ws, parents=parents, temperature=heat)
        torch.cuda.synchronize()
        graphs[heat] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[heat]):
            ops.verify_tree(target, tokens, u, path, result, ws, parents=parents, temperature=heat)
    for c in cases:
        target.copy_(torch.from_numpy(c[0]))
        tokens.copy_(torch.from_numpy(c[2]))
        parents.copy_(torch.tensor(c[3], dtype=torch.int32))
        u.copy_(torch.from_numpy(c[4]))
        for heat, graph in graphs.items():
            graph.replay()
            torch.cuda.synchronize()
            count, token = result.tolist()
            assert (path.tolist()[:count], token) == verify_oracle(c[0], c[2], c[3], c[4], heat)


def test_the_front_end_refuses(dev):
    x = torch.zeros(4, 100, device=dev)
    i32 = lambda k: torch.zeros(k, dtype=torch.int32, device=dev)
    ws = torch.empty(ops.verify_workspace_bytes(4, 100) // 4, device=dev)
    ok = dict(target_logits=x, tokens=i32(4), uniform=torch.zeros(4, device=dev), path=i32(4), result=i32(2), workspace=ws)
    ops.verify_tree(**ok)
    torch.cuda.synchronize()
    for change, error, text in [
            (dict(tokens=i32(3)), ValueError, "tokens has 3 elements"), (dict(path=i32(3)), ValueError, "path has 3"),
            (dict(result=i32(1)), ValueError, "result has 1"), (dict(uniform=torch.zeros(2, device=dev)), ValueError, "uniform has 2"),
            (dict(tokens=torch.zeros(4, dtype=torch.int64, device=dev)), ValueError, "tokens has dtype"),
            (dict(target_logits=x.half()), ValueError, "target_logits has dtype"), (dict(target_logits=x[0]), ValueError, "must be a"),
            (dict(target_logits=x.t()), ValueError, "1 to 64 rows"), (dict(target_logits=x[:, ::2]), ValueError, "contiguous rows"),
            (dict(target_logits=x.cpu()), ValueError, "device tensor"), (dict(parents=i32(2)), ValueError, "parents has 2"),
            (dict(draft_logits=x.to(torch.bfloat16)), ValueError, "draft_logits has dtype"),
            (dict(draft_logits=x[:, :99]), ValueError, "draft_logits must be"),
            (dict(draft_logits=x, parents=i32(4)), B.LlmiError, "out of range"), (dict(draft_logits=x, temperature=0.0), B.LlmiError, "out of range"),
            (dict(temperature=-1.0), B.LlmiError, "out of range"), (dict(temperature=1e-6), B.LlmiError, "out of range"),
            (dict(temperature=math.nan), B.LlmiError, "out of range"), (dict(workspace=ws[:8]), B.LlmiError, "workspace"),
            (dict(temperature="1"), TypeError, "real number")]:
        with pytest.raises(error, match=text):
            ops.verify_tree(**dict(ok, **change))
