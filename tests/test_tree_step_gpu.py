"""A speculative decoding step as a program runs it -- rows into the cache, attention of all nodes, verification, accepted rows to
their places, layer after layer and step after step -- against decoding the same tokens one by one with the framework's own calls."""
import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

from tree_cases import D, depths_of, parents_of, rows, words_of, words_tensor

pytestmark = pytest.mark.gpu

HEAD, POS = B.KV_LAYOUT_HEAD_MAJOR, B.KV_LAYOUT_POS_MAJOR


class Toy:
    """A model that is nothing but attention blocks: embedding, per layer QKV projection, QK-Norm + RoPE, attention, output projection
    and residual, logits. Products in float32 by torch, rounded to bf16: both ways of decoding share them."""

    def __init__(self, dev, layers=3, n_q=16, n_kv=8, hidden=256, vocab=500, msl=400, layout=HEAD):
        self.dev, self.layers, self.n_q, self.n_kv, self.vocab, self.msl, self.layout = dev, layers, n_q, n_kv, vocab, msl, layout
        dim, kv = n_q * D, n_kv * D
        self.emb = rows(1, vocab, hidden, dev=dev).float()
        self.wqkv = [(rows(10 + l, hidden, dim + 2 * kv, dev=dev, unit=False).float() * hidden ** -0.5) for l in range(layers)]
        self.wo = [(rows(20 + l, dim, hidden, dev=dev, unit=False).float() * dim ** -0.5) for l in range(layers)]
        self.head = rows(30, hidden, vocab, dev=dev, unit=False).float() * 3.0 * hidden ** -0.5
        self.norm = (1 + 0.05 * rows(40, layers, 2 * D, dev=dev, unit=False).float()).to(torch.bfloat16)
        self.sin, self.cos = ops.sincos_table(D, msl, dev)
        shape = (layers, msl, n_kv, D) if layout == POS else (layers, n_kv, msl, D)
        self.kc, self.vc = (torch.full(shape, float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
        self.cache = dict(kv_dim=kv, head_num=n_q, head_dim=D, max_seq_len=msl, kv_layout=layout)
        self.dims = [dim, kv, kv]

    def one(self, token, pos):
        """A decode step of the framework as it was: logits behind one token."""
        x = self.emb[token]
        ws = torch.empty(ops.workspace_bytes(self.n_q, D, self.msl) // 4, device=self.dev)
        for l in range(self.layers):
            q, k, v = (t.contiguous() for t in (x @ self.wqkv[l]).to(torch.bfloat16).split(self.dims))
            out, qn = torch.empty_like(q), torch.empty_like(q)
            ops.qk_norm_rope_append(qn, k, v, self.kc, self.vc, self.norm[l], self.sin, self.cos, layer_id=l, pos=pos, query_src=q, **self.cache)
            ops.mha_decode(qn, self.kc, self.vc, out, ws, layer_id=l, pos=pos, kv_mul=self.n_q // self.n_kv, **self.cache)
            x = x + out.float() @ self.wo[l]
        return x @ self.head

    def tree(self, tokens, mask, depth, pos, word=None, n=None):
        """All nodes of a tree: logits [n][vocab]."""
        n = tokens.shape[0]
        x = self.emb[tokens.long()]
        ws = torch.empty(max(4, ops.tree_workspace_bytes(self.n_q, D, n) // 4), device=self.dev)
        q = torch.empty(n, self.dims[0], dtype=torch.bfloat16, device=self.dev)
        out = torch.empty_like(q)
        for l in range(self.layers):
            packed = (x @ self.wqkv[l]).to(torch.bfloat16)
            qr, k, v = packed.split(self.dims, dim=1)
            ops.qk_norm_rope_append_tree(q, k, v, self.kc, self.vc, self.norm[l], self.sin, self.cos, node_num=n, depth=depth, layer_id=l, pos=pos,
                                         query_src=qr, pos_device=word, **self.cache)
            ops.mha_decode_tree(q, self.kc, self.vc, out, ws, node_num=n, tree_mask=mask, layer_id=l, pos=pos, kv_mul=self.n_q // self.n_kv,
                                pos_device=word, **self.cache)
            x = x + out.float() @ self.wo[l]
        return x @ self.head

    def commit(self, path, result, n, pos, word=None):
        kw = {k: v for k, v in self.cache.items() if k != "head_num"}
        ops.kv_commit_tree(self.kc, self.vc, path, result, node_num=n, layer_num=self.layers, pos=pos, pos_device=word, **kw)


def greedy(dev, layout, prompt, steps):
    """Tokens and logits one by one."""
    toy, tokens, logits = Toy(dev, layout=layout), list(prompt), []
    for i in range(len(prompt) + steps - 1):
        y = toy.one(tokens[i], i)
        if i >= len(prompt) - 1:
            logits.append(y)
            tokens.append(int(y.argmax()))
    return toy, tokens, logits


@pytest.mark.parametrize("layout", [POS, HEAD])
def test_greedy_steps_give_the_tokens_of_single_steps(dev, layout):
    prompt = [(37 * i + 5) % 500 for i in range(90)]
    plain, want, logits = greedy(dev, layout, prompt, 40)
    # (the two ways differ by roundings: the test needs a likeliest token that stands out)
    margin = min(float((y.topk(2).values[0] - y.topk(2).values[1])) for y in logits)
    assert margin > 0.02, margin
    toy = Toy(dev, layout=layout)
    for i, t in enumerate(prompt[:-1]):
        toy.one(t, i)
    got, pos, drafted, calls = [prompt[-1]], len(prompt) - 1, 0, 0
    path, result = torch.zeros(64, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    while len(got) <= 40:
        n = [26, 5, 64, 1][calls % 4]
        parents = parents_of(calls, n, "chain" if n == 5 else "tree")
        depth = depths_of(parents)
        # a draft that knows the answer on one branch, as far as it goes, and guesses wrong elsewhere
        known = {0}
        tokens = [got[-1]]
        for i in range(1, n):
            at = pos + depth[i]
            if parents[i] in known and not any(j in known and parents[j] == parents[i] for j in range(1, i)) and at < len(want) and (i * 7 + calls) % 5:
                known.add(i)
                tokens.append(want[at])
            else:
                tokens.append((got[-1] + 11 * i + 3) % 500)
        t = torch.tensor(tokens, dtype=torch.int32, device=dev)
        y = toy.tree(t, words_tensor(words_of(parents), dev), torch.tensor(depth, dtype=torch.int32, device=dev), pos)
        ws = torch.empty(ops.verify_workspace_bytes(n, 500) // 4, device=dev)
        ops.verify_tree(y, t, torch.zeros(n, device=dev), path[:n], result, ws, parents=torch.tensor(parents, dtype=torch.int32, device=dev), temperature=0.0)
        toy.commit(path, result, n, pos)
        count, following = result.tolist()
        got += [tokens[i] for i in path.tolist()[1:count]] + [following]
        pos += count
        drafted += count - 1
        calls += 1
    assert got[:40] == want[89:129] and drafted > 15
    # the rows the steps have left in the cache are those of single steps, up to what a rounding of the attention's output shifts
    a, b = ((c[:, :pos] if layout == POS else c[:, :, :pos]).float() for c in (toy.kc, plain.kc))
    used = min(pos, len(want) - 1)
    a, b = (x[:, :used] if layout == POS else x[:, :, :used] for x in (a, b))
    assert float((a - b).norm() / b.norm()) < 2.0 ** -6


def test_a_captured_step_follows_its_words(dev):
    """Rows, attention, verification, commit and the position's advance in one graph, replayed step after step: the same as the
    calls made one by one."""
    n, parents = 12, parents_of(4, 12)
    mask, depth = words_tensor(words_of(parents), dev), torch.tensor(depths_of(parents), dtype=torch.int32, device=dev)
    up = torch.tensor(parents, dtype=torch.int32, device=dev)
    runs = []
    for captured in (False, True):
        toy = Toy(dev)
        for i in range(30):
            toy.one((91 * i + 7) % 500, i)
        word = torch.full((1,), 30, dtype=torch.int32, device=dev)
        tokens, u = torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(n, device=dev)
        path, result = torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
        ws = torch.empty(ops.verify_workspace_bytes(n, 500) // 4, device=dev)

        def step():
            y = toy.tree(tokens, mask, depth, toy.msl - n, word)
            ops.verify_tree(y, tokens, u, path, result, ws, parents=up, temperature=0.8)
            toy.commit(path, result, n, toy.msl - n, word)
            return y

        if captured:
            keep = toy.kc.clone(), toy.vc.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # (what a library sets up at its first call is not captured)
                step()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            toy.kc.copy_(keep[0])
            toy.vc.copy_(keep[1])
        gen = torch.Generator(device=dev)
        gen.manual_seed(11)
        seen, root = [], 3
        for _ in range(12):
            drafts = torch.randint(0, 500, (n,), generator=gen, device=dev, dtype=torch.int32)
            drafts[1::2] = drafts[0]
            tokens.copy_(drafts)
            tokens[0] = root
            u.copy_(torch.rand(n, generator=gen, device=dev) * torch.tensor([1.0] + [1e-5] * (n - 1), device=dev))
            graph.replay() if captured else step()
            torch.cuda.synchronize()
            seen.append((path.tolist(), result.tolist(), int(word)))
            word.add_(result[:1])
            root = result[1].item()
        runs.append((seen, toy.kc.clone(), toy.vc.clone()))
    assert runs[0][0] == runs[1][0]
    assert any(r[1][0] > 1 for r in runs[0][0])
    end = runs[0][0][-1][2] + runs[0][0][-1][1][0]  # (behind the last accepted row lie rows of the last tree)
    for a, b in zip(runs[0][1:], runs[1][1:]):
        assert torch.equal(a[:, :, :end], b[:, :, :end])
