"""How many bits of a weight llmi_hip_mha_decode_tree keeps. With an output_f32: those of two bf16 numbers, at every size (tree_weights.weight_bound).
Without one, beyond 128 query rows of a KV head, those of one: a kernel of its own, so what the other tests ask through output_f32 is asked here of
the bf16 output alone."""
import ctypes
import math

import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

from test_mha_tree_gpu import FORMS, Case
from tree_cases import D, attention64, attention_bound, by_head, parents_of, words_of, words_tensor
from tree_weights import few_keys, weight_bound

pytestmark = pytest.mark.gpu

HEAD, POS = B.KV_LAYOUT_HEAD_MAJOR, B.KV_LAYOUT_POS_MAJOR
NAN = float("nan")
MORE_FORMS = [(61, 32, 8, 1000, 128), (33, 64, 8, 900, 128), (64, 40, 8, 6000, 128)]  # (more of those with one number a weight)


class Bf16Case(Case):
    """The bf16 output, with no output_f32 asked for."""

    def run(self, mask="words", ws=None, **over):
        ws = torch.full((max(ops.tree_workspace_bytes(self.n_q, D, self.n) // 4, 4),), NAN, device=self.dev) if ws is None else ws
        out = torch.full((self.n + 1, self.n_q * D), 7.0, dtype=torch.bfloat16, device=self.dev)
        mask = words_tensor(self.words, self.dev) if mask == "words" else mask
        ops.mha_decode_tree(self.q, self.kc, self.vc, out[:self.n], ws, tree_mask=mask, **self.scalars(**over))
        torch.cuda.synchronize()
        assert bool((out[self.n] == 7).all())
        return out[:self.n].view(self.n, self.n_q, D)

    def check(self, got, words=None, ctx=None, what=""):
        ctx = self.ctx if ctx is None else ctx
        k, v = (by_head(c[self.layer], self.layout) for c in (self.kc, self.vc))
        want, size = attention64(self.q, k, v, ctx, self.words if words is None else words)
        # the fp32 result's bound, and half a bf16 step of what is then rounded
        bound = attention_bound(size, ctx + self.n, 1.02 * math.sqrt(D))
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
        worst = float(((got.double() - want).abs() / bound).max())
        assert torch.isfinite(got).all() and worst <= 1, "%s: %.2f of the bound" % (what, worst)


def weighed(case_type, dev, n, n_q, n_kv, ctx, layout):
    """A case of few_keys, every node seeing itself alone: 6 to 8 cached keys count."""
    every = max(1, ctx // 6 - 1)
    c = case_type(dev, n, n_q, n_kv, ctx, layout, words=[1 << i for i in range(n)], seed=n)
    c.q, k, v = few_keys(n, n, n_q, n_kv, ctx, dev, every)
    for cache, x in ((c.kc, k), (c.vc, v)):
        by_head(cache[0], layout)[:, :ctx + n] = x.transpose(0, 1)
    return c, every


@pytest.mark.parametrize("layout", [POS, HEAD])
@pytest.mark.parametrize("n,n_q,n_kv,ctx,rows_of_group", FORMS + MORE_FORMS)
def test_fp32_outputs_have_two_numbers_a_weight(dev, n, n_q, n_kv, ctx, rows_of_group, layout):
    c, every = weighed(Case, dev, n, n_q, n_kv, ctx, layout)
    k, v = (by_head(x[0], layout) for x in (c.kc, c.vc))
    word = torch.zeros(1, dtype=torch.int32, device=dev)
    for pos, over in ((ctx, {}), (ctx, dict(num_splits=5, ws=torch.full((32 << 20,), NAN, device=dev))), (2 * every + 1, dict(pos_device=word))):
        word.fill_(pos)
        if pos != ctx:  # (the nodes' rows lie behind the position)
            for x in (k, v):
                x[:, pos:pos + n] = x[:, ctx:ctx + n].clone()
        got = c.run(**over)
        want, size = attention64(c.q, k, v, pos, c.words)
        worst = float(((got.double() - want).abs() / weight_bound(size, -(-pos // every) + 1)).max())
        assert torch.isfinite(got).all() and worst <= 1, "%d positions: %.2f of the bound" % (pos, worst)


@pytest.mark.parametrize("n,n_q,n_kv,ctx,rows_of_group", FORMS)
def test_the_bf16_output_is_that_rounded(dev, n, n_q, n_kv, ctx, rows_of_group):
    """Up to 128 query rows of a KV head, and in blocks of sixteen, asking for the fp32 output changes nothing."""
    full, short = Case(dev, n, n_q, n_kv, ctx, seed=n), Bf16Case(dev, n, n_q, n_kv, ctx, seed=n)
    a, b = full.run(), short.run()
    short.check(b)
    if n * n_q // n_kv <= 128 or rows_of_group == 16:
        assert torch.equal(a.to(torch.bfloat16), b)


@pytest.mark.parametrize("layout", [POS, HEAD])
@pytest.mark.parametrize("n,n_q,n_kv,ctx,rows_of_group", FORMS + MORE_FORMS)
def test_every_form(dev, n, n_q, n_kv, ctx, rows_of_group, layout):
    """Trees, an empty word, rows that hold what no output may show, positions on the device, split counts."""
    bad = [i for i in range(1, n) if i % 4 == 1]
    hidden = sum(1 << i for i in bad)
    words = [w & ~hidden for w in words_of(parents_of(7, n))]
    words[n - 1] = 0
    c = Bf16Case(dev, n, n_q, n_kv, ctx, layout, words=words, seed=n)
    args, plan = B.MhaTreeArgs(), B.MhaPlan()
    args.mha = ops.make_mha_args(c.q, c.kc, c.vc, c.q, torch.empty(24 << 20, device=dev), **{k: v for k, v in c.scalars().items() if k != "node_num"})
    args.node_num = n
    assert B.lib().llmi_hip_mha_tree_plan(ctypes.byref(args), ctypes.byref(plan)) == 0 and plan.group_pad == rows_of_group
    clean = c.run()
    c.check(clean)
    word = torch.zeros(1, dtype=torch.int32, device=dev)
    for pos in (0, 1, ctx // 2 + 3, ctx - 1):
        word.fill_(pos)
        c.check(c.run(pos_device=word), ctx=pos, what="position %d" % pos)
    for splits in (1, 2, 7, 61):
        c.check(c.run(num_splits=splits, ws=torch.full((32 << 20,), NAN, device=dev)), what="%d splits" % splits)
    for k, i in enumerate(bad):
        for cache in (c.kc, c.vc):
            by_head(cache[0], layout)[:, ctx + i] = [NAN, math.inf, -math.inf, -3.3895e38][k % 4]
    assert torch.equal(c.run(), clean)
    sees = [i for i in range(n) if words[i] & 1]
    v = by_head(c.vc[0], layout)
    for at, who in ((ctx, sees), (ctx - 1, list(range(n))), (ctx // 3, list(range(n)))):
        for poison in (math.inf, NAN):
            kept = v[:, at, 77].clone()
            v[:, at, 77] = poison
            got = c.run()
            v[:, at, 77] = kept
            assert not bool(torch.isfinite(got[who][:, :, 77]).any()), "position %d" % at
            assert torch.equal(got[:, :, :77], clean[:, :, :77]) and torch.equal(got[:, :, 78:], clean[:, :, 78:])


@pytest.mark.parametrize("n,n_q,n_kv,ctx", [(61, 32, 8, 3000), (64, 64, 8, 1500)])
def test_replays(dev, n, n_q, n_kv, ctx):
    """One graph for every position, two workspaces' worth of calls in a row; the same bits as the calls made one by one, every time."""
    c = Bf16Case(dev, n, n_q, n_kv, ctx)
    word, mask = torch.full((1,), ctx, dtype=torch.int32, device=dev), words_tensor(c.words, dev)
    ws = torch.full((ops.tree_workspace_bytes(n_q, D, n) // 4 + 4,), NAN, device=dev)
    outs = [torch.zeros(n, n_q * D, dtype=torch.bfloat16, device=dev) for _ in range(2)]

    def steps():
        for out in outs:
            ops.mha_decode_tree(c.q, c.kc, c.vc, out, ws, tree_mask=mask, pos_device=word, **c.scalars())

    steps()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps()
    for pos in (ctx, 3, 333, 0, 64, ctx - 1, ctx):
        word.fill_(pos)
        for out in outs:
            out.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        eager = c.run(pos_device=word)
        assert all(torch.equal(out.view_as(eager), eager) for out in outs)


@pytest.mark.parametrize("layout", [POS, HEAD])
def test_offsets_past_32_bits(dev, layout):
    c = Bf16Case(dev, 33, 64, 8, 131000, layout, layers=17, layer=16, spare=66)
    c.check(c.run())
