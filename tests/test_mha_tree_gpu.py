"""llmi_hip_mha_decode_tree on the device against its definition in 64 bits: the same bf16 inputs, the fp32 result within the bound of
tree_cases.attention_bound, the bf16 output the rounding of the fp32 result. Whatever the call must not read holds NaN."""
import ctypes
import math

import pytest
import torch

from llminfer_amd import _binding as B
from llminfer_amd import ops

from tree_cases import D, attention64, attention_bound, by_head, parents_of, rows, words_of, words_tensor

pytestmark = pytest.mark.gpu

HEAD, POS = B.KV_LAYOUT_HEAD_MAJOR, B.KV_LAYOUT_POS_MAJOR
NAN = float("nan")


class Case:
    def __init__(self, dev, n, n_q, n_kv, ctx, layout=HEAD, kind="tree", words=None, seed=0, layers=1, layer=0, spare=3):
        self.n, self.n_q, self.n_kv, self.ctx, self.layout, self.layer = n, n_q, n_kv, ctx, layout, layer
        self.words = words_of(parents_of(seed + n, n, kind)) if words is None else words
        self.msl = ctx + n + spare
        shape = (self.msl, n_kv, D) if layout == POS else (n_kv, self.msl, D)
        self.kc, self.vc = (torch.full((layers,) + shape, NAN, dtype=torch.bfloat16, device=dev) for _ in range(2))
        k, v = rows(seed + 1, ctx + n, n_kv, D, dev=dev), rows(seed + 2, ctx + n, n_kv, D, dev=dev, unit=False)
        for cache, x in ((self.kc, k), (self.vc, v)):
            by_head(cache[layer], layout)[:, :ctx + n] = x.transpose(0, 1)
        self.q = rows(seed + 3, n, n_q, D, dev=dev)
        self.dev = dev

    def scalars(self, **over):
        return dict(dict(node_num=self.n, layer_id=self.layer, pos=self.ctx, kv_dim=self.n_kv * D, kv_mul=self.n_q // self.n_kv,
                         head_num=self.n_q, head_dim=D, max_seq_len=self.msl, kv_layout=self.layout), **over)

    def run(self, mask="words", ws=None, **over):
        ws_bytes = ops.tree_workspace_bytes(self.n_q, D, self.n)
        ws = torch.full((max(ws_bytes // 4, 4),), NAN, device=self.dev) if ws is None else ws
        out = torch.full((self.n + 1, self.n_q * D), 7.0, dtype=torch.bfloat16, device=self.dev)
        tap = torch.full((self.n + 1, self.n_q * D), 7.0, device=self.dev)
        mask = words_tensor(self.words, self.dev) if mask == "words" else mask
        ops.mha_decode_tree(self.q, self.kc, self.vc, out[:self.n], ws, tree_mask=mask, output_f32=tap[:self.n], **self.scalars(**over))
        torch.cuda.synchronize()
        assert bool((out[self.n] == 7).all()) and bool((tap[self.n] == 7).all())  # nothing behind the last node
        assert torch.equal(out[:self.n].nan_to_num(9.0), tap[:self.n].to(torch.bfloat16).nan_to_num(9.0))
        return tap[:self.n].view(self.n, self.n_q, D)

    def check(self, got, words=None, ctx=None, what=""):
        ctx = self.ctx if ctx is None else ctx
        k, v = (by_head(c[self.layer], self.layout) for c in (self.kc, self.vc))
        want, size = attention64(self.q, k, v, ctx, self.words if words is None else words)
        # (unit rows: a sum of |q k| is at most 128)
        bound = attention_bound(size, ctx + self.n, 1.02 * math.sqrt(D))
        off = (got.double() - want).abs()
        worst = float((off / bound).max())
        assert torch.isfinite(got).all() and worst <= 1, "%s: %.2f of the bound" % (what, worst)


@pytest.mark.parametrize("n_q,n_kv", [(16, 8), (8, 8), (24, 8), (40, 8), (64, 8), (32, 2), (8, 1)])
@pytest.mark.parametrize("n", [1, 2, 5, 17, 64])
def test_heads_and_nodes(dev, n, n_q, n_kv):
    for ctx, layout in ((0, HEAD), (77, POS), (700, HEAD)):
        c = Case(dev, n, n_q, n_kv, ctx, layout, seed=n_q + ctx)
        c.check(c.run(), what="n %d ctx %d layout %d" % (n, ctx, layout))


@pytest.mark.parametrize("layout", [POS, HEAD])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 2049, 5000])
def test_lengths(dev, ctx, layout):
    for n, n_q in ((3, 32), (31, 32), (33, 16)):
        c = Case(dev, n, n_q, 8, ctx, layout, seed=ctx)
        c.check(c.run(), what="n %d n_q %d" % (n, n_q))


@pytest.mark.parametrize("kind", ["chain", "star"])
def test_words(dev, kind):
    c = Case(dev, 40, 32, 8, 150, kind=kind)
    c.check(c.run(), what=kind)
    if kind == "chain":
        assert torch.equal(c.run(), c.run(mask=None))  # NULL is the chain
    # bits from node_num on do not count
    high = [w | (~0 << 40) & (1 << 64) - 1 for w in c.words]
    assert torch.equal(c.run(), c.run(mask=words_tensor(high, dev)))
    # any set of nodes, later ones and not itself included
    odd = [(0x5A5A5A5A5A5A5A5A * (i + 1) >> 3) & (1 << 40) - 1 for i in range(40)]
    c.check(c.run(mask=words_tensor(odd, dev)), words=odd, what="any word")


@pytest.mark.parametrize("ctx", [0, 5, 300])
def test_empty_words(dev, ctx):
    """Nodes that see no node: the cached positions alone, zeros where there are none."""
    n = 20
    words = [0 if i % 3 == 0 else 1 << i for i in range(n)]
    c = Case(dev, n, 32, 8, ctx, words=words)
    got = c.run()
    c.check(got)
    if ctx == 0:
        assert bool((got[::3] == 0).all())


@pytest.mark.parametrize("poison", [NAN, math.inf, -math.inf, -3.3895e38])
@pytest.mark.parametrize("n,n_q,ctx", [(6, 16, 0), (6, 16, 50), (33, 32, 90), (64, 64, 700)])
def test_unseen_rows_leave_no_trace(dev, poison, n, n_q, ctx):
    """Every third node's K and V rows hold what no output may show, and no word but those nodes' own names them."""
    bad = [i for i in range(n) if i % 3 == 1]
    hidden = sum(1 << i for i in bad)
    words = [w & ~hidden | (1 << i if i in bad else 0) for i, w in enumerate(words_of(parents_of(3, n)))]
    c = Case(dev, n, n_q, 8, ctx, words=words)
    clean = c.run()
    for cache in (c.kc, c.vc):
        at = by_head(cache[0], c.layout)
        for i in bad:
            at[:, ctx + i] = poison
    got = c.run()
    good = [i for i in range(n) if i not in bad]
    assert torch.equal(got[good], clean[good])
    if poison != poison:
        assert bool(torch.isnan(got[bad]).all())


def test_seen_values_keep_their_infinities(dev):
    """A V row with an infinity that a node sees gives it that infinity, in that column alone."""
    c = Case(dev, 12, 32, 8, 40, kind="chain")
    by_head(c.vc[0], c.layout)[:, 40 + 4, 17] = math.inf
    got = c.run()
    assert bool((got[4:, :, 17] == math.inf).all()) and bool(torch.isfinite(got[:4]).all())
    rest = [d for d in range(D) if d != 17]
    assert bool(torch.isfinite(got[:, :, rest]).all())


# nodes, query heads, KV heads, cached positions, query rows of a workgroup: every way the kernels take a call (blocks of 16 rows, one and
# several; one block of 32; two, over short and long splits; four, one workgroup and several to a tile)
FORMS = [(5, 16, 8, 50, 16), (26, 32, 8, 500, 16), (8, 32, 8, 9000, 32), (16, 32, 8, 6000, 64), (16, 32, 8, 14000, 64), (26, 32, 8, 6007, 128),
         (61, 32, 8, 3000, 128), (64, 64, 8, 2500, 128), (33, 32, 2, 9000, 128)]


@pytest.mark.parametrize("layout", [POS, HEAD])
@pytest.mark.parametrize("n,n_q,n_kv,ctx,rows_of_group", FORMS)
def test_every_form(dev, n, n_q, n_kv, ctx, rows_of_group, layout):
    """A tree with nodes that hold NaN, infinities and the lowest value for those that do not see them, one empty word; then shorter contexts
    from the device, which the same launch serves."""
    bad = [i for i in range(1, n) if i % 4 == 1]
    hidden = sum(1 << i for i in bad)
    words = [w & ~hidden for w in words_of(parents_of(7, n))]
    words[n - 1] = 0
    c = Case(dev, n, n_q, n_kv, ctx, layout, words=words, seed=n)
    args = B.MhaTreeArgs()
    args.mha = ops.make_mha_args(c.q, c.kc, c.vc, c.q, torch.empty(24 << 20, device=dev), **{k: v for k, v in c.scalars().items() if k != "node_num"})
    args.node_num = n
    plan = B.MhaPlan()
    assert B.lib().llmi_hip_mha_tree_plan(ctypes.byref(args), ctypes.byref(plan)) == 0 and plan.group_pad == rows_of_group
    clean = c.run()
    c.check(clean)
    word = torch.zeros(1, dtype=torch.int32, device=dev)
    for pos in (0, 1, ctx // 2 + 3, ctx - 1):
        word.fill_(pos)
        c.check(c.run(pos_device=word), ctx=pos, what="position %d" % pos)
    for k, i in enumerate(bad):
        for cache in (c.kc, c.vc):
            by_head(cache[0], layout)[:, ctx + i] = [NAN, math.inf, -math.inf, -3.3895e38][k % 4]
    assert torch.equal(c.run(), clean)
    # ... and who sees one value that is not finite has it, in its column alone
    sees = [i for i in range(n) if words[i] & 1]
    by_head(c.vc[0], layout)[:, ctx, 77] = math.inf
    got = c.run()
    assert bool((got[sees][:, :, 77] == math.inf).all()) and torch.equal(got[:, :, :77], clean[:, :, :77]) and torch.equal(got[:, :, 78:], clean[:, :, 78:])
    by_head(c.vc[0], layout)[:, ctx, 77] = NAN
    got = c.run()
    assert bool(torch.isnan(got[sees][:, :, 77]).all()) and torch.equal(got[:, :, :77], clean[:, :, :77]) and torch.equal(got[:, :, 78:], clean[:, :, 78:])


@pytest.mark.parametrize("poison", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("n,n_q,n_kv,ctx,rows_of_group", FORMS)
def test_cached_values_that_are_not_finite(dev, n, n_q, n_kv, ctx, rows_of_group, poison):
    """Every node sees the cached positions: a V row there with an infinity or NaN shows in that column of every output and in no other, in the
    tile that cached positions share with the nodes (the last one) as in those before."""
    assert ctx % 32 != 0
    c = Case(dev, n, n_q, n_kv, ctx, seed=n)
    clean = c.run()
    v = by_head(c.vc[0], c.layout)
    for at in (ctx - 1, ctx - ctx % 32, ctx // 3):
        kept = v[:, at, 77].clone()
        v[:, at, 77] = poison
        got = c.run()
        v[:, at, 77] = kept
        assert not bool(torch.isfinite(got[:, :, 77]).any()), "position %d" % at
        assert torch.equal(got[:, :, :77], clean[:, :, :77]) and torch.equal(got[:, :, 78:], clean[:, :, 78:]), "position %d" % at


def test_overflowing_scores(dev):
    """Scores below the least fp32 number have no weight; a node with no other key gets zeros."""
    c = Case(dev, 8, 16, 8, 0, kind="star")
    k = by_head(c.kc[0], c.layout)
    k[:, :8] = (-3e38 * c.q[:, ::2].transpose(0, 1).sign().float()).to(torch.bfloat16)  # (every node's own key against its first head)
    c.q[:, 1::2] = c.q[:, ::2]
    words = [1 << i for i in range(8)]
    got = c.run(mask=words_tensor(words, dev))
    assert bool((got == 0).all())


@pytest.mark.parametrize("n,n_q,n_kv,ctx", [(5, 32, 8, 3000), (40, 32, 8, 3000), (64, 64, 8, 1500), (7, 8, 1, 4000)])
def test_split_counts(dev, n, n_q, n_kv, ctx):
    c = Case(dev, n, n_q, n_kv, ctx)
    for splits in (1, 2, 3, 7, 16, 61):
        c.check(c.run(num_splits=splits, ws=torch.full((32 << 20,), NAN, device=dev)), what="%d splits" % splits)
    # a workspace that holds fewer splits than the rule would take
    small = torch.full((max(4, ops.tree_workspace_bytes(n_q, D, n) // 4 // 3 // 4 * 4),), NAN, device=dev)
    c.check(c.run(ws=small), what="small workspace")


@pytest.mark.parametrize("layout", [POS, HEAD])
def test_device_position(dev, layout):
    """The word decides, up to the host's bound: the rows from there on are the nodes'."""
    n, ctx = 9, 900
    c = Case(dev, n, 32, 8, ctx, layout)
    word = torch.zeros(1, dtype=torch.int32, device=dev)
    for pos in (0, 1, 31, 64, 500, 899, 900):
        word.fill_(pos)
        c.check(c.run(pos_device=word), ctx=pos, what="position %d" % pos)
    for pos, as_if in ((5000, 900), (-3, 0)):
        word.fill_(pos)
        c.check(c.run(pos_device=word), ctx=as_if, what="position %d" % pos)


def test_captured(dev):
    """One graph for every position, on two workspaces' worth of calls in a row, replayed between other work."""
    n, ctx = 13, 700
    c = Case(dev, n, 32, 8, ctx)
    word = torch.full((1,), ctx, dtype=torch.int32, device=dev)
    mask = words_tensor(c.words, dev)
    ws = torch.full((ops.tree_workspace_bytes(32, D, n) // 4 + 4,), NAN, device=dev)
    outs = [torch.zeros(n, 32 * D, device=dev) for _ in range(2)]
    low = torch.zeros(n, 32 * D, dtype=torch.bfloat16, device=dev)

    def step(out):
        ops.mha_decode_tree(c.q, c.kc, c.vc, low, ws, tree_mask=mask, output_f32=out, pos_device=word, **c.scalars())

    step(outs[0])
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(outs[0])
    with torch.cuda.graph(second):  # (shares the workspace)
        step(outs[1])
    for pos in (700, 3, 333, 0, 64, 699, 700):
        word.fill_(pos)
        for out in outs:
            out.fill_(NAN)
        graph.replay()
        second.replay()
        graph.replay()
        torch.cuda.synchronize()
        eager = c.run(pos_device=word)
        assert torch.equal(outs[0].view_as(eager), eager) and torch.equal(outs[1].view_as(eager), eager)


def test_same_bits_every_time(dev):
    c = Case(dev, 50, 32, 8, 6000)
    first = c.run()
    for _ in range(5):
        assert torch.equal(first, c.run())


def test_streams(dev):
    """Two streams with a workspace each, side by side."""
    a, b = Case(dev, 9, 32, 8, 2500, seed=5), Case(dev, 64, 32, 8, 2500, seed=6)
    want = [a.run(), b.run()]
    got = [[], []]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for i, (c, s) in enumerate(zip((a, b), streams)):
            out, tap = torch.zeros(c.n, c.n_q * D, dtype=torch.bfloat16, device=dev), torch.zeros(c.n, c.n_q * D, device=dev)
            ws, mask = torch.full((ops.tree_workspace_bytes(32, D, c.n) // 4 + 4,), NAN, device=dev), words_tensor(c.words, dev)
            s.wait_stream(torch.cuda.current_stream())
            ops.mha_decode_tree(c.q, c.kc, c.vc, out, ws, tree_mask=mask, output_f32=tap, stream=s, **c.scalars())
            got[i].append((tap, out, ws, mask))
    torch.cuda.synchronize()
    for i in range(2):
        for tap, _, _, _ in got[i]:
            assert torch.equal(tap.view_as(want[i]), want[i])


@pytest.mark.parametrize("layout", [POS, HEAD])
def test_offsets_past_32_bits(dev, layout):
    """The last layer of a cache of more than 2^32 bytes and 2^31 elements."""
    c = Case(dev, 6, 16, 8, 131000, layout, layers=17, layer=16, spare=66)
    c.check(c.run())


def test_one_node_is_a_decode_step(dev):
    """Against llmi_hip_mha_decode, which the same bound holds for."""
    c = Case(dev, 1, 32, 8, 1234)
    out, tap = torch.zeros(32 * D, dtype=torch.bfloat16, device=dev), torch.zeros(32 * D, device=dev)
    ws = torch.empty(ops.workspace_bytes(32, D, c.msl) // 4, device=dev)
    kw = c.scalars()
    del kw["node_num"]
    ops.mha_decode(c.q[0], c.kc, c.vc, out, ws, output_f32=tap, **kw)
    torch.cuda.synchronize()
    c.check(c.run())
    c.check(tap.view(1, 32, D))
