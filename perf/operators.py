"""The operators of a speculative decoding step, as measurable cases.

A step of a Qwen3-shaped model at batch 1 that checks a tree (or a chain) of drafted tokens in one pass: the nodes' rows
normalised, rotated by their depth and filed behind the cached positions ("append"), attention of all nodes over the cache and
their ancestors ("attend"), the drafts verified against the target's logits from given random numbers ("verify"), and the
accepted nodes' rows brought to where a decode step expects them, in all layers ("commit").

`listed()` holds the measured cases, `draw()` gives more of the same ranges, `prepare()` makes what a program has in hand before
the call, `run()` is one pass: with `own` the calls of llminfer_amd.ops, otherwise the same in elementary torch operations.
`exact()` is the definition in 64 bits, `work()` the bytes and operations a pass cannot do without.
"""
import math
import random

import numpy as np
import torch

own = False

HEAD_DIM = 128
EPS = 1e-6
BF16, F32 = torch.bfloat16, torch.float32
MOST_NODES = 64
# What a program keeps for the attention's partial results and the verification's: enough for every case below.
WORKSPACE_BYTES = 96 << 20
# Query heads, KV heads: the Qwen3-0.6B, Qwen3-4B and Qwen3-32B layer shapes ...
MODELS = [(16, 8), (32, 8), (64, 8)]
# ... and the head layouts that else occur: shards by KV head, one query head per KV head, odd groups.
OTHER_HEADS = [(16, 4), (16, 2), (8, 2), (8, 1), (8, 8), (24, 8), (40, 8), (32, 2)]


def listed():
    return [
        # a short chat on the smallest model, four tokens drafted by a smaller one: nothing but latency
        dict(name="attend-16q8kv-57-chain5", kind="attend", n_q=16, n_kv=8, ctx=57, nodes=5, tree=False, max_seq_len=4096, layout="head"),
        # a chain of seven drafts a few thousand tokens in: the cache is read, the rows are few
        dict(name="attend-32q8kv-4099-chain8", kind="attend", n_q=32, n_kv=8, ctx=4099, nodes=8, tree=False, max_seq_len=8192, layout="head"),
        # a small tree in the reference engine's own cache layout
        dict(name="attend-32q8kv-6007-tree26-pos", kind="attend", n_q=32, n_kv=8, ctx=6007, nodes=26, tree=True, max_seq_len=8192,
             layout="pos"),
        # a full tree over a long context: as much arithmetic as memory
        dict(name="attend-32q8kv-32768-tree61", kind="attend", n_q=32, n_kv=8, ctx=32768, nodes=61, tree=True, max_seq_len=33024,
             layout="head"),
        # the largest: full tree, largest model, longest context
        dict(name="attend-64q8kv-131000-tree64", kind="attend", n_q=64, n_kv=8, ctx=131000, nodes=64, tree=True, max_seq_len=131072,
             layout="head"),
        # the rows of a short chain, smallest model
        dict(name="append-16q8kv-chain5", kind="append", n_q=16, n_kv=8, ctx=1000, nodes=5, tree=False, max_seq_len=4096, layout="head"),
        # the rows of a full tree, largest model, cut out of the projection's packed result
        dict(name="append-64q8kv-tree64-pos", kind="append", n_q=64, n_kv=8, ctx=5003, nodes=64, tree=True, max_seq_len=8192, layout="pos"),
        # tokens sampled from a draft model and its own logits: the ratio test and the rest of the target's mass
        dict(name="verify-draft-chain6-32000", kind="verify", mode="draft", nodes=6, vocab=32000, temperature=1.0, keep=0, dtype="f32"),
        # the most likely tokens of a tree checked for what the target itself would take
        dict(name="verify-greedy-tree26-151936", kind="verify", mode="tree", nodes=26, vocab=151936, temperature=0.0, keep=0, dtype="f32"),
        # a full tree, sampled, from half-precision logits that a top-k filter has cut to 50 tokens
        dict(name="verify-tree64-151936-top50", kind="verify", mode="tree", nodes=64, vocab=151936, temperature=0.7, keep=50, dtype="bf16"),
        # four of a tree's nodes stay, all layers of the middle model
        dict(name="commit-36x8kv-4of26", kind="commit", n_kv=8, layers=36, ctx=1500, nodes=26, path=4, max_seq_len=2048, layout="head"),
        # a long accepted path, all layers of the largest model, the reference's layout
        dict(name="commit-64x8kv-11of64-pos", kind="commit", n_kv=8, layers=64, ctx=700, nodes=64, path=11, max_seq_len=1024, layout="pos"),
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; odd ones as likely as even ones."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _window(rng, used):
    """Positions a cache is sized for: the context window, a round number, or just what is needed."""
    return rng.choice([max(4096, -(-used // 4096) * 4096), -(-used // 1024) * 1024, used + rng.randrange(0, 40)])


def draw(rng):
    kind = rng.choice(["attend"] * 6 + ["append", "verify", "verify", "verify", "commit"])
    n_q, n_kv = rng.choice(MODELS if rng.random() < 0.6 else OTHER_HEADS)
    nodes = _log_int(rng, 1, MOST_NODES)
    layout = rng.choice(["head", "head", "pos"])
    if kind in ("attend", "append"):
        ctx = _log_int(rng, 1, 131000) - (rng.random() < 0.1)
        return dict(kind=kind, n_q=n_q, n_kv=n_kv, ctx=ctx, nodes=nodes, tree=rng.random() < 0.6,
                    max_seq_len=_window(rng, ctx + nodes), layout=layout)
    if kind == "verify":
        vocab = _log_int(rng, 100, 152000)
        mode = rng.choice(["tree", "tree", "chain", "draft"])
        temperature = rng.choice([0.0, 0.6, 1.0, 1.3]) if mode != "draft" else rng.choice([0.6, 1.0, 1.3])
        return dict(kind=kind, mode=mode, nodes=nodes, vocab=vocab, temperature=temperature,
                    keep=rng.choice([0, 0, _log_int(rng, 5, 90)]), dtype=rng.choice(["f32", "f32", "bf16"]))
    layers = _log_int(rng, 1, 64)
    nodes = max(2, nodes)
    ctx = _log_int(rng, 1, 900)
    return dict(kind=kind, n_kv=n_kv, layers=layers, ctx=ctx, nodes=nodes, path=rng.randint(1, min(nodes, 16)),
                max_seq_len=ctx + nodes + rng.randrange(0, 40), layout=layout)


class _Inputs:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.gen = torch.Generator(device=self.dev)
        self.gen.manual_seed(seed)
        self.rng = random.Random(seed)

    def normal(self, *shape, scale=1.0, mean=0.0, dtype=BF16):
        x = torch.randn(shape, generator=self.gen, device=self.dev, dtype=dtype)
        if scale != 1.0:
            x.mul_(scale)
        return x.add_(mean) if mean else x

    def unit_rows(self, *shape):
        """Rows as QK-Norm leaves them: unit root mean square over a head's 128 values."""
        x = self.normal(*shape)
        f = x.float()
        return x.copy_(f * torch.rsqrt(f.square().mean(-1, keepdim=True)))

    def ints(self, values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device=self.dev)


def _parents(rng, nodes, tree):
    """Node 0 is the last token that is certain, a node's parent comes before it: a chain, or a tree grown near its newest nodes."""
    return [-1] + [rng.randrange(max(0, i - 9), i) if tree else i - 1 for i in range(1, nodes)]


def _bits(parents):
    """For every node the set of nodes it sees, itself and its ancestors, as a 64-bit word."""
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return [b - (1 << 64) if b >> 63 else b for b in seen]


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return depth


def _cache_shape(case, layers):
    n_kv, msl = case["n_kv"], case["max_seq_len"]
    return (layers, msl, n_kv, HEAD_DIM) if case["layout"] == "pos" else (layers, n_kv, msl, HEAD_DIM)


def _workspace(rnd):
    return torch.empty(WORKSPACE_BYTES // 4, dtype=F32, device=rnd.dev)


def prepare(case, seed):
    rnd, kind = _Inputs(seed), case["kind"]
    s = {"kind": kind, "case": case, "nodes": case["nodes"]}
    if kind == "verify":
        return _prepare_verify(case, rnd, s)
    shape = _cache_shape(case, case.get("layers", 1))
    s["kc"], s["vc"] = rnd.unit_rows(*shape), rnd.normal(*shape)
    s["pos"], s["n_kv"] = case["ctx"], case["n_kv"]
    s["cache"] = dict(pos=case["ctx"], node_num=case["nodes"], kv_dim=case["n_kv"] * HEAD_DIM, head_dim=HEAD_DIM,
                      max_seq_len=case["max_seq_len"], kv_layout={"pos": 0, "head": 1}[case["layout"]])
    if kind == "commit":
        # node 0, some that are in their places already, and others from further back than the path is long (so a pass can be
        # repeated: it reads nothing that it has written)
        k = case["path"]
        stay = rnd.rng.randint(1, k)
        stay = k if case["nodes"] - k < k - stay else stay
        path = list(range(stay)) + sorted(rnd.rng.sample(range(k, case["nodes"]), k - stay))
        s["path"] = rnd.ints(path + [-1] * (case["nodes"] - k))
        s["result"] = rnd.ints([k, 17])
        return s
    parents = _parents(rnd.rng, case["nodes"], case["tree"])
    n_q, n_kv, n = case["n_q"], case["n_kv"], case["nodes"]
    s["n_q"] = n_q
    if kind == "attend":
        s["mask"] = rnd.ints(_bits(parents), torch.int64)
        s["q"], s["out"] = rnd.unit_rows(n, n_q, HEAD_DIM), torch.zeros(n, n_q * HEAD_DIM, dtype=BF16, device=rnd.dev)
        s["ws"] = _workspace(rnd)
        return s
    # the three projections of all nodes as one product leaves them, a node's query, key and value behind one another
    packed = rnd.normal(n, (n_q + 2 * n_kv) * HEAD_DIM)
    s["q_raw"], s["k_raw"], s["v_raw"] = packed.split([n_q * HEAD_DIM, n_kv * HEAD_DIM, n_kv * HEAD_DIM], dim=1)
    s["q"] = torch.zeros(n, n_q * HEAD_DIM, dtype=BF16, device=rnd.dev)
    s["norm"] = rnd.normal(2 * HEAD_DIM, scale=0.02, mean=1.0)
    freq = torch.exp(torch.arange(HEAD_DIM // 2, device=rnd.dev, dtype=torch.float64) * (-2.0 / HEAD_DIM * math.log(1e6)))
    angle = torch.arange(case["max_seq_len"], device=rnd.dev, dtype=torch.float64)[:, None] * freq
    s["sin"], s["cos"] = angle.sin().float(), angle.cos().float()
    s["depth"] = rnd.ints(_depths(parents))
    return s


def _prepare_verify(case, rnd, s):
    n, vocab, mode = case["nodes"], case["vocab"], case["mode"]
    parents = _parents(rnd.rng, n, mode == "tree")
    target = rnd.normal(n, vocab, scale=3.0, dtype=F32)
    draft = target + rnd.normal(n, vocab, scale=0.6, dtype=F32)
    if case["keep"]:  # what a top-k filter leaves of the target's logits
        least = target.topk(min(case["keep"], vocab), dim=-1).values[:, -1:]
        target = target.masked_fill(target < least, -math.inf)
    dtype = F32 if case["dtype"] == "f32" else BF16
    target, draft = target.to(dtype), draft.to(dtype)
    # the drafted tokens: sampled from the draft's distribution, or the most likely ones by the draft's logits, sibling by sibling
    at = [max(p, 0) for p in parents]
    if mode == "draft":
        probs = (draft.float() / case["temperature"]).softmax(-1)
        tokens = torch.multinomial(probs, 1, generator=rnd.gen)[:, 0][rnd.ints(at, torch.int64)]
        s["draft"] = draft
    else:
        rank = [min(at[:i].count(p), vocab - 1) for i, p in enumerate(at)]
        best = draft.float().topk(max(rank) + 1, dim=-1).indices
        tokens = best[rnd.ints(at, torch.int64), rnd.ints(rank, torch.int64)]
        s["draft"] = None
    s["target"], s["tokens"], s["vocab"], s["temperature"] = target, tokens.to(torch.int32).contiguous(), vocab, case["temperature"]
    s["parents"] = rnd.ints(parents) if mode == "tree" else None
    s["parent_of"], s["mask"] = rnd.ints(at, torch.int64), rnd.ints(_bits(parents), torch.int64)
    s["uniform"] = torch.rand(n, generator=rnd.gen, device=rnd.dev)
    s["path"], s["result"] = rnd.ints([0] * n), rnd.ints([0, 0])
    s["ws"] = _workspace(rnd)
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"attend": _attend, "append": _append, "verify": _verify, "commit": _commit}[s["kind"]](s)


def _run_own(s):
    from llminfer_amd import ops
    kind = s["kind"]
    if kind == "attend":
        return ops.mha_decode_tree(s["q"], s["kc"], s["vc"], s["out"], s["ws"], tree_mask=s["mask"], layer_id=0, kv_mul=s["n_q"] // s["n_kv"],
                                   head_num=s["n_q"], **s["cache"])
    if kind == "append":
        ops.qk_norm_rope_append_tree(s["q"], s["k_raw"], s["v_raw"], s["kc"], s["vc"], s["norm"], s["sin"], s["cos"], query_src=s["q_raw"],
                                     depth=s["depth"], layer_id=0, head_num=s["n_q"], **s["cache"])
        return {"query": s["q"], "keys": s["kc"], "values": s["vc"]}
    if kind == "verify":
        ops.verify_tree(s["target"], s["tokens"], s["uniform"], s["path"], s["result"], s["ws"], parents=s["parents"], draft_logits=s["draft"],
                        temperature=s["temperature"])
        return {"path": s["path"], "result": s["result"]}
    ops.kv_commit_tree(s["kc"], s["vc"], s["path"], s["result"], layer_num=s["case"]["layers"], **s["cache"])
    return {"keys": s["kc"], "values": s["vc"]}


def _by_position(s, cache):
    """[layers][position][KV head][128], as a view."""
    return cache if s["case"]["layout"] == "pos" else cache.transpose(1, 2)


def _allowed(s):
    """Which node sees which, from the nodes' words."""
    at = torch.arange(s["nodes"], device=s["mask"].device)
    return (s["mask"][:, None] >> at) & 1 == 1


def _attend(s):
    n, n_q, n_kv, ctx = s["nodes"], s["n_q"], s["n_kv"], s["pos"]
    used = ctx + n
    k, v = (_by_position(s, c)[0, :used].transpose(0, 1).float().contiguous() for c in (s["kc"], s["vc"]))  # [KV head][position][128]
    q = s["q"].view(n, n_kv, n_q // n_kv, HEAD_DIM).permute(1, 0, 2, 3).reshape(n_kv, -1, HEAD_DIM).float()
    score = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(HEAD_DIM ** -0.5).view(n_kv, n, n_q // n_kv, used)
    score[..., ctx:].masked_fill_(~_allowed(s)[None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(F32).min)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(n_kv, -1, used), v).view(n_kv, n, n_q // n_kv, HEAD_DIM) / total.clamp_min(torch.finfo(F32).tiny)
    return out.permute(1, 0, 2, 3).reshape(n, n_q * HEAD_DIM).to(BF16)


def _rotated(x, weight, sin, cos):
    """RMS norm over a head's 128 values, then the rotation of the pairs (i, i + 64)."""
    f = x.float()
    f = f * weight.float() * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    a, b = f[..., :HEAD_DIM // 2], f[..., HEAD_DIM // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(BF16)


def _append(s):
    n, pos = s["nodes"], s["pos"]
    at = (pos + s["depth"]).long()
    sin, cos = s["sin"][at][:, None], s["cos"][at][:, None]
    keys, values = _by_position(s, s["kc"])[0], _by_position(s, s["vc"])[0]
    keys[pos:pos + n] = _rotated(s["k_raw"].reshape(n, -1, HEAD_DIM), s["norm"][HEAD_DIM:], sin, cos)
    values[pos:pos + n] = s["v_raw"].reshape(n, -1, HEAD_DIM)
    s["q"].copy_(_rotated(s["q_raw"].reshape(n, -1, HEAD_DIM), s["norm"][:HEAD_DIM], sin, cos).view(n, -1))
    return {"query": s["q"], "keys": s["kc"], "values": s["vc"]}


def _first(true, width):
    """The lowest place that is true along the last dimension, `width` if none is."""
    return torch.where(true, torch.arange(width, device=true.device), width).amin(-1)


def _verify(s):
    # In 64 bits: tests and sums next to a border have to fall on the same side.
    n, vocab, dev = s["nodes"], s["vocab"], s["target"].device
    at, token, u = s["parent_of"], s["tokens"].long(), s["uniform"].double()
    node = torch.arange(n, device=dev)
    sibling = (at[:, None] == at[None, :]) & (node[None, :] < node[:, None]) & (node[None, :] > 0)  # [i][j]: j an earlier sibling of i
    logits = s["target"].double()
    top = logits.amax(-1, keepdim=True)
    likeliest = _first(logits == top, vocab)
    if s["temperature"] == 0:
        accepted = token == likeliest[at]
    else:
        weight = ((logits - top) / s["temperature"]).exp()
        total = weight.sum(-1)
        mass = weight[at, token]
        if s["draft"] is None:
            again = (sibling & (token[:, None] == token[None, :])).any(-1)
            before = (sibling & ~again[None, :]).double() @ mass
            accepted = (u * (total[at] - before) < mass) & ~again
        else:
            d = s["draft"].double()
            p, q = weight / total[:, None], ((d - d.amax(-1, keepdim=True)) / s["temperature"]).softmax(-1)
            accepted = u * q[at, token] < p[at, token]
    taken = accepted & ~(sibling & accepted[None, :]).any(-1)
    taken[0] = True
    on_path = ~(_allowed(s) & ~taken[None, :]).any(-1)
    path = torch.where(on_path, node, n).sort().values
    last = torch.where(on_path, node, 0).amax()
    if s["temperature"] == 0:
        following = likeliest[last]
    else:
        if s["draft"] is None:
            refused = torch.zeros(vocab, device=dev, dtype=torch.float64).index_add_(0, token, ((at == last) & (node > 0)).double())
            left = weight[last] * (refused == 0)
        else:
            left = torch.where(last < n - 1, (p[last] - q[last]).clamp_min(0), p[last])
        sums = left.cumsum(0)
        following = _first(sums > u[0] * sums[-1], vocab)
    s["path"].copy_(torch.where(path < n, path, -1))
    s["result"].copy_(torch.stack([on_path.sum(), following]))
    return {"path": s["path"], "result": s["result"]}


def _commit(s):
    n, pos = s["nodes"], s["pos"]
    place = torch.arange(n, device=s["path"].device)
    source = torch.where(place < s["result"][0], s["path"].long(), place) + pos
    for cache in (s["kc"], s["vc"]):
        rows = _by_position(s, cache)
        rows[:, pos:pos + n] = rows[:, source]
    return {"keys": s["kc"], "values": s["vc"]}


def work(case):
    kind, n = case["kind"], case["nodes"]
    if kind == "verify":
        rows = n * (2 if case["mode"] == "draft" else 1)
        return {"bytes": rows * case["vocab"] * (4 if case["dtype"] == "f32" else 2) + 16 * n, "flops": 4 * rows * case["vocab"]}
    row = case["n_kv"] * HEAD_DIM * 2
    if kind == "commit":
        return {"bytes": 2 * 2 * case["layers"] * (case["path"] - 1) * row + 4 * n, "flops": 0}
    head_bytes = 2 * n * case["n_q"] * HEAD_DIM * 2  # queries in, outputs or queries out
    if kind == "append":
        return {"bytes": head_bytes + 4 * n * row + n * (2 * HEAD_DIM // 2 * 4) + 4 * HEAD_DIM, "flops": 10 * n * (case["n_q"] + case["n_kv"]) * HEAD_DIM}
    used = case["ctx"] + n
    return {"bytes": 2 * used * row + head_bytes + 8 * n, "flops": 4 * n * case["n_q"] * HEAD_DIM * used}


def exact(case, seed):
    """What run() returns for these inputs, from the definitions, in 64 bits."""
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "verify": _exact_verify, "commit": _exact_commit}[case["kind"]](case, s)


def _head_rows(case, cache, layer, head):
    """[position][128] of one KV head, as a view."""
    return cache[layer, :, head] if case["layout"] == "pos" else cache[layer, head]


def _exact_attend(case, s):
    n, group, ctx = case["nodes"], case["n_q"] // case["n_kv"], case["ctx"]
    out = torch.zeros(n, case["n_q"], HEAD_DIM, dtype=torch.float64, device=s["q"].device)
    words = [int(w) & (1 << 64) - 1 for w in s["mask"].tolist()]
    sees = torch.ones(n, ctx + n, dtype=torch.bool, device=s["q"].device)
    sees[:, ctx:] = torch.tensor([[bool(w >> j & 1) for j in range(n)] for w in words], device=s["q"].device)
    for head in range(case["n_kv"]):
        k = _head_rows(case, s["kc"], 0, head)[:ctx + n].double()
        v = _head_rows(case, s["vc"], 0, head)[:ctx + n].double()
        for hq in range(head * group, (head + 1) * group):
            logit = (s["q"][:, hq].double() @ k.t().contiguous()) / math.sqrt(HEAD_DIM)
            logit[~sees] = -math.inf
            log_sum = torch.logsumexp(logit, -1, keepdim=True)
            out[:, hq] = torch.exp(logit - log_sum) @ v
    return out.view(n, -1)


def _exact_append(case, s):
    n, pos, half = case["nodes"], case["ctx"], HEAD_DIM // 2
    at = [pos + d for d in s["depth"].tolist()]

    def turn(rows, weight):
        x = rows.reshape(n, -1, HEAD_DIM).double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / HEAD_DIM + EPS) * weight.double()
        z = torch.complex(y[..., :half], y[..., half:])
        z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        return torch.cat([z.real, z.imag], -1)

    keys, values = s["kc"].double(), s["vc"].double()
    k_new, v_new = turn(s["k_raw"], s["norm"][HEAD_DIM:]), s["v_raw"].reshape(n, -1, HEAD_DIM).double()
    for head in range(case["n_kv"]):
        _head_rows(case, keys, 0, head)[pos:pos + n] = k_new[:, head]
        _head_rows(case, values, 0, head)[pos:pos + n] = v_new[:, head]
    return {"query": turn(s["q_raw"], s["norm"][:HEAD_DIM]).reshape(n, -1), "keys": keys, "values": values}


def _exact_verify(case, s):
    """Node by node, as the definition goes, on the host."""
    target = s["target"].double().cpu().numpy()
    draft = None if s["draft"] is None else s["draft"].double().cpu().numpy()
    parent, token, u = s["parent_of"].tolist(), s["tokens"].tolist(), s["uniform"].double().tolist()
    n, heat = case["nodes"], case["temperature"]

    def chances(row):
        w = np.exp((row - row.max()) / heat)
        return w / w.sum()

    at, path = 0, [0]
    while True:
        left = None if heat == 0 else chances(target[at])
        follow = None
        for c in range(1, n):
            if parent[c] != at:
                continue
            if heat == 0:
                yes = token[c] == int(np.argmax(target[at]))
            elif draft is None:
                yes = left[token[c]] > 0 and u[c] * left.sum() < left[token[c]]
                if not yes:
                    left[token[c]] = 0.0
            else:
                q = chances(draft[at])
                yes = u[c] * q[token[c]] < left[token[c]]
                if not yes:
                    left = np.maximum(left - q, 0.0)
            if yes:
                follow = c
                break
        if follow is None:
            break
        at = follow
        path.append(at)
    if heat == 0:
        following = int(np.argmax(target[at]))
    else:
        sums = np.cumsum(left)
        following = int(np.searchsorted(sums, u[0] * sums[-1], side="right"))
    return {"path": torch.tensor(path + [-1] * (n - len(path)), dtype=torch.int32), "result": torch.tensor([len(path), following], dtype=torch.int32)}


def _exact_commit(case, s):
    pos, path = case["ctx"], s["path"].tolist()[:case["path"]]
    found = {}
    for name, cache in (("keys", s["kc"]), ("values", s["vc"])):
        old, new = cache, cache.clone()
        for i, node in enumerate(path):
            if case["layout"] == "pos":
                new[:, pos + i] = old[:, pos + node]
            else:
                new[:, :, pos + i] = old[:, :, pos + node]
        found[name] = new
    return found
