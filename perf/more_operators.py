"""The operators of an 8-bit KV cache, as measurable cases.

A Qwen3-shaped model at batch 1 whose K and V rows are kept as 8-bit codes with a scale per row: the rows of new tokens
normalised, rotated and quantised as they are filed ("rows"), attention of one token that reads the codes ("decode"), both in one
call ("step"), and whole ranges of a bf16 cache quantised ("store") and read back ("load").

A row (128 values of a KV head's K or V at a position, as bf16) is 128 codes and a scale s: the smallest number of eight significant
bits with s * top >= the row's largest magnitude, 2^-64 at least; top is 448 for E4M3 codes, 127 for whole numbers. A code is x / s
rounded to the nearest one, ties to even. Rows are kept in records of 32 positions (position 16 t + 4 g + i): 4096 bytes of K codes
[p / 16][16-channel chunk][p % 16][16], 4096 of V codes [channel / 32][g][channel % 16][channel / 16 % 2][t][i], then the scales of K
and of V as bf16 [g][t][i]. The cache is [layer][KV head][record].

`listed()` holds the measured cases, `draw()` gives more of the same ranges, `prepare()` makes what a program has in hand before
the call, `run()` is one pass: with `own` the calls of llminfer_amd.ops, otherwise the same in elementary torch operations.
`exact()` is the definition in 64 bits, `work()` the bytes and operations a pass cannot do without.
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
EPS = 1e-6
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
RECORD, PLACES = 8320, 32  # bytes of a record, positions in it
TOP = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LEAST = 2.0 ** -64
# What a program keeps for the attention's partial results: enough for every case below.
WORKSPACE_BYTES = 96 << 20
# Query heads, KV heads: the Qwen3-0.6B, Qwen3-4B and Qwen3-32B layer shapes ...
MODELS = [(16, 8), (32, 8), (64, 8)]
# ... and the head layouts that else occur: shards by KV head, one query head per KV head, odd groups and counts.
OTHER_HEADS = [(8, 1), (8, 2), (16, 1), (16, 2), (32, 2), (40, 8), (5, 5), (48, 4), (33, 3)]


def listed():
    return [
        # a short chat on the smallest model: nothing but latency
        dict(name="decode-16q8kv-57-e4m3", kind="decode", n_q=16, n_kv=8, ctx=57, max_seq_len=4096, codes="e4m3", device=False),
        # a few thousand tokens in, whole-number codes
        dict(name="decode-32q8kv-6007-int8", kind="decode", n_q=32, n_kv=8, ctx=6007, max_seq_len=8192, codes="int8", device=False),
        # the longest context of the largest model: all memory
        dict(name="decode-64q8kv-131000-e4m3", kind="decode", n_q=64, n_kv=8, ctx=131000, max_seq_len=131072, codes="e4m3", device=False),
        # a layer's call of an eager decode step, short context
        dict(name="step-16q8kv-300-e4m3", kind="step", n_q=16, n_kv=8, ctx=300, max_seq_len=4096, codes="e4m3", device=False),
        # a layer's call of a captured step: the position is in device memory, the launch is sized for the window
        dict(name="step-32q8kv-4099-e4m3-device", kind="step", n_q=32, n_kv=8, ctx=4099, max_seq_len=8192, codes="e4m3", device=True),
        # a long document
        dict(name="step-32q8kv-32768-e4m3", kind="step", n_q=32, n_kv=8, ctx=32768, max_seq_len=33024, codes="e4m3", device=False),
        # the rows of one token, for a program that calls the attention by itself
        dict(name="rows-16q8kv-1-e4m3", kind="rows", n_q=16, n_kv=8, ctx=1000, rows=1, max_seq_len=4096, codes="e4m3"),
        # a chunk of a prompt, cut out of the projections' packed result
        dict(name="rows-32q8kv-1001-e4m3", kind="rows", n_q=32, n_kv=8, ctx=2013, rows=1001, max_seq_len=4096, codes="e4m3"),
        # a short prompt, prefilled in bf16 in the reference engine's own layout, goes to 8 bits
        dict(name="store-28x8kv-500-int8-pos", kind="store", n_kv=8, layers=28, first=0, count=500, max_seq_len=1024, codes="int8", layout="pos"),
        # a long one, all layers of the middle model
        dict(name="store-36x8kv-3777-e4m3", kind="store", n_kv=8, layers=36, first=0, count=3777, max_seq_len=4096, codes="e4m3", layout="head"),
        # the last positions back to bf16, for a program that works on them there
        dict(name="load-28x8kv-200-e4m3-pos", kind="load", n_kv=8, layers=28, first=811, count=200, max_seq_len=1024, codes="e4m3", layout="pos"),
        # everything back
        dict(name="load-36x8kv-3777-int8", kind="load", n_kv=8, layers=36, first=0, count=3777, max_seq_len=4096, codes="int8", layout="head"),
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; odd ones as likely as even ones."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _window(rng, used):
    """Positions a cache is sized for: the context window, a round number, or just what is needed."""
    return rng.choice([max(4096, -(-used // 4096) * 4096), -(-used // 1024) * 1024, used + rng.randrange(0, 40)])


def draw(rng):
    kind = rng.choice(["decode"] * 4 + ["step"] * 4 + ["rows", "rows", "store", "store", "load", "load"])
    n_q, n_kv = rng.choice(MODELS if rng.random() < 0.6 else OTHER_HEADS)
    if kind in ("decode", "step"):
        ctx = _log_int(rng, 1, 131000) - (rng.random() < 0.1)
        # (a step's codes are compared one by one, and whole numbers as equal or not; a K value next to a border of theirs falls by the
        # last bit of its row's root mean square. The two kinds of codes differ in nothing but the conversion.)
        codes = rng.choice(["e4m3", "int8"]) if kind == "decode" else "e4m3"
        return dict(kind=kind, n_q=n_q, n_kv=n_kv, ctx=ctx, max_seq_len=_window(rng, ctx + 1), codes=codes, device=rng.random() < 0.3)
    if kind == "rows":
        ctx, rows = _log_int(rng, 1, 9000) - 1, _log_int(rng, 1, 1001)
        return dict(kind=kind, n_q=n_q, n_kv=n_kv, ctx=ctx, rows=rows, max_seq_len=_window(rng, ctx + rows), codes="e4m3")
    layers = _log_int(rng, 1, 64)
    count = _log_int(rng, 1, max(1, 36 * 8 * 3777 // (layers * n_kv * 2)))
    first = rng.choice([0, 0, _log_int(rng, 1, 1000)])
    return dict(kind=kind, n_kv=n_kv, layers=layers, first=first, count=count, max_seq_len=first + count + rng.choice([0, rng.randrange(0, 200)]),
                codes=rng.choice(["e4m3", "int8"]), layout=rng.choice(["head", "head", "pos"]))


class _Inputs:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.gen = torch.Generator(device=self.dev)
        self.gen.manual_seed(seed)

    def normal(self, *shape, scale=1.0, mean=0.0, dtype=BF16):
        x = torch.randn(shape, generator=self.gen, device=self.dev, dtype=dtype)
        if scale != 1.0:
            x.mul_(scale)
        return x.add_(mean) if mean else x

    def keys(self, *shape):
        """Rows as QK-Norm leaves them: unit root mean square over a head's 128 values, some channels several times the others."""
        x = self.normal(*shape)
        gain = 1.0 + 3.0 * (torch.rand(shape[-1], generator=self.gen, device=self.dev) < 0.05)
        f = x.float() * gain
        return x.copy_(f * torch.rsqrt(f.square().mean(-1, keepdim=True)))


def _places(dev):
    """Where a record keeps what belongs to its positions: bytes of the K and V codes [32][128], bf16 words of the K and V scales [32]."""
    p, c = torch.arange(PLACES, device=dev)[:, None], torch.arange(HEAD_DIM, device=dev)[None, :]
    t, g, i = p // 16, p // 4 % 4, p % 4
    key = t * 2048 + c // 16 * 256 + p % 16 * 16 + c % 16
    value = 4096 + c // 32 * 1024 + g * 256 + c % 16 * 16 + c // 16 % 2 * 8 + t * 4 + i
    scale = (4096 + g * 8 + t * 4 + i)[:, 0]
    return (key, scale), (value, scale + 32)


def _at(case, first, count, dev):
    """Records and places in them of `count` positions from `first` on."""
    at = torch.arange(first, first + count, device=dev)
    return at // PLACES, at % PLACES


def _quantised(x, codes):
    """Codes (as bytes) and scales of rows of 128. In 64 bits, and divided by tensors (a division by a number is a product with its
    reciprocal): both have to fall on the right side of their borders."""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    least = (most / torch.full_like(most, TOP[codes])).float().view(torch.int32)
    s = (least + 0xffff >> 16 << 16).view(F32).clamp_min(LEAST)
    q = (x / s.double()).float()
    return (q.to(torch.float8_e4m3fn) if codes == "e4m3" else q.round().to(torch.int8)).view(torch.uint8), s.to(BF16)


def _file(case, cache, first, rows, which):
    """Quantises rows [layer][KV head][position][128] into the cache, from position `first` on."""
    record, place = _at(case, first, rows.shape[2], cache.device)
    at, scale_at = _places(cache.device)[which]
    q, s = _quantised(rows, case["codes"])
    cache[:, :, record[:, None], at[place]] = q
    cache.view(BF16)[:, :, record, scale_at[place]] = s[..., 0]


def _fetch(case, cache, first, count, which):
    """What the codes of the positions stand for, [layer][KV head][position][128] in 32 bits."""
    record, place = _at(case, first, count, cache.device)
    at, scale_at = _places(cache.device)[which]
    q = cache[:, :, record[:, None], at[place]].view(CODE[case["codes"]])
    return q.float() * cache.view(BF16)[:, :, record, scale_at[place]].float()[..., None]


def prepare(case, seed):
    rnd, kind, n_kv, msl = _Inputs(seed), case["kind"], case["n_kv"], case["max_seq_len"]
    layers = case.get("layers", 1)
    cache = torch.zeros(layers, n_kv, -(-msl // PLACES), RECORD, dtype=torch.uint8, device=rnd.dev)
    s = {"kind": kind, "case": case, "cache": cache, "dims": dict(kv_dim=n_kv * HEAD_DIM, head_dim=HEAD_DIM, max_seq_len=msl, kv8_format=["e4m3", "int8"].index(case["codes"]))}
    # the cache as numbers, without what lies between
    s["codes"], s["scales"] = cache[..., :8192].view(CODE[case["codes"]]), cache[..., 8192:].view(BF16)
    if kind in ("store", "load"):
        shape = (layers, n_kv, msl, HEAD_DIM)
        k, v = rnd.keys(*shape), rnd.normal(*shape)
        if kind == "load":
            for which, rows in enumerate((k, v)):
                _file(case, cache, case["first"], rows[:, :, case["first"]:case["first"] + case["count"]], which)
            k, v = torch.zeros_like(k), torch.zeros_like(v)
        if case["layout"] == "pos":
            k, v = (x.transpose(1, 2).contiguous() for x in (k, v))
        s["k"], s["v"] = k, v
        s["dims"].update(layer_num=layers, first_pos=case["first"], num_pos=case["count"], kv_layout={"pos": 0, "head": 1}[case["layout"]])
        return s
    n_q, ctx = case["n_q"], case["ctx"]
    n = case.get("rows", 1)
    if ctx:
        _file(case, cache, 0, rnd.keys(1, n_kv, ctx, HEAD_DIM), 0)
        _file(case, cache, 0, rnd.normal(1, n_kv, ctx, HEAD_DIM), 1)
    if kind != "rows":
        s["out"] = torch.zeros(n_q * HEAD_DIM, dtype=BF16, device=rnd.dev)
        s["ws"] = torch.empty(WORKSPACE_BYTES // 4, dtype=F32, device=rnd.dev)
        # "decode" attends to ctx + 1 positions, "step" to ctx and the one it files
        s["at"] = dict(pos=ctx, kv_mul=n_q // n_kv, head_num=n_q, layer_id=0)
        if case["device"]:
            s["at"].update(pos=msl - 1, pos_device=torch.tensor([ctx], dtype=torch.int32, device=rnd.dev))
    if kind == "decode":
        _file(case, cache, ctx, rnd.keys(1, n_kv, 1, HEAD_DIM), 0)
        _file(case, cache, ctx, rnd.normal(1, n_kv, 1, HEAD_DIM), 1)
        s["q"] = rnd.keys(n_q, HEAD_DIM)
        return s
    # the three projections of all tokens as one product leaves them, a token's query, key and value behind one another
    packed = rnd.normal(n, (n_q + 2 * n_kv) * HEAD_DIM)
    s["q_raw"], s["k_raw"], s["v_raw"] = packed.split([n_q * HEAD_DIM, n_kv * HEAD_DIM, n_kv * HEAD_DIM], dim=1)
    s["norm"] = rnd.normal(2 * HEAD_DIM, scale=0.02, mean=1.0)
    freq = torch.exp(torch.arange(HEAD_DIM // 2, device=rnd.dev, dtype=F64) * (-2.0 / HEAD_DIM * math.log(1e6)))
    angle = torch.arange(msl, device=rnd.dev, dtype=F64)[:, None] * freq
    s["sin"], s["cos"] = angle.sin().float(), angle.cos().float()
    if kind == "rows":
        s["q"] = torch.zeros(n, n_q * HEAD_DIM, dtype=BF16, device=rnd.dev)
    else:
        s["q_raw"], s["k_raw"], s["v_raw"] = s["q_raw"][0], s["k_raw"][0], s["v_raw"][0]
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"decode": _decode, "step": _step, "rows": _rows, "store": _store, "load": _load}[s["kind"]](s)


def _run_own(s):
    from llminfer_amd import ops
    kind = s["kind"]
    if kind == "decode":
        return ops.mha_decode_kv8(s["q"], s["cache"], s["out"], s["ws"], **s["at"], **s["dims"])
    if kind == "step":
        ops.mha_decode_append_kv8(s["q_raw"], s["k_raw"], s["v_raw"], s["norm"], s["sin"], s["cos"], s["cache"], s["out"], s["ws"], **s["at"], **s["dims"])
        return {"out": s["out"], "codes": s["codes"], "scales": s["scales"]}
    if kind == "rows":
        ops.qk_norm_rope_append_kv8(s["q"], s["k_raw"], s["v_raw"], s["cache"], s["norm"], s["sin"], s["cos"], query_src=s["q_raw"], layer_id=0,
                                    pos=s["case"]["ctx"], row_num=s["case"]["rows"], head_num=s["case"]["n_q"], **s["dims"])
        return {"query": s["q"], "codes": s["codes"], "scales": s["scales"]}
    if kind == "store":
        ops.kv8_store(s["k"], s["v"], s["cache"], **s["dims"])
        return {"codes": s["codes"], "scales": s["scales"]}
    ops.kv8_load(s["cache"], s["k"], s["v"], **s["dims"])
    return {"keys": s["k"], "values": s["v"]}


def _attended(s, q):
    """Attention of one token's query heads [heads][128] over the cache."""
    case = s["case"]
    n_q, n_kv, used = case["n_q"], case["n_kv"], case["ctx"] + 1
    k, v = (_fetch(case, s["cache"], 0, used, which)[0] for which in (0, 1))
    score = torch.matmul(q.view(n_kv, n_q // n_kv, HEAD_DIM).float(), k.transpose(1, 2).contiguous()).mul_(HEAD_DIM ** -0.5)
    weight = score.sub_(score.amax(-1, keepdim=True)).exp_()
    return (torch.matmul(weight, v) / weight.sum(-1, keepdim=True)).view(-1).to(BF16)


def _decode(s):
    return s["out"].copy_(_attended(s, s["q"]))


def _rotated(x, weight, sin, cos):
    """RMS norm over a head's 128 values, then the rotation of the pairs (i, i + 64)."""
    f = x.float()
    f = f * weight.float() * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    a, b = f[..., :HEAD_DIM // 2], f[..., HEAD_DIM // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(BF16)


def _filed(s, n):
    """n tokens' K and V rows into the cache; their queries, normalised and rotated."""
    case, pos = s["case"], s["case"]["ctx"]
    sin, cos = s["sin"][pos:pos + n, None], s["cos"][pos:pos + n, None]
    _file(case, s["cache"], pos, _rotated(s["k_raw"].reshape(n, -1, HEAD_DIM), s["norm"][HEAD_DIM:], sin, cos).transpose(0, 1)[None], 0)
    _file(case, s["cache"], pos, s["v_raw"].reshape(n, -1, HEAD_DIM).transpose(0, 1)[None], 1)
    return _rotated(s["q_raw"].reshape(n, -1, HEAD_DIM), s["norm"][:HEAD_DIM], sin, cos)


def _step(s):
    q = _filed(s, 1)
    s["out"].copy_(_attended(s, q[0]))
    return {"out": s["out"], "codes": s["codes"], "scales": s["scales"]}


def _rows(s):
    s["q"].copy_(_filed(s, s["case"]["rows"]).view(s["case"]["rows"], -1))
    return {"query": s["q"], "codes": s["codes"], "scales": s["scales"]}


def _by_head(s, x):
    """[layer][KV head][position][128] of the case's range, as a view."""
    case = s["case"]
    x = x.transpose(1, 2) if case["layout"] == "pos" else x
    return x[:, :, case["first"]:case["first"] + case["count"]]


def _store(s):
    for which, rows in enumerate((s["k"], s["v"])):
        _file(s["case"], s["cache"], s["case"]["first"], _by_head(s, rows), which)
    return {"codes": s["codes"], "scales": s["scales"]}


def _load(s):
    for which, rows in enumerate((s["k"], s["v"])):
        _by_head(s, rows).copy_(_fetch(s["case"], s["cache"], s["case"]["first"], s["case"]["count"], which))
    return {"keys": s["k"], "values": s["v"]}


def work(case):
    kind, row = case["kind"], case["n_kv"] * 2 * (HEAD_DIM + 2)  # bytes of a position's codes and scales
    if kind in ("store", "load"):
        return {"bytes": case["layers"] * case["count"] * (row + case["n_kv"] * 2 * HEAD_DIM * 2), "flops": 0}
    n = case.get("rows", 1)
    heads = 2 * n * case["n_q"] * HEAD_DIM * 2  # queries in, queries or outputs out
    new = n * (2 * case["n_kv"] * HEAD_DIM * 2 + row + HEAD_DIM * 4) + 4 * HEAD_DIM  # raw rows, filed rows, sines and cosines; norm weights
    turn = 10 * n * (case["n_q"] + case["n_kv"]) * HEAD_DIM
    if kind == "rows":
        return {"bytes": heads + new, "flops": turn}
    used = case["ctx"] + 1
    flops = 4 * case["n_q"] * HEAD_DIM * used
    if kind == "decode":
        return {"bytes": used * row + heads, "flops": flops}
    return {"bytes": case["ctx"] * row + heads + new, "flops": flops + turn}


def exact(case, seed):
    """What run() returns for these inputs, from the definitions, in 64 bits."""
    s = prepare(case, seed)
    kind, n_kv, msl = case["kind"], case["n_kv"], case["max_seq_len"]
    whole = s["cache"].shape[2] * PLACES
    if kind in ("store", "load"):
        first, end = case["first"], case["first"] + case["count"]
        if kind == "load":
            found = {}
            for name, which, cache in (("keys", 0, s["k"]), ("values", 1, s["v"])):
                by_head = torch.zeros(cache.shape[0], n_kv, msl, HEAD_DIM, dtype=F64, device=cache.device)
                q, scale = _read(case, s["cache"], which)
                by_head[:, :, first:end] = q[:, :, first:end] * scale[:, :, first:end, None]
                found[name] = by_head.transpose(1, 2) if case["layout"] == "pos" else by_head
            return found
        for which, cache in ((0, s["k"]), (1, s["v"])):
            rows = (cache.transpose(1, 2) if case["layout"] == "pos" else cache)[:, :, first:end]
            q, scale = _read(case, s["cache"], which)
            q[:, :, first:end], scale[:, :, first:end] = _nearest(rows, case["codes"])
            _write(case, s["cache"], which, q, scale)
        return {"codes": s["codes"], "scales": s["scales"].double()}
    ctx, n, n_q = case["ctx"], case.get("rows", 1), case["n_q"]
    if kind == "decode":
        query = s["q"].double()
    else:
        angle = torch.complex(s["cos"][ctx:ctx + n].double(), s["sin"][ctx:ctx + n].double())[:, None]

        def turn(rows, weight):
            x = rows.reshape(n, -1, HEAD_DIM).double()
            y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / HEAD_DIM + EPS) * weight.double()
            z = torch.complex(y[..., :HEAD_DIM // 2], y[..., HEAD_DIM // 2:]) * angle
            return torch.cat([z.real, z.imag], -1)

        new = turn(s["k_raw"], s["norm"][HEAD_DIM:]).to(BF16), s["v_raw"].reshape(n, -1, HEAD_DIM)
        for which in (0, 1):
            q, scale = _read(case, s["cache"], which)
            q[0, :, ctx:ctx + n], scale[0, :, ctx:ctx + n] = _nearest(new[which].transpose(0, 1), case["codes"])
            _write(case, s["cache"], which, q, scale)
        query = turn(s["q_raw"], s["norm"][:HEAD_DIM])
        if kind == "rows":
            return {"query": query.reshape(n, -1), "codes": s["codes"], "scales": s["scales"].double()}
        query = query[0].to(BF16).double()  # (what the rows' call hands to the attention's, and this one call to itself)
    out = torch.zeros(n_q, HEAD_DIM, dtype=F64, device=s["cache"].device)
    (k, k_scale), (v, v_scale) = _read(case, s["cache"], 0), _read(case, s["cache"], 1)
    for head in range(n_kv):
        rows = slice(head * (n_q // n_kv), (head + 1) * (n_q // n_kv))
        keys, values = (x[0, head, :ctx + 1] * y[0, head, :ctx + 1, None] for x, y in ((k, k_scale), (v, v_scale)))
        logit = (query[rows] @ keys.t().contiguous()) / math.sqrt(HEAD_DIM)
        out[rows] = torch.exp(logit - torch.logsumexp(logit, -1, keepdim=True)) @ values
    if kind == "decode":
        return out.view(-1)
    return {"out": out.view(-1), "codes": s["codes"], "scales": s["scales"].double()}


def _nearest(rows, codes):
    """Codes and scales of rows in 64 bits, from the definition."""
    x = rows.double()
    mantissa, exponent = torch.frexp(torch.div(x.abs().amax(-1), torch.tensor([TOP[codes]], dtype=F64, device=x.device)))
    scale = torch.ldexp(torch.ceil(mantissa * 256.0) / 256.0, exponent).clamp_min(LEAST)
    y = x / scale[..., None]
    if codes == "int8":
        return torch.round(y), scale
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp_min(-5) - 4)  # three bits behind the first; even spacing below 2^-6
    return torch.round(y / step) * step, scale


def _read(case, cache, which):
    """Codes [layer][KV head][position][128] and scales [layer][KV head][position] of a whole cache in 64 bits, by reshaping."""
    layers, n_kv, records = cache.shape[:3]
    q = cache[..., 4096 * which:4096 * (which + 1)].contiguous().view(CODE[case["codes"]]).double()
    if which == 0:
        q = q.view(layers, n_kv, records, 2, 8, 16, 16).transpose(4, 5)
    else:
        q = q.view(layers, n_kv, records, 4, 4, 16, 2, 2, 4).permute(0, 1, 2, 7, 4, 8, 3, 6, 5)  # t, g, i, channel / 32, / 16 % 2, % 16
    scale = cache.view(BF16)[..., 4096 + 32 * which:4128 + 32 * which].double().view(layers, n_kv, records, 4, 2, 4).transpose(3, 4)
    return q.reshape(layers, n_kv, -1, HEAD_DIM), scale.reshape(layers, n_kv, -1)


def _write(case, cache, which, q, scale):
    layers, n_kv, records = cache.shape[:3]
    q = q.to(CODE[case["codes"]]).view(torch.uint8)
    if which == 0:
        q = q.view(layers, n_kv, records, 2, 16, 8, 16).transpose(4, 5)
    else:
        q = q.view(layers, n_kv, records, 2, 4, 4, 4, 2, 16).permute(0, 1, 2, 6, 4, 8, 7, 3, 5)
    cache[..., 4096 * which:4096 * (which + 1)] = q.reshape(layers, n_kv, records, 4096)
    scale = scale.to(BF16).view(layers, n_kv, records, 2, 4, 4).transpose(3, 4)
    cache.view(BF16)[..., 4096 + 32 * which:4128 + 32 * which] = scale.reshape(layers, n_kv, records, 32)
