"""The 8-bit KV cache from its definition, in 64 bits on the host: codes, scales, layout, and the attention over them."""
import math

import torch

D, RECORD, PLACES = 128, 8320, 32
E4M3, INT8 = 0, 1
TOP = {E4M3: 448.0, INT8: 127.0}
BF16, F64 = torch.bfloat16, torch.float64


def quantise(rows, fmt):
    """Codes as bytes [..., 128] and scales as bf16 [...] of bf16 rows."""
    x = rows.double()
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine[..., None], x, torch.zeros_like(x))
    mantissa, exponent = torch.frexp(x.abs().amax(-1) / TOP[fmt])
    scale = torch.ldexp(torch.ceil(mantissa * 256.0) / 256.0, exponent).clamp_min(2.0 ** -64)
    y = x / scale[..., None]
    if fmt == INT8:
        codes = torch.round(y).to(torch.int8).view(torch.uint8)
    else:
        step = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp_min(-5) - 4)
        exact = torch.round(y / step) * step
        codes = exact.float().to(torch.float8_e4m3fn).view(torch.uint8)
        assert torch.equal(codes.view(torch.float8_e4m3fn).double(), exact)
    return codes, torch.where(fine, scale, torch.full_like(scale, math.nan)).to(BF16)


def stands_for(codes, scale, fmt):
    """code * scale in 64 bits."""
    return codes.view(torch.int8 if fmt == INT8 else torch.float8_e4m3fn).double() * scale.double()[..., None]


def records(msl):
    return (msl + PLACES - 1) // PLACES


def pack(kc, ks, vc, vs):
    """[layers][KV heads][positions (whole records)][128] codes and [...] scales -> [layers][KV heads][records][8320] bytes."""
    layers, heads, n, _ = kc.shape
    r = n // PLACES
    k = kc.view(layers, heads, r, 2, 16, 8, 16).transpose(4, 5).reshape(layers, heads, r, 4096)
    v = vc.view(layers, heads, r, 2, 4, 4, 4, 2, 16).permute(0, 1, 2, 6, 4, 8, 7, 3, 5).reshape(layers, heads, r, 4096)
    parts = [k, v]
    for s in (ks, vs):
        parts.append(s.view(layers, heads, r, 2, 4, 4).transpose(3, 4).reshape(layers, heads, r, 32).contiguous().view(torch.uint8))
    return torch.cat(parts, -1).contiguous()


def unpack(cache):
    """The inverse: K codes, K scales, V codes, V scales."""
    layers, heads, r, _ = cache.shape
    k = cache[..., :4096].reshape(layers, heads, r, 2, 8, 16, 16).transpose(4, 5).reshape(layers, heads, r * PLACES, D)
    v = cache[..., 4096:8192].reshape(layers, heads, r, 4, 4, 16, 2, 2, 4).permute(0, 1, 2, 7, 4, 8, 3, 6, 5).reshape(layers, heads, r * PLACES, D)
    ks, vs = (cache[..., a:a + 64].contiguous().view(BF16).view(layers, heads, r, 4, 2, 4).transpose(3, 4).reshape(layers, heads, r * PLACES)
              for a in (8192, 8256))
    return k, ks, v, vs


def garbage(layers, heads, msl, seed):
    """A cache of bytes that are NaN as E4M3 codes and as scales, here and there anything."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(0, 256, (layers, heads, records(msl), RECORD), generator=g, dtype=torch.uint8)
    return torch.where(torch.rand(x.shape, generator=g) < 0.5, torch.tensor(0x7F, dtype=torch.uint8), x | 0x80)


def rows(gen, *shape, outliers=True):
    """bf16 rows, some channels several times the others, magnitudes that differ from row to row."""
    x = torch.randn(*shape, D, generator=gen)
    if outliers:
        x = x * (1.0 + 7.0 * (torch.rand(D, generator=gen) < 0.04)) * torch.exp2(torch.randint(-3, 4, (*shape, 1), generator=gen).float())
    return x.to(BF16)


def filled(layers, heads, msl, used, fmt, seed):
    """A cache whose first `used` positions hold rows, the rest garbage; with the rows K, V as they stand there, in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    cache = garbage(layers, heads, msl, seed + 1)
    kc, ks, vc, vs = unpack(cache)
    values = []
    for c, s in ((kc, ks), (vc, vs)):
        q, t = quantise(rows(g, layers, heads, used), fmt)
        c[:, :, :used], s[:, :, :used] = q, t
        values.append(stands_for(q, t, fmt))
    return pack(kc, ks, vc, vs), values[0], values[1]


def attention(q, k, v):
    """Outputs of query heads [heads][128] (bf16) over K, V [KV heads][keys][128] in 64 bits, and how far a kernel's fp32 result may be off.

    The roundings: a score is the fp32 sum of 128 exact products (each addition 2^-24 of what is summed so far, at most the sum of the magnitudes),
    times two scales (2^-24 each for their product and the score's); it enters exp2, one unit (2^-23) off, through a subtraction (2^-24 of the
    two scores, which are at most A): the weight is off by 2^-23 + ln 2 * (130 + 4) * 2^-24 * 2 A / ln 2. A weight times V's scale rounds once (2^-24) and enters the sum over V
    as two bf16 numbers: 2^-9 of 2^-9 are lost at most, 2^-17 to be safe with the second's own rounding; sums over n keys lose n * 2^-24 at most, once for V
    and once for the weights; joining the parts (wavefronts, splits) another exp2 and product each, twice, and one division.
    What is under fp32's least normal number, 2^-126, counts as 0: a weight (the largest is 1 at least, so is their sum), which loses 2^-126 |v| of the output at
    most, and its product with V's scale or either of the two bf16 numbers, 2^-126 times a code of 448 at most each: keys * 2^-125 * (|v| + 448)."""
    n_q, n_kv = q.shape[0], k.shape[0]
    x = q.double().view(n_kv, n_q // n_kv, D)
    score = x @ k.transpose(1, 2) / math.sqrt(D)
    most = (x.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) / math.sqrt(D)
    w = torch.softmax(score, -1)
    out = w @ v
    off = 2.0 ** -23 + 2 * 134 * 2.0 ** -24 * most + 2.0 ** -16 + 2 * (k.shape[1] + 64) * 2.0 ** -24 + 8 * 2.0 ** -23
    least = k.shape[1] * 2.0 ** -125 * (v.abs().amax(1, keepdim=True) + 448.0)
    return out.reshape(n_q, D), (2 * off * (w @ v.abs()) + least).reshape(n_q, D)


def close(got, ref, off, rounded=None):
    """Asserts |got - ref| <= off; `rounded`: a bf16 output besides, another half a step of it (2^-8) off."""
    d = (got.double() - ref).abs()
    assert bool((d <= off).all()), "off by up to %.3g times the bound" % float((d / off.clamp_min(1e-300)).max())
    if rounded is not None:
        d = (rounded.double() - ref).abs()
        assert bool((d <= off + 2.0 ** -8 * (ref.abs() + off)).all())


def tables(msl):
    freq = torch.exp(torch.arange(64, dtype=F64) * (-2.0 / D * math.log(1e6)))
    angle = torch.arange(msl, dtype=F64)[:, None] * freq
    return angle.sin().float(), angle.cos().float()


def normed(x, w, sin, cos, eps=1e-6):
    """RMS norm and rotation of rows [tokens][heads][128] in 64 bits; sin, cos [tokens][64]."""
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    a, b, s, c = y[..., :64], y[..., 64:], sin.double()[:, None], cos.double()[:, None]
    return torch.cat([a * c - b * s, a * s + b * c], -1)
