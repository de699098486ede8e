"""What the calls for an 8-bit KV cache write has to be apart from what they read and from what else they write: refused without a GPU."""
import ctypes

import pytest

from llminfer_amd import _binding as B
from llminfer_amd import ops

REFUSED = B.STATUS["INVALID_ARG"]
N_Q, N_KV, MSL, LAYER, POS, SPLITS = 32, 8, 5000, 2, 4000, 7
CACHE = ops.kv8_bytes(LAYER + 1, MSL, N_KV * 128, 128)
# Where everything lies, and how long it is: gigabytes apart.
MHA = {n: ((i + 1) << 32, size) for i, (n, size) in enumerate((
    ("query", N_Q * 256), ("output", N_Q * 256), ("output_f32", N_Q * 512), ("workspace", N_Q * 528 * SPLITS), ("cache8", CACHE), ("pos_device", 4), ("key_new", N_KV * 256),
    ("value_new", N_KV * 256), ("norm_weight", 512), ("sin_cache", (POS + 1) * 256), ("cos_cache", (POS + 1) * 256)))}
NEW = ("key_new", "value_new", "norm_weight", "sin_cache", "cos_cache")


def mha(at, append):
    a = B.MhaKv8Args(workspace_bytes=MHA["workspace"][1] + 16, layer_id=LAYER, pos=POS, kv_dim=N_KV * 128, kv_mul=N_Q // N_KV, head_num=N_Q, head_dim=128, max_seq_len=MSL, num_splits=SPLITS)
    for name, where in at.items():
        if name not in NEW:
            setattr(a, name, where)
    return B.MhaKv8AppendArgs(mha=a, eps=1e-6, **{n: at[n] for n in NEW}) if append else a


def over(places, write, other):
    """Places of `write` that share a byte, or some, with `other`: its end, its beginning, all of it."""
    (start, size), mine = places[other], places[write][1]
    unit = 4 if write == "output_f32" else 16
    first = start + (size - 1) // unit * unit
    return {first, start, start - mine + 16, start - mine // 2 // 16 * 16}


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("write", ["output", "output_f32", "workspace", "cache8"])
def test_attention(write, append):
    call = B.lib().llmi_hip_mha_decode_append_kv8 if append else B.lib().llmi_hip_mha_decode_kv8
    if write == "cache8" and not append:
        return  # (read only)
    for other in MHA:
        if other == write or (other in NEW and not append):
            continue
        for place in over(MHA, write, other):
            at = {n: x[0] for n, x in MHA.items()}
            at[write] = place
            assert call(ctypes.byref(mha(at, append))) == REFUSED, (write, other, hex(place))


def test_a_cache_past_any_address():
    """Sizes that no memory has: the end of the address space is the cache's."""
    for layer, msl in ((1 << 30, (1 << 31) - 1), ((1 << 31) - 1, MSL)):
        at = {n: x[0] for n, x in MHA.items()}
        at["output"], at["output_f32"], at["cache8"] = 1 << 62, 0, 1 << 40
        a = mha(at, False)
        a.layer_id, a.max_seq_len = layer, msl
        assert B.lib().llmi_hip_mha_decode_kv8(ctypes.byref(a)) == REFUSED
