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


# The rows' call: three tokens whose projections lie in one buffer, a token's query, key and value behind one another.
N, PACKED = 3, (N_Q + 2 * N_KV) * 256
ROWS = {n: ((i + 20) << 32, size) for i, (n, size) in enumerate((
    ("query", N * N_Q * 256), ("query_src", 2 * PACKED + N_Q * 256), ("cache8", CACHE), ("pos_device", 4), ("norm_weight", 512), ("sin_cache", (POS + N) * 256), ("cos_cache", (POS + N) * 256)))}
ROWS["key_new"] = (ROWS["query_src"][0] + N_Q * 256, 2 * PACKED + N_KV * 256)
ROWS["value_new"] = (ROWS["key_new"][0] + N_KV * 256, 2 * PACKED + N_KV * 256)


def append_rows(at, **more):
    a = B.QkNormRopeKv8Args(layer_id=LAYER, pos=POS, row_num=N, kv_dim=N_KV * 128, head_num=N_Q, head_dim=128, max_seq_len=MSL, eps=1e-6, query_src_stride=PACKED // 2,
                            key_new_stride=PACKED // 2, value_new_stride=PACKED // 2)
    for name, value in {**at, **more}.items():
        setattr(a, name, value)
    return B.lib().llmi_hip_qk_norm_rope_append_kv8(ctypes.byref(a))


def test_rows():
    """Dense query rows, and the cache, over each of the things that are read; over one another."""
    for write in ("query", "cache8"):
        for other in ROWS:
            if other == write:
                continue
            for place in over(ROWS, write, other):
                at = {n: x[0] for n, x in ROWS.items()}
                if other == "query_src" and place == at["query_src"]:
                    at["query_src"] += 16  # (in its place: below)
                at[write] = place
                assert append_rows(at) == REFUSED, (write, other, hex(place))


@pytest.mark.parametrize("shift", [16, 256, N_Q * 256 - 16, N_Q * 256, (N_Q + N_KV) * 256, PACKED - 16, PACKED - N_Q * 256 + 16, -16, -N_Q * 256 + 16, 16 - PACKED])
def test_rows_of_the_packed_buffer(shift):
    """Query rows with the packed rows' stride whose place in them is another one's: a neighbouring head's, the key's, the value's, past the row's end."""
    at = {n: x[0] for n, x in ROWS.items()}
    at["query"] = at["query_src"] + shift
    assert append_rows(at, query_stride=PACKED // 2) == REFUSED


def test_rows_in_place():
    """In the raw rows' place only with their stride; one row in another one's place not at all; a stride that has no end."""
    at = {n: x[0] for n, x in ROWS.items()}
    at["query"] = at["query_src"]
    assert append_rows(at) == REFUSED  # (dense over packed)
    assert append_rows(at, query_stride=PACKED) == REFUSED
    at["query"] = at["query_src"] + PACKED
    assert append_rows(at, query_stride=PACKED // 2) == REFUSED
    at["query"], at["query_src"] = at["query_src"], 0
    assert append_rows(at, query_stride=PACKED // 2 - 8) == REFUSED  # (runs into the keys)
    at = {n: x[0] for n, x in ROWS.items()}
    assert append_rows({**at, "query": at["cos_cache"] - (1 << 20)}, query_stride=(1 << 62)) == REFUSED


@pytest.mark.parametrize("call,also", [("llmi_hip_kv8_store", False), ("llmi_hip_kv8_load", True)])
def test_copies(call, also):
    """Caches of three layers over one another, by a little or altogether; nothing to copy is no overlap."""
    call, rows = getattr(B.lib(), call), 3 * MSL * N_KV * 256
    places = {"key_cache": (1 << 36, rows), "value_cache": (2 << 36, rows), "cache8": (3 << 36, ops.kv8_bytes(3, MSL, N_KV * 128, 128))}
    for one, other in (("key_cache", "cache8"), ("cache8", "key_cache"), ("value_cache", "cache8"), ("cache8", "value_cache")) + ((("key_cache", "value_cache"), ("value_cache", "key_cache")) if also else ()):
        for place in over(places, one, other):
            a = B.Kv8CopyArgs(layer_num=3, first_pos=7, num_pos=10, kv_dim=N_KV * 128, head_dim=128, max_seq_len=MSL)
            for name, (where, _) in places.items():
                setattr(a, name, where)
            setattr(a, one, place)
            assert call(ctypes.byref(a)) == REFUSED, (one, other, hex(place))
            a.num_pos = 0
            assert call(ctypes.byref(a)) == 0
    a = B.Kv8CopyArgs(layer_num=(1 << 31) - 1, num_pos=1, kv_dim=1 << 20, head_dim=128, max_seq_len=1 << 15, key_cache=1 << 30, value_cache=1 << 62, cache8=1 << 20)
    assert call(ctypes.byref(a)) == REFUSED  # (sizes that no memory has)
