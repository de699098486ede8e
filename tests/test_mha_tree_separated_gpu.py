"""llmi_hip_mha_decode_tree where scores lie so far apart that a split's weight is 0 in fp32: a V row that a node sees with an infinity or NaN makes
its column one that is not finite all the same, however the keys are split, and no other column."""
import math

import pytest
import torch

from llminfer_amd import _binding as B

from test_mha_tree_gpu import FORMS, Case
from tree_cases import by_head

pytestmark = pytest.mark.gpu

HEAD = B.KV_LAYOUT_HEAD_MAJOR


def separated(dev, n, n_q, n_kv, ctx, top):
    """Queries with a first value of 1; the cached key at `top` has one that puts its score 1600 / sqrt(128) = 141 (204 in log2) above the others'."""
    c = Case(dev, n, n_q, n_kv, ctx, seed=n)
    c.q[:, :, 0] = 1.0
    k = by_head(c.kc[0], c.layout)
    k[:, :ctx + n, 0] = 0.0
    k[:, top, 0] = 1600.0
    return c


def check(c, at, poison, what, **over):
    v = by_head(c.vc[0], c.layout)
    clean = c.run(**over)
    kept = v[:, at, 77].clone()
    v[:, at, 77] = poison
    got = c.run(**over)
    v[:, at, 77] = kept
    assert torch.isfinite(clean).all(), what
    assert not bool(torch.isfinite(got[:, :, 77]).any()), what
    assert torch.equal(got[:, :, :77], clean[:, :, :77]) and torch.equal(got[:, :, 78:], clean[:, :, 78:]), what


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 40])
def test_split_counts(dev, splits, poison):
    for n, n_q, n_kv in ((5, 32, 8), (40, 32, 8), (16, 32, 8), (7, 8, 1)):
        c = separated(dev, n, n_q, n_kv, 3000, 10)
        ws = torch.full((32 << 20,), math.nan, device=dev)
        for at in (11, 1500, 2990):
            check(c, at, poison, "n %d at %d" % (n, at), num_splits=splits, ws=ws)


@pytest.mark.parametrize("n,n_q,n_kv,ctx,rows_of_group", FORMS)
def test_every_form(dev, n, n_q, n_kv, ctx, rows_of_group):
    for top in (3, ctx - 40 if ctx > 60 else 20):
        c = separated(dev, n, n_q, n_kv, ctx, top)
        for at in (0, ctx // 2, ctx - 1):
            if at != top:
                check(c, at, math.nan, "top %d at %d" % (top, at))


def test_the_heaviest_row_alone_decides_the_rest(dev):
    """The outputs are that row's V: every other weight is 2^-170 of it. (Off by its weight's rounding to bf16, 2^-8, and a division.)"""
    for n, n_q, n_kv, ctx, _ in FORMS:
        c = separated(dev, n, n_q, n_kv, ctx, 7)
        got = c.run()
        want = by_head(c.vc[0], c.layout)[:, 7].float().repeat_interleave(n_q // n_kv, 0)
        assert bool(((got - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs()).all()), (n, n_q, ctx)
