"""The tree attention's plan at the largest positions a caller can give as a bound (what is read follows the position on the device). No GPU."""
import pytest

from llminfer_amd import _binding as B

from test_tree_api import plan, tree_args

TOP = (1 << 31) - 1


@pytest.mark.parametrize("n,n_q,n_kv", [(1, 8, 1), (5, 16, 8), (16, 32, 8), (33, 32, 8), (64, 64, 8)])
@pytest.mark.parametrize("below", [0, 1, 30, 31, 32, 63])
def test_bounds_near_the_largest_position(n, n_q, n_kv, below):
    for forced in (0, 1, 7, 256):
        near, far = (plan(tree_args(node_num=n, head_num=n_q, kv_dim=128 * n_kv, kv_mul=n_q // n_kv, pos=pos, max_seq_len=TOP, num_splits=forced,
                                    workspace_bytes=1 << 40)) for pos in (TOP - n - below, 1 << 30))
        assert near[0] == far[0] == 0
        for field in ("path", "num_splits", "group_pad", "workspace_needed"):  # (long is long)
            assert getattr(near[1], field) == getattr(far[1], field)
        assert near[1].rows_per_split * near[1].num_splits >= TOP - below
        assert near[1].num_splits == forced or not forced
