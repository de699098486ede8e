"""Does the bound of tree_weights see a weight that is rounded once? The mistake planted in the formula, no GPU."""
import pytest
import torch

from tree_cases import attention64
from tree_weights import few_keys, rounded_attention, weight_bound


@pytest.mark.parametrize("n,n_q,n_kv,ctx,every", [(5, 16, 8, 50, 13), (4, 8, 2, 700, 140), (12, 8, 1, 2000, 399)])
def test_the_bound_tells_two_numbers_from_one(n, n_q, n_kv, ctx, every):
    q, k, v = few_keys(n, n, n_q, n_kv, ctx, torch.device("cpu"), every)
    k, v = (x.transpose(0, 1) for x in (k, v))
    words = [1 << i for i in range(n)]
    want, size = attention64(q, k, v, ctx, words)
    bound = weight_bound(size, -(-ctx // every) + 1)
    worst = [float(((rounded_attention(q, k, v, ctx, words, parts) - want).abs() / bound).max()) for parts in (1, 2, 3)]
    assert worst[0] > 2 and worst[1] < 0.1 and worst[2] < 0.01, worst
