"""Caches without a place: every query gets 0."""

import pytest
import torch

from _util import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,n,HQ,HK,window", [(1, 1, 2, 1, None), (4096, 1, 8, 4, None), (3, 40, 12, 2, 16)])
def test_empty_cache(B, n, HQ, HK, window, D):
    from solution.body.attention import cache_attention

    q = torch.full((B, n, HQ, D), float("nan"), device=DEV, dtype=torch.float16)
    k = torch.empty(B, 0, HK, D, device=DEV, dtype=torch.float16)
    lengths = torch.full((B,), 5, device=DEV, dtype=torch.int32)
    o = cache_attention(q, k, k, lengths, window=window)
    assert o.shape == q.shape and not o.any()
