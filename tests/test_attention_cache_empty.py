"""The workspace of attention over caches without a place, without a GPU: the join reads two numbers of every group
whatever its length."""

import pytest

from solution.body import _hip


@pytest.mark.parametrize("B,n,HQ,HK,window", [(1, 1, 2, 1, None), (4096, 1, 8, 4, None), (3, 40, 12, 2, 16)])
def test_workspace_of_an_empty_cache(B, n, HQ, HK, window):
    groups = B * HK * -(-n * (HQ // HK) // 32)
    for D in (64, 128):
        assert _hip.attn_cache_workspace(B, n, 0, HQ, HK, D, window) >= 2 * groups
