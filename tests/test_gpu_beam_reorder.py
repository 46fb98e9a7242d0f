"""beam_reorder where the pieces of a token's heads leave some lanes of a wavefront without work, against a token at a time on
the host, bit for bit."""

import random

import pytest
import torch

from test_gpu_paged_upkeep import _i, _pages, _parents, _reorder_ref

pytestmark = pytest.mark.gpu


# Busy lanes of a block's four wavefronts: 136 pieces 64, 64, 8, 0; 88 (two tokens at once) 64, 64, 48, 0; 72 (three) 64, 64,
# 64, 24; 3 (85) 64, 64, 64, 63; 264 and 1 all.
@pytest.mark.parametrize("how", ["swap", "one", "any"])
@pytest.mark.parametrize("HK,D", [(17, 64), (11, 64), (9, 64), (33, 64), (3, 8), (1, 8)])
@pytest.mark.parametrize("W", [3, 8, 16, 32])
def test_lanes_without_a_piece(W, HK, D, how):
    from solution.body.paged import beam_reorder

    rng, R, L, P, top = random.Random(W + HK), 2, 2, 16, 37
    M = -(-top // P)
    ids = list(range(R * W * M))
    rng.shuffle(ids)
    tables = [[ids.pop() for _ in range(M)] for _ in range(R * W)]
    parents, lengths, start = _parents(rng, R, W, how), [top, top - 5], [3, 0]
    kp, vp = (_pages((L, R * W * M, P, HK, D), torch.float16, s) for s in (1, 2))
    want = [_reorder_ref(parents, t, tables, lengths, start) for t in (kp, vp)]
    beam_reorder(_i(parents), kp, vp, _i(tables), _i(lengths), _i(start))
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
