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


def test_pages_past_32_bit_offsets():
    """Layers of more than 2^32 bytes, pages at both ends of each: every offset's part needs 64 bits."""
    from solution.body.paged import beam_reorder

    L, N, P, HK, D = 2, 4100, 1024, 4, 128  # 4.3 GB a layer
    tables = [[5, N - 1], [5, 0], [5, 2050], [5, N - 2]]
    parents, lengths, start = [[1, 0, 0, 2]], [P + 60], [P - 9]  # the first page is shared
    kp, vp = (torch.zeros(L, N, P, HK, D, dtype=torch.float16, device="cuda") for _ in range(2))
    for i, t in enumerate((kp, vp)):
        for page in (0, 5, 2050, N - 2, N - 1):
            t[:, page] = _pages((L, P, HK, D), torch.float16, 10 * i + page)
    want = [_reorder_ref(parents, t, tables, lengths, start) for t in (kp, vp)]
    assert not torch.equal(want[0], kp)
    beam_reorder(_i(parents), kp, vp, _i(tables), _i(lengths), _i(start))
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
