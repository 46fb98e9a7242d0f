"""The rows of a batch under sliding-window layers, without a GPU: runs of tokens and gaps, and a batch without
columns."""

import pytest
import torch

from solution.body import packed


@pytest.mark.parametrize("rows,lens,gaps", [
    ([[1, 1, 1], [1, 1, 0]], [3, 2], False),
    ([[0, 1, 1], [0, 0, 1]], [2, 1], False),
    ([[1, 0, 1], [1, 1, 0]], [2, 2], True),
    ([[0, 1, 0], [0, 0, 0]], [1, 0], False),
    ([[], []], [0, 0], False),  # goes to the original forward, as under full attention
])
def test_runs(rows, lens, gaps):
    mask = torch.tensor(rows, dtype=torch.int64)
    pack = packed._Packing(mask, None, True)
    assert (pack.lens, pack.gaps) == (lens, gaps)
    assert packed._Packing(mask, None).lens == lens
