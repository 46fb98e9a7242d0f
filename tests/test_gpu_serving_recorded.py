"""cache_attention traced on the GPU: the traced module runs the kernel on its inputs, lengths among them."""

import pytest
import torch

from _util import DEV, gen

pytestmark = pytest.mark.gpu


def test_traced_cache_attention():
    from solution.body.attention import cache_attention

    def inputs(seed, lengths):
        g = gen(seed)
        q = torch.randn(2, 1, 6, 64, generator=g).half().to(DEV)
        k, v = (torch.randn(2, 300, 2, 64, generator=g).half().to(DEV) for _ in range(2))
        return q, k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV)

    def step(q, k, v, lengths):
        return cache_attention(q, k, v, lengths, scale=0.125, window=100, sinks=4)

    first, second = inputs(1, [300, 17]), inputs(2, [5, 290])
    want = step(*first), step(*second)
    traced = torch.jit.trace(step, first, check_trace=False)
    for x, w in ((first, want[0]), (second, want[1])):
        assert torch.equal(traced(*x), w)
