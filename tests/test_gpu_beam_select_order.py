"""The order of beam selection, place by place, against a stable sort in float64: of equal values the lowest beam and then the
lowest token, of values that fp32 cannot hold the greatest."""

import numpy as np
import pytest
import torch

from _util import DEV, gen

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _places(logits, scores, keep):
    """(float64 values, parents, tokens) of each request, [R, keep]. Equal rows with equal scores have equal values."""
    R, W, V = logits.shape
    x = logits.double().cpu()
    top = x.amax(-1, keepdim=True)
    v = ((x - top) - torch.log(torch.exp(x - top).sum(-1, keepdim=True)) + scores.double().cpu()[..., None])
    v = v.reshape(R, W * V).numpy()
    at = np.stack([np.lexsort((np.arange(W * V), -row))[:keep] for row in v])
    return np.take_along_axis(v, at, 1), at // V, at % V


def _same(logits, scores, keep):
    from solution.head import beam_select

    out, parents, tokens = (t.cpu().numpy() for t in beam_select(logits, scores, keep))
    _, want_parents, want_tokens = _places(logits, scores, keep)
    assert (parents == want_parents).all(), (parents, want_parents)
    assert (tokens == want_tokens).all(), (tokens, want_tokens)
    return out


@pytest.mark.parametrize("lowest", [False, True], ids=["some", "most"])
def test_values_below_the_range_of_fp32(lowest):
    """score + logit - lse down to -1e39: above -inf, and in their order, where too few others are left."""
    top, inf = torch.finfo(torch.float32).max, float("inf")
    rows = torch.full((3, 2, 700), -inf)
    rows[..., 300] = top
    rows[0, :, 600], rows[0, :, 500] = -top, -0.5 * top   # -2 and -1.5 times fp32's greatest
    rows[1, 1, 2] = -top
    rows[2, 0, 5], rows[2, 1, 4] = -top, -0.75 * top
    if lowest:
        rows[0, :, 400:] = -top
    scores = torch.tensor([[0.0, -3.0], [-1.0, -3e38], [0.0, -2e38]], device=DEV)
    for keep in (2, 5, 9, 40):
        out = _same(rows.to(DEV), scores, keep)
        assert (out[:, 1:] < -1e38).any() and not np.isnan(out).any()
