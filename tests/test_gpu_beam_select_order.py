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


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [50, 5003, 151936])
@pytest.mark.parametrize("W", [2, 5, 16])
def test_equal_beams_take_turns(W, V, dtype):
    """W times the same row, expanded and (at other alignments) stored, its greatest values apart from each other: each
    token for the beams in order."""
    from solution.head import beam_select

    g = gen(V + W)
    row = torch.randn(V, generator=g).to(dtype)
    best = torch.randperm(V, generator=g)[:20]
    row[best] = torch.arange(30, 10, -1).to(dtype)
    expanded = row.to(DEV).expand(1, W, V)
    scores = torch.full((1, W), -3.0, device=DEV)
    keep = min(4 * W, 64)
    for logits in (expanded, expanded.contiguous(), torch.cat([expanded[:, :1], expanded], 1)[:, 1:]):
        out, parents, tokens = beam_select(logits, scores, keep)
        assert parents.tolist() == [[i % W for i in range(keep)]]
        assert tokens.tolist() == [[best[i // W].item() for i in range(keep)]]
        for i in range(0, keep, W):
            assert len(set(out[0, i:i + W].tolist())) == 1
        _same(logits, scores, keep)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [40, 3001, 40000])
@pytest.mark.parametrize("few", [3, 40])
def test_ties_within_and_between_beams(few, V, dtype):
    """Values that come many times in a row, and rows that come several times in a request (their scores equal, or 100 apart,
    so that no two different rows' values meet)."""
    g = gen(V * few)
    rows = (torch.randint(0, few, (2, V), generator=g) * 0.25).to(dtype)
    logits = rows[torch.tensor([[0, 0, 1, 1, 0], [1, 1, 1, 1, 1], [0, 1, 0, 1, 1]])].to(DEV)
    scores = torch.tensor([[-1.0, -1.0, -101.0, -101.0, -1.0], [0.0] * 5, [-200.0, -1.0, -200.0, -1.0, -100.0]],
                          device=DEV)
    for keep in (1, 5, 33, 64):
        _same(logits, scores, keep)
