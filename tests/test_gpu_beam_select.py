"""Beam search's selection (esep_beam_select, head.beam_select) against float64.

A value is score + logit - lse. The kernel's only roundings before 64 bits are lse's: an exponential of (x - max) is off by
|x - max| 3 / 2^24 for its argument (difference, product, the constant) and 2^-22 of its own, a sum of up to 32 terms
a lane, 8 steps of a tree and up to 75 pieces in fp32 / fp64 by 2^-24 for each of 32 + 8; with |x - max| <= 30 for all
that counts, lse is off by at most (3 * 30 + 4 + 40) 2^-24 = 8e-6 < LSE. The result is rounded to fp32 once more.
Candidates of one beam share lse, so their order is exact; two beams' may come in either order where their values
lie within 2 LSE of each other."""

import numpy as np
import pytest
import torch

from _util import DEV, gen

pytestmark = pytest.mark.gpu

LSE = 1e-5
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _values(logits, scores):
    """float64 [R, W, V], -inf where a beam is out."""
    x = logits.double().cpu()
    top = x.amax(-1, keepdim=True)
    lse = torch.log(torch.exp(x - top).sum(-1, keepdim=True)) + top
    s = scores.double().cpu()[..., None]
    return torch.where(torch.isfinite(lse) & torch.isfinite(s), s + (x - lse), -torch.inf).nan_to_num(
        nan=-torch.inf, neginf=-torch.inf)


def _check(got, logits, scores, keep):
    R, W, V = logits.shape
    out, parents, tokens = (t.cpu() for t in got)
    assert out.dtype == torch.float32 and parents.dtype == tokens.dtype == torch.int32
    assert out.shape == parents.shape == tokens.shape == (R, keep)
    values = _values(logits, scores).view(R, W * V).numpy()
    place = (parents.long() * V + tokens.long()).numpy()
    for r in range(R):
        v = values[r]
        want = np.lexsort((np.arange(W * V), -v))[:keep] if W * V <= 4096 else None
        if want is None:  # the same without sorting all of it
            border = np.partition(v, W * V - keep)[W * V - keep]
            above = np.nonzero(v > border)[0]
            want = np.concatenate([above, np.nonzero(v == border)[0][:keep - len(above)]])
            want = want[np.lexsort((want, -v[want]))]
        assert len(set(place[r])) == keep
        got_v = v[place[r]]
        fin = np.isfinite(v[want])
        assert (np.abs(out[r].numpy()[fin] - got_v[fin]) <= LSE + 2.0 ** -24 * np.abs(got_v[fin])).all()
        assert (out[r].numpy()[~fin] == -np.inf).all()
        assert (place[r][~fin] == want[~fin]).all(), (r, place[r], want)
        swap = np.nonzero(place[r] != want)[0]
        for j in swap:
            assert abs(got_v[j] - v[want[j]]) <= 2 * LSE, (r, j, place[r], want, got_v, v[want])
        for w in range(W):  # within a beam in order, ties by token
            mine = [p for p in place[r][fin] if p // V == w]
            x = v[mine]
            assert all(a > b or (a == b and p < q) for a, b, p, q in zip(x, x[1:], mine, mine[1:])), (r, w)


def _go(logits, scores, keep=None):
    from solution.head import beam_select

    return beam_select(logits, scores, keep)


def _inputs(R, W, V, dtype, seed, scale=2.5):
    g = gen(seed)
    logits = (torch.randn(R, W, V, generator=g) * scale).to(dtype).to(DEV)
    return logits, -(5 * torch.randn(R, W, generator=g)).abs().to(DEV)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,W,V,keep", [(1, 1, 1, 1), (1, 2, 5, 10), (2, 64, 100, 64), (1, 4, 151936, 8),
                                        (3, 5, 50001, 10), (70, 3, 1000, 6), (24, 5, 50000, 5), (2, 3, 2049, 64),
                                        (30, 8, 32000, 16), (1, 1, 70000, 1), (1, 1, 151936, 64),
                                        (300, 3, 1000, 8), (260, 2, 4099, 20)])
def test_select(R, W, V, keep, dtype):
    logits, scores = _inputs(R, W, V, dtype, R * 7 + V % 13)
    got = _go(logits, scores, keep)
    _check(got, logits, scores, keep)
    for a, b in zip(got, _go(logits, scores, keep)):
        assert torch.equal(a, b)  # the same bits twice
    # only the first beam alive, as at the first step
    scores[:] = -torch.inf
    scores[:, 0] = 0
    _check(_go(logits, scores, keep), logits, scores, keep)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [1000, 5003, 40000])
def test_ties_go_to_the_lowest_place(V, dtype):
    """Rows of one value, of 0 and -0, of a few values many times each (lists of candidates that overflow)."""
    g = gen(V)
    flat = torch.full((2, 3, V), 1.5).to(dtype).to(DEV)
    zero = torch.zeros(2, 3, V)
    zero[..., ::2] = -0.0
    few = torch.randint(0, 3, (2, 3, V), generator=g)
    same = torch.zeros(2, 3, device=DEV)
    for logits in (flat, zero.to(dtype).to(DEV), few.to(dtype).to(DEV)):
        for keep in (1, 7, 64):
            out, parents, tokens = _go(logits, same, keep)
            values = _values(logits, same)
            if logits is not flat and (logits != 0).any():
                _check((out, parents, tokens), logits, same, keep)
                continue
            assert not parents.any() and (tokens.cpu() == torch.arange(min(keep, V))).all()
            assert (out.cpu().double() - values[:, 0, :1]).abs().max() <= LSE + 2.0 ** -20
    # equal beams: the first one's candidate before the second's of the same token
    logits, _ = _inputs(1, 1, V, dtype, 3)
    twice = logits.expand(1, 2, V)
    out, parents, tokens = _go(twice, torch.full((1, 2), -3.0, device=DEV), 8)
    assert torch.equal(parents[0, ::2], torch.zeros_like(parents[0, ::2])) or (out[0, :-1] == out[0, 1:]).any()
    _check((out, parents, tokens), twice, torch.full((1, 2), -3.0, device=DEV), 8)
    x = logits[0, 0].double()
    want = torch.sort(x, descending=True, stable=True).values[:4]
    assert torch.equal(out[0, ::2], out[0, 1::2]) or want.unique().numel() < 4


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [37, 3000, 20000])
def test_beams_that_are_out(V, dtype):
    """-inf, infinite and NaN scores; rows with a NaN, +inf, nothing finite; masked tokens; fewer than `keep` left."""
    logits, scores = _inputs(9, 4, V, dtype, V)
    nan, inf = float("nan"), float("inf")
    scores[0, 1], scores[0, 2], scores[0, 3] = -inf, nan, inf
    logits[1, 0, V // 2] = nan
    logits[2, 1, V - 1] = inf
    logits[3, 2] = -inf
    logits[4] = -inf                      # nothing at all
    logits[5, :, 3:] = -inf               # three tokens a beam
    logits[6] = -inf
    logits[6, 2, V - 2] = 4.0             # one candidate
    logits[7, :, :V // 2] = -inf
    scores[8] = -inf
    for keep in (1, 4, 30):
        _check(_go(logits, scores, keep), logits, scores, keep)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("W,V,keep", [(16, 151936, 32), (8, 100003, 64), (1, 2048, 64)])
def test_rows_in_order(W, V, keep, dtype):
    """Rows that rise or fall all along (a piece's greatest lie with a few of its threads), beside ones in no order."""
    logits, scores = _inputs(3, W, V, dtype, V + keep)
    logits[1] = logits[1].float().sort(-1).values.to(dtype)
    logits[2] = logits[2].float().sort(-1, descending=True).values.to(dtype)
    _check(_go(logits, scores, keep), logits, scores, keep)


def test_extremes():
    """The largest values of each type, differences that the exponentials flush, far apart scores."""
    for dtype in DTYPES:
        big = torch.finfo(dtype).max
        logits = torch.tensor([[[big, 0, -big, big], [1, 2, 3, -big]]]).to(dtype).to(DEV)
        scores = torch.tensor([[-1.0, -1e30]], device=DEV)
        out, parents, tokens = _go(logits, scores, 2)
        assert parents.tolist() == [[0, 0]] and tokens.tolist() == [[0, 3]]
        assert torch.allclose(out, torch.full_like(out, -1.0 - 0.6931472), atol=1e-6)


def test_strides():
    """Rows of a padded vocabulary at any stride and address, a transposed request dimension, a step in the vocabulary."""
    big, scores = _inputs(3, 4, 1500, torch.float16, 1)
    for logits in (big[..., :1003], big[..., 3:1200], big[..., ::2], big.transpose(0, 1)[:, :3], big[:, :2],
                   big[:1].expand(3, 4, 1500)):
        R, W, V = logits.shape
        sc = scores.t() if R == 4 else scores[:, :W]
        got = _go(logits, sc, 6)
        want = _go(logits.contiguous(), sc.contiguous(), 6)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        _check(got, logits, sc, 6)


def test_default_keep_and_no_requests():
    logits, scores = _inputs(2, 3, 50, torch.float32, 2)
    out, parents, tokens = _go(logits, scores)
    assert out.shape == (2, 3)
    _check((out, parents, tokens), logits, scores, 3)
    assert [t.shape for t in _go(logits[:0], scores[:0], 5)] == [(0, 5)] * 3


def test_far_rows():
    """A row that begins past 2^32 bytes."""
    V = (1 << 24) - 5
    logits = torch.zeros(130, 1, V, dtype=torch.bfloat16, device=DEV)
    logits[129, 0, V - 3] = 5.0
    logits[129, 0, 7] = 4.0
    out, parents, tokens = _go(logits[128:], torch.zeros(2, 1, device=DEV), 2)
    assert tokens.tolist() == [[0, 1], [V - 3, 7]]
    got = _go(logits, torch.zeros(130, 1, device=DEV), 2)
    assert torch.equal(got[2][128:], tokens) and torch.equal(got[0][128:], out)


def test_graph_and_streams():
    a, sa = _inputs(2, 4, 40000, torch.bfloat16, 5)
    b, sb = _inputs(30, 5, 9001, torch.float32, 6)
    want = _go(a, sa, 8), _go(b, sb, 5)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for st, args in zip(streams, ((a, sa, 8), (b, sb, 5))):
            with torch.cuda.stream(st):
                got.append(_go(*args))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for x, y in zip(outs, want[i % 2]):
            assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _go(a, sa, 8)
    for i in range(4):
        a.copy_(torch.randn(a.shape, generator=gen(i)))
        sa.copy_(-torch.rand(sa.shape, generator=gen(i)))
        graph.replay()
        want = _go(a, sa, 8)
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y)
