"""Windowed attention with sinks on the GPU (esep_attn_win_fwd / _bwd, varlen_attention(window=, sinks=))
against float64.

The bounds are derived per element, with u half a step of the stored type (bf16 2^-8, fp16 2^-11) and the
sums taken over the keys (or queries) that the definition lets through:
  o   the probabilities enter P V rounded (u relative each), the result is rounded once:
      u (sum p |v| + |o|)
  dv  the same with dO: u (sum p |do| + |dv|)
  dq  dS is rounded (u), and delta = rowsum(dO o) sees the o above, so each dS is off by p sum |do| |o's error|:
      scale (u sum |ds| |k| + sum p |k| E) + u |dq|, E = u sum_d |do| (sum p |v| + |o|); with o_low, o's own
      rounding is not in it: E = u sum_d |do| (sum p |v|) + u^2 |do| |o|
  dk  the same over queries.
fp16 holds small probabilities and dS as subnormals, 2^-25 off at most: 2^-25 times the sum of |v| (|do|, |k|,
|q|). The 32-bit arithmetic (scores of up to about 30, their exponentials, sums) adds less than 4e-5 of the same
sums of magnitudes."""

import numpy as np
import pytest
import torch

from _util import DEV, gen

pytestmark = pytest.mark.gpu

# (lengths, query heads, kv heads, head dim, window, sinks)
CASES = [
    ([1], 2, 2, 64, 1, 0),
    ([0, 1, 0, 5, 2, 0], 2, 1, 128, 2, 1),
    ([31, 33, 64, 65, 127, 128, 129, 200], 12, 2, 128, 64, 4),
    ([513, 7], 4, 2, 64, 100, 16),
    ([300, 1, 257], 28, 4, 128, 1, 0),          # every query sees itself alone
    ([96, 160], 8, 8, 128, 33, 40),             # sinks that reach the window
    ([130, 260], 4, 4, 64, 129, 129),
    ([640, 576, 577], 2, 1, 128, 64, 3),        # at and around the length of far blocks
    ([1500, 30, 700], 4, 2, 128, 64, 5),        # sink keys seen from afar
    ([1400], 6, 2, 64, 130, 200),               # sinks in two key tiles
    ([700], 2, 1, 64, 100, 650),                # a tile of sinks that no far query sees
    ([1300], 2, 1, 128, 40, 1300),              # all sinks: causal
    ([2100], 3, 1, 64, 1, 1),
    ([95, 33, 0, 1, 250, 32], 10, 2, 128, 20, 2),  # items of several heads to a block
    ([70, 129, 31, 160], 16, 1, 64, 50, 0),
    ([257, 64, 31, 97], 9, 3, 128, 32, 5),
    ([40] * 70 + [0] * 3 + [33], 5, 1, 64, 17, 1),
    ([3001, 1400, 1607], 14, 2, 64, 300, 5),       # heads dealt unevenly to the dK / dV blocks
    ([1501, 900, 1607], 28, 4, 128, 300, 0),
]


def _reference(q, k, v, do, lengths, scale, window, sinks, u, sub, low=True):
    """(o, dq, dk, dv) in float64 and their bounds (low: the backward has o_low)."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    res = [torch.zeros_like(t) for t in (q, q, k, v)]
    tol = [torch.zeros_like(t) for t in (q, q, k, v)]
    G, t0, f = q.shape[1] // k.shape[1], 0, u + 4e-5
    for n in lengths:
        s = slice(t0, t0 + n)
        t0 += n
        if n == 0:
            continue
        i = torch.arange(n, device=q.device)
        seen = i[None, :] <= i[:, None]
        if window is not None:
            seen &= (i[:, None] - i[None, :] < window) | (i[None, :] < sinks)
        for h in range(q.shape[1]):
            kh = h // G
            Q, K, V, DO = q[s, h], k[s, kh], v[s, kh], do[s, h]
            sc = (scale * Q @ K.t()).masked_fill(~seen, -torch.inf)
            p = torch.softmax(sc, 1)
            w = seen.double()
            o = p @ V
            ds = p * (DO @ V.t() - (DO * o).sum(1, keepdim=True))
            res[0][s, h], res[1][s, h] = o, scale * ds @ K
            res[2][s, kh] += scale * ds.t() @ Q
            res[3][s, kh] += p.t() @ DO
            eo = f * (p @ V.abs() + o.abs()) + sub * (w @ V.abs())
            E = (DO.abs() * (eo - (u - u * u) * o.abs() if low else eo)).sum(1, keepdim=True)
            tol[0][s, h] = eo
            tol[1][s, h] = (scale * (f * ds.abs() + p * E + sub * w) @ K.abs()
                            + f * res[1][s, h].abs())
            tol[2][s, kh] += scale * (f * ds.abs() + p * E + sub * w).t() @ Q.abs()
            tol[3][s, kh] += (f * p + sub * w).t() @ DO.abs()
    tol[2] += f * res[2].abs()
    tol[3] += f * res[3].abs()
    return res, tol


def _limits(dtype):
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0


def _inputs(lengths, HQ, HK, D, dtype, seed, tail=0):
    g = gen(seed)
    T = int(sum(lengths)) + tail
    q, do = (torch.randn(T, HQ, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    k, v = (torch.randn(T, HK, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    cu = torch.tensor([0, *np.cumsum(lengths)], dtype=torch.int32, device=DEV)
    return q, k, v, do, cu


def _check(got, ref, tol, what):
    for name, a, r, t in zip(("o", "dq", "dk", "dv"), got, ref, tol):
        err = (a.double() - r).abs()
        # results of the stored type's least step and below
        bad = ~(err <= t + torch.finfo(a.dtype).smallest_normal)
        assert not bad.any(), (what, name, int(bad.sum()), float((err / t.clamp(min=1e-30)).max()))


def _run(q, k, v, do, cu, longest, **kw):
    from solution.body.attention import varlen_attention

    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = varlen_attention(q, k, v, cu, longest, **kw)
    return o.detach(), *torch.autograd.grad(o, (q, k, v), do)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_window_vs_float64(case, dtype):
    from solution.body import _hip

    lengths, HQ, HK, D, window, sinks = CASES[case]
    q, k, v, do, cu = _inputs(lengths, HQ, HK, D, dtype, 300 + case)
    scale = D ** -0.5
    ref, tol = _reference(q, k, v, do, lengths, scale, window, sinks, *_limits(dtype))
    o = torch.full_like(q, float("nan"))
    lse = torch.full((HQ, q.shape[0]), float("nan"), device=DEV)
    low = torch.full_like(q, float("nan"))
    _hip.attn_win_fwd(q, k, v, o, cu, max(lengths), scale, window, sinks, lse=lse, o_low=low)
    grads = [torch.full_like(t, float("nan")) for t in (q, k, v)]
    back = (q, k, v, o, do, lse, *grads, cu, max(lengths), scale, window, sinks)
    _hip.attn_win_bwd(*back)
    _check([o, *grads], ref, _reference(q, k, v, do, lengths, scale, window, sinks, *_limits(dtype),
                                        low=False)[1], CASES[case])
    _hip.attn_win_bwd(*back, o_low=low)
    _check([o, *grads], ref, tol, CASES[case])
    assert ((o.double() + low.double() - ref[0]).abs() <= tol[0]).all()
    again = _run(q, k, v, do, cu, max(lengths), window=window, sinks=sinks)
    for a, b in zip([o, *grads], again):
        assert torch.equal(a, b)  # the public entry, and the same bits twice
    # a looser bound on the lengths: the windowed kernels also where nothing is left out
    _check(_run(q, k, v, do, cu, max(lengths) + window + sinks, window=window, sinks=sinks), ref, tol,
           CASES[case])


@pytest.mark.parametrize("n_seq", [65, 200, 700])
def test_many_sequences(n_seq):
    """More sequences than a wavefront has lanes, empty ones among them."""
    rng = np.random.default_rng(n_seq)
    lengths = [int(n) for n in rng.integers(0, 40, n_seq)]
    lengths[n_seq // 2] = 650
    q, k, v, do, cu = _inputs(lengths, 4, 2, 64, torch.float16, 7)
    ref, tol = _reference(q, k, v, do, lengths, 0.125, 17, 2, *_limits(torch.float16))
    _check(_run(q, k, v, do, cu, 650, window=17, sinks=2), ref, tol, n_seq)


def test_longer_bound_and_scale():
    """max_seqlen far above the longest sequence, a scale of one's own."""
    lengths = [200, 77, 900]
    q, k, v, do, cu = _inputs(lengths, 6, 2, 128, torch.bfloat16, 8)
    ref, tol = _reference(q, k, v, do, lengths, 0.2, 90, 6, *_limits(torch.bfloat16))
    _check(_run(q, k, v, do, cu, 30000, scale=0.2, window=90, sinks=6), ref, tol, "bound")


@pytest.mark.parametrize("window", [60, 200])
@pytest.mark.parametrize("tail", [1, 127, 128, 3000])
def test_tokens_behind_the_last_sequence(tail, window):
    """They get an output and gradients of 0 from varlen_attention, whatever they hold; the entry itself
    leaves their output as it was."""
    from solution.body import _hip

    lengths = [150, 40]
    q, k, v, do, cu = _inputs(lengths, 4, 2, 128, torch.bfloat16, 9, tail=tail)
    n = 190
    for t in (q, k, v, do):
        t[n:] = float("nan")
    got = _run(q, k, v, do, cu, 150, window=window, sinks=3)
    alone = _run(*(t[:n] for t in (q, k, v, do)), cu, 150, window=window, sinks=3)
    for a, b in zip(got, alone):
        assert torch.equal(a[:n], b) and not a[n:].any()
    o = torch.full_like(q, 7.0)
    _hip.attn_win_fwd(q, k, v, o, cu, 150, 128 ** -0.5, window, 3)
    assert torch.equal(o[:n], alone[0]) and (o[n:] == 7.0).all()


def test_hidden_tokens_do_not_matter():
    """Tokens that no query of a block sees may hold anything: infinities and NaN in another sequence, and
    in tiles between the sinks and the window."""
    lengths = [900, 300]
    q, k, v, do, cu = _inputs(lengths, 4, 2, 128, torch.bfloat16, 10)
    o = _run(q, k, v, do, cu, 900, window=64, sinks=4)[0]
    k2, v2 = k.clone(), v.clone()
    k2[200:300], v2[200:300] = float("nan"), float("inf")
    k2[900:], v2[900:] = float("inf"), float("nan")
    from solution.body.attention import varlen_attention

    o2 = varlen_attention(q, k2, v2, cu, 900, window=64, sinks=4)
    # queries 512 .. 899: their blocks' keys start at 449
    assert torch.equal(o[512:900], o2[512:900])


def test_views_of_one_buffer():
    """q, k and v as column blocks of one fused output, dO as a column block, a leading 1."""
    from solution.body.attention import varlen_attention

    lengths, HQ, HK, D = [400, 33], 6, 2, 64
    q, k, v, do, cu = _inputs(lengths, HQ, HK, D, torch.float16, 11)
    T = q.shape[0]
    want = _run(q, k, v, do, cu, 400, window=50, sinks=2)
    y = torch.cat([t.reshape(T, -1) for t in (q, k, v)], 1).requires_grad_()
    parts = [p.view(1, T, -1, D) for p in y.split([HQ * D, HK * D, HK * D], 1)]
    wide = torch.cat([do.reshape(T, -1), do.reshape(T, -1)], 1)
    o = varlen_attention(*parts, cu, 400, window=50, sinks=2)
    (dy,) = torch.autograd.grad(o, y, wide[:, HQ * D:].view(T, HQ, D))
    assert torch.equal(o.detach(), want[0])
    for a, b in zip(dy.split([HQ * D, HK * D, HK * D], 1), want[1:]):
        assert torch.equal(a.reshape(b.shape), b)


def test_gradients_against_differences():
    """The gradient's component along a direction against a difference of the float64 operator of the
    inputs as stored: the bound of the test above, summed over the direction, plus the difference's own."""
    lengths, D, window, sinks = [620], 64, 50, 3
    q, k, v, do, cu = _inputs(lengths, 2, 1, D, torch.float16, 12)
    got = _run(q, k, v, do, cu, 620, window=window, sinks=sinks)
    ref, tol = _reference(q, k, v, do, lengths, D ** -0.5, window, sinks, *_limits(torch.float16))
    from oracle import attention_ref

    cun, don = cu.cpu().numpy(), do.double().cpu().numpy()
    xs = [t.double().cpu().numpy() for t in (q, k, v)]
    g = np.random.default_rng(3)
    for i in range(3):
        step = g.standard_normal(xs[i].shape)
        vals = []
        for eps in (1e-4, -1e-4):
            moved = list(xs)
            moved[i] = xs[i] + eps * step
            o, _ = attention_ref.attn_fwd(*moved, cun, D ** -0.5, window, sinks)
            vals.append(float((o * don).sum()))
        slope = (vals[0] - vals[1]) / 2e-4
        along = float((got[1 + i].double().cpu().numpy() * step).sum())
        limit = float((tol[1 + i].cpu().numpy() * np.abs(step)).sum())
        assert abs(along - slope) <= limit + 1e-5 * abs(slope), (i, along, slope, limit)


def test_graph_replays():
    """Forward and backward captured, replayed between eager passes on new inputs."""
    lengths = [700, 100]
    q, k, v, do, cu = _inputs(lengths, 4, 2, 128, torch.bfloat16, 13)
    static = [t.clone() for t in (q, k, v, do)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _run(*static, cu, 700, window=80, sinks=5)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(*static, cu, 700, window=80, sinks=5)
    for seed in (20, 21, 22):
        new = _inputs(lengths, 4, 2, 128, torch.bfloat16, seed)[:4]
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        want = _run(*new, cu, 700, window=80, sinks=5)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_side_stream():
    lengths = [300, 300]
    q, k, v, do, cu = _inputs(lengths, 4, 2, 64, torch.bfloat16, 14)
    want = _run(q, k, v, do, cu, 300, window=31, sinks=1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _run(q, k, v, do, cu, 300, window=31, sinks=1)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_window_of_everything_is_causal():
    lengths = [200, 90]
    q, k, v, do, cu = _inputs(lengths, 4, 2, 128, torch.bfloat16, 15)
    want = _run(q, k, v, do, cu, 200)
    got = _run(q, k, v, do, cu, 200, window=200, sinks=9)
    assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])  # o and dv
    ref, tol = _reference(q, k, v, do, lengths, 128 ** -0.5, None, 0, 2.0 ** -8, 0.0)
    _check(got, ref, tol, "causal")  # dq and dk without o's rounding


def test_empty_inputs():
    cu = torch.zeros(2, dtype=torch.int32, device=DEV)
    q, k, v, do, _ = _inputs([0], 4, 2, 64, torch.float16, 16)
    assert all(t.numel() == 0 for t in _run(q, k, v, do, cu, 5, window=3))
    q, k, v, do, _ = _inputs([4], 4, 2, 64, torch.float16, 17)
    for c in (cu, cu[:1]):  # an empty sequence, no sequence
        for t in _run(q, k, v, do, c, 5, window=3, sinks=1):
            assert not t.any()
