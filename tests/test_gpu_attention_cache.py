"""Attention of the newest tokens over a cache (esep_attn_cache, cache_attention) against float64.

Bound per element, with u half a step of the stored type, as in test_gpu_attention_window.py:
u (sum p |v| + |o|) + 4e-5 of the same for the 32-bit arithmetic, and in fp16 2^-25 sum |v| for probabilities
held as subnormals. (A cut group's parts add in 32 bits.)"""

import numpy as np
import pytest
import torch

from _util import DEV, gen

pytestmark = pytest.mark.gpu


def _reference(q, k, v, lengths, scale, window, sinks, u, sub):
    B, n, HQ, D = q.shape
    G = HQ // k.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for b, length in enumerate(lengths):
        length = min(max(length, 0), k.shape[1])
        pos = torch.arange(length - n, length, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)[None, :]
        seen = j <= pos
        if window is not None:
            seen = seen & ((pos - j < window) | (j < sinks))
        some = seen.any(1)
        for h in range(HQ):
            K, V = (t[b, :length, h // G].double() for t in (k, v))
            sc = (scale * q[b, :, h].double() @ K.t()).masked_fill(~seen, -torch.inf)
            p = torch.softmax(sc, 1)
            p[~some] = 0
            # hidden keys may hold anything
            V = torch.where(seen.any(0)[:, None], V, 0.0)
            o[b, :, h] = p.nan_to_num(0.0) @ V
            f = u + 4e-5
            tol[b, :, h] = f * (p.nan_to_num(0.0) @ V.abs() + o[b, :, h].abs()) + sub * (
                seen.double() @ V.abs())
    return o, tol


def _inputs(B, n, S, HQ, HK, D, dtype, seed, layout="bshd"):
    g = gen(seed)
    q = torch.randn(B, n, HQ, D, generator=g).to(dtype).to(DEV)
    shape = (B, HK, S, D) if layout == "bhsd" else (B, S, HK, D)
    k, v = (torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(2))
    return (q, k.transpose(1, 2), v.transpose(1, 2)) if layout == "bhsd" else (q, k, v)


def _check(o, ref, tol, what):
    err = (o.double() - ref).abs()
    bad = ~(err <= tol + torch.finfo(o.dtype).smallest_normal)
    assert not bad.any(), (what, int(bad.sum()), float((err / tol.clamp(min=1e-30)).max()))


def _go(q, k, v, lengths, **kw):
    from solution.body.attention import cache_attention

    return cache_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), **kw)


# (lengths, n, S, HQ, HK, D, window, sinks, layout)
CASES = [
    ([1], 1, 1, 2, 2, 64, None, 0, "bshd"),
    ([1], 1, 40, 12, 2, 128, None, 0, "bhsd"),
    ([31, 32, 33, 64, 65, 0, 500], 1, 500, 12, 2, 128, None, 0, "bhsd"),
    ([700], 1, 1024, 14, 2, 64, None, 0, "bhsd"),
    ([9000, 3, 4000], 1, 9000, 28, 4, 128, None, 0, "bshd"),
    ([2000, 150, 60], 1, 2048, 12, 2, 128, 100, 4, "bhsd"),
    ([2000, 150, 60], 1, 2048, 8, 8, 64, 1, 0, "bshd"),
    ([2000, 999], 1, 2048, 8, 8, 64, 33, 70, "bshd"),
    ([300, 5, 77], 5, 300, 12, 2, 128, None, 0, "bhsd"),
    ([300, 40, 17], 17, 333, 14, 2, 64, 25, 3, "bshd"),      # 119 query rows
    ([1200, 64], 64, 1200, 4, 1, 128, 300, 40, "bhsd"),      # 256 query rows
    ([3, 0, 7], 7, 16, 4, 2, 64, None, 0, "bshd"),           # rows shorter than the new tokens
    ([50], 1, 64, 64, 1, 128, None, 0, "bshd"),              # 64 query heads on one kv head
    ([5000] * 3, 1, 5000, 6, 3, 128, 4096, 4096, "bhsd"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_cache_vs_float64(case, dtype):
    lengths, n, S, HQ, HK, D, window, sinks, layout = CASES[case]
    q, k, v = _inputs(len(lengths), n, S, HQ, HK, D, dtype, case, layout)
    o = _go(q, k, v, lengths, window=window, sinks=sinks)
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    ref, tol = _reference(q, k, v, lengths, D ** -0.5, window, sinks, torch.finfo(dtype).eps / 2, sub)
    _check(o, ref, tol, CASES[case])
    assert torch.equal(o, _go(q, k, v, lengths, window=window, sinks=sinks))  # the same bits twice


@pytest.mark.parametrize("rows", [64, 65, 300])
def test_many_rows(rows):
    """More rows than a wavefront has lanes, of all lengths, empty ones among them."""
    rng = np.random.default_rng(rows)
    lengths = [int(n) for n in rng.integers(0, 90, rows)]
    lengths[rows // 3] = 600
    q, k, v = _inputs(rows, 1, 600, 4, 2, 64, torch.float16, 5)
    ref, tol = _reference(q, k, v, lengths, 0.125, None, 0, 2.0 ** -11, 2.0 ** -25)
    _check(_go(q, k, v, lengths), ref, tol, rows)


def test_more_groups_than_wavefronts():
    """9600 (row, kv head) groups of one to three tiles: a wavefront walks several."""
    rng = np.random.default_rng(1)
    lengths = [int(n) for n in rng.integers(0, 96, 1200)]
    q, k, v = _inputs(1200, 1, 96, 8, 8, 64, torch.bfloat16, 6)
    ref, tol = _reference(q, k, v, lengths, 0.125, None, 0, 2.0 ** -8, 0.0)
    _check(_go(q, k, v, lengths), ref, tol, "groups")


@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 5)])
def test_what_is_not_seen_is_not_read(window, sinks):
    """NaN and infinities behind a row's length, and between the sinks and the window, change nothing."""
    lengths = [700, 33, 0, 1]
    q, k, v = _inputs(4, 1, 800, 12, 2, 128, torch.float16, 7, "bhsd")
    want = _go(q, k, v, lengths, window=window, sinks=sinks)
    for b, n in enumerate(lengths):
        for t, bad in ((k, float("nan")), (v, float("inf"))):
            t[b, n:] = bad
            if window is not None and n - window > sinks:
                t[b, sinks:n - window] = bad
    got = _go(q, k, v, lengths, window=window, sinks=sinks)
    assert torch.equal(want, got) and not got[2].any()


def test_lengths_past_the_cache_count_as_its_size():
    q, k, v = _inputs(3, 2, 50, 4, 2, 64, torch.bfloat16, 8)
    assert torch.equal(_go(q, k, v, [60, 1 << 30, -4]), _go(q, k, v, [50, 50, 0]))


def test_agrees_with_the_training_form():
    """Decoding a prompt's last token is the training form's last row, up to the order of the sums: each
    is within the bound of float64."""
    from solution.body.attention import varlen_attention

    for window, sinks in ((None, 0), (64, 4)):
        q, k, v = _inputs(1, 1, 400, 12, 2, 128, torch.bfloat16, 9)
        qs = torch.randn(400, 12, 128, generator=gen(1)).bfloat16().to(DEV)
        qs[-1] = q[0, 0]
        cu = torch.tensor([0, 400], dtype=torch.int32, device=DEV)
        o = varlen_attention(qs, k[0], v[0], cu, 400, window=window, sinks=sinks)
        ref, tol = _reference(q, k, v, [400], 128 ** -0.5, window, sinks, 2.0 ** -8, 0.0)
        _check(o[-1:][None], ref, tol, "training form")
        _check(_go(q, k, v, [400], window=window, sinks=sinks), ref, tol, "cache")


def test_strides_and_three_dims():
    """q as a slice of the fused q / k / v output, k and v as slices of one cache of both; q [B, HQ, D]."""
    B, HQ, HK, D, S = 3, 6, 2, 64, 90
    q, k, v = _inputs(B, 1, S, HQ, HK, D, torch.float16, 10)
    want = _go(q, k, v, [90, 17, 64])
    both = torch.stack((k, v), 3)  # [B, S, HK, 2, D]
    fused = torch.randn(B, 1, (HQ + 2 * HK) * D, device=DEV).half()
    fused[..., :HQ * D] = q.reshape(B, 1, -1)
    qv = fused[..., :HQ * D].view(B, 1, HQ, D)
    assert torch.equal(_go(qv, both[..., 0, :], both[..., 1, :], [90, 17, 64]), want)
    assert torch.equal(_go(qv[:, 0], k, v, [90, 17, 64]), want[:, 0])
    odd = torch.empty(B, 1, HQ, D + 1, device=DEV).half()[..., 1:]
    odd.copy_(q)
    assert torch.equal(_go(odd, k, v, [90, 17, 64]), want)


def test_long_cache_past_32_bit_offsets():
    """Batch rows more than 2^31 bytes apart, the last one's end past 2^32 bytes."""
    B, S, HK, D = 3, 1 << 21, 4, 128  # 2 GiB a row and tensor
    base = torch.zeros(B, S, HK, D, device=DEV, dtype=torch.float16)
    g = gen(11)
    n = 200
    small_k, small_v = (torch.randn(B, n, HK, D, generator=g).half().to(DEV) for _ in range(2))
    q = torch.randn(B, 1, 4, D, generator=g).half().to(DEV)
    window = n
    k, v = base, base.clone()
    for t, s in ((k, small_k), (v, small_v)):
        t[:, S - n:] = s
    o = _go(q, k, v, [S] * B, window=window)
    want = _go(q, small_k, small_v, [n] * B)
    ref, tol = _reference(q, small_k, small_v, [n] * B, D ** -0.5, None, 0, 2.0 ** -11, 2.0 ** -25)
    _check(o, ref, tol, "long")
    _check(want, ref, tol, "short")


def test_graph_replays_follow_the_lengths():
    """A captured step replayed while the cache fills: the lengths are read on the device."""
    q, k, v = _inputs(2, 1, 600, 12, 2, 128, torch.bfloat16, 12)
    lens = torch.tensor([10, 300], dtype=torch.int32, device=DEV)
    from solution.body.attention import cache_attention

    cache_attention(q, k, v, lens, window=200, sinks=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache_attention(q, k, v, lens, window=200, sinks=4)
    for step in range(1, 5):
        lens.add_(70)
        q.copy_(torch.randn(q.shape, generator=gen(step)))
        graph.replay()
        want = cache_attention(q, k, v, lens, window=200, sinks=4)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_two_streams_at_once():
    """Two calls in flight: their scratch memory is their own."""
    a = _inputs(4, 1, 3000, 12, 2, 128, torch.bfloat16, 13)
    b = _inputs(2, 3, 2500, 12, 2, 128, torch.bfloat16, 14)
    la, lb = [3000, 1, 2999, 64], [2500, 700]
    want = _go(*a, la), _go(*b, lb)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        for s, x, lens in ((s1, a, la), (s2, b, lb)):
            with torch.cuda.stream(s):
                got.append(_go(*x, lens))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


def test_gradients_are_refused():
    from solution.body import _hip

    q, k, v = _inputs(1, 1, 8, 2, 2, 64, torch.float16, 15)
    q.requires_grad_()
    with pytest.raises(_hip.EsepError, match="no gradient"):
        _go(q, k, v, [8])
    with torch.no_grad():
        _go(q, k, v, [8])
