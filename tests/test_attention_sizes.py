"""Sizes and counts past 32 bits, without a GPU: no call reads them modulo 2^32."""

import pytest
import torch

from solution.body import _hip, attention


@pytest.mark.parametrize("bound", [(1 << 31) - 1, 1 << 31, 1 << 32, (1 << 32) + 3, 1 << 63])
@pytest.mark.parametrize("kw", [dict(), dict(window=2)], ids=["causal", "window"])
def test_any_bound_on_the_lengths(monkeypatch, bound, kw):
    seen = []
    for name in ("attn_fwd", "attn_win_fwd"):
        monkeypatch.setattr(_hip, name, lambda q, k, v, o, cu, longest, *a, **kw: seen.append(longest))
    q = torch.zeros(5, 2, 64).half()
    cu = torch.tensor([0, 5], dtype=torch.int32)
    attention.varlen_attention(q, q, q, cu, bound, **kw)
    assert 5 <= seen[0] < 1 << 31


@pytest.mark.parametrize("kw", [dict(), dict(window=2)], ids=["causal", "window"])
def test_negative_bounds_are_refused(kw):
    q = torch.zeros(5, 2, 64).half()
    cu = torch.tensor([0, 5], dtype=torch.int32)
    for bound in (-1, -(1 << 32) + 5):
        with pytest.raises(_hip.EsepError, match="max_seqlen"):
            attention.varlen_attention(q, q, q, cu, bound, **kw)


@pytest.mark.parametrize("B,n,S", [(1, 1, (1 << 32) + 1), (1, (1 << 32) + 1, 4), ((1 << 32) + 1, 1, 4)])
def test_caches_past_32_bits_are_refused(monkeypatch, B, n, S):
    monkeypatch.setattr(_hip, "_dev", lambda *t: torch.device("cpu"))
    q = torch.zeros(1, 1, 1, 64).half()
    k = q.expand(B, S, 1, 64)
    o = torch.empty(B, n, 1, 64, device="meta", dtype=torch.float16)
    lengths = torch.empty(B, device="meta", dtype=torch.int32)
    with pytest.raises(_hip.EsepError, match="sizes"):
        _hip.attn_cache(q.expand(B, n, 1, 64), k, k, o, lengths, 0.125)
