"""Dense tensors at odd addresses, without a GPU: what the attention entries hand on is readable 16 bytes at a time."""

import pytest
import torch

from solution.body import _hip, attention


def _odd(*shape):
    n = torch.Size(shape).numel()
    t = torch.arange(n + 1).remainder(89).half()[1:].view(shape)
    assert t.is_contiguous() and t.data_ptr() % 16
    return t


def test_cache_attention_copies_its_queries(monkeypatch):
    seen = []
    monkeypatch.setattr(_hip, "attn_cache", lambda q, *a, **kw: seen.append(q))
    k, lengths = torch.zeros(2, 8, 1, 64).half(), torch.ones(2, dtype=torch.int32)
    for q in (_odd(2, 1, 4, 64), _odd(2, 4, 64)):
        attention.cache_attention(q, k, k, lengths)
        got = seen.pop()
        assert got.data_ptr() % 16 == 0 and torch.equal(got, q.view(2, 1, 4, 64))


@pytest.mark.parametrize("kw", [dict(), dict(window=2)], ids=["causal", "window"])
def test_varlen_attention_copies_its_inputs(monkeypatch, kw):
    seen = []
    for name in ("attn_fwd", "attn_win_fwd"):
        monkeypatch.setattr(_hip, name, lambda q, k, v, o, *a, **kw: seen.append((q, k, v, o)))
    cu = torch.tensor([0, 5], dtype=torch.int32)
    q, k, v = _odd(5, 2, 64), _odd(5, 1, 64), _odd(5, 1, 64)
    attention.varlen_attention(q, k, v, cu, 5, **kw)
    (got,) = seen
    assert all(t.data_ptr() % 16 == 0 for t in got)
    assert all(torch.equal(a, b) for a, b in zip(got, (q, k, v)))


@pytest.mark.parametrize("kw", [dict(), dict(window=2)], ids=["causal", "window"])
def test_the_backward_copies_the_gradient(monkeypatch, kw):
    seen = []
    for name in ("attn_fwd", "attn_win_fwd"):
        monkeypatch.setattr(_hip, name, lambda *a, **kw: None)
    for name in ("attn_bwd", "attn_win_bwd"):
        monkeypatch.setattr(_hip, name, lambda q, k, v, o, do, *a, **kw: seen.append(do))
    cu = torch.tensor([0, 5], dtype=torch.int32)
    q, k = torch.zeros(5, 2, 64).half().requires_grad_(), torch.zeros(5, 1, 64).half()
    do = _odd(5, 2, 64)
    torch.autograd.grad(attention.varlen_attention(q, k, k, cu, 5, **kw), q, do)
    assert seen[0].data_ptr() % 16 == 0 and torch.equal(seen[0], do)
