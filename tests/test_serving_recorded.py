"""The windowed, cache and few-row operators where torch records them, without a GPU: a stand-in takes the
kernel's place and fills the output by its address, as the kernel does. A trace runs the operator again on its
inputs, tangents and proxy graphs are refused, modes that only look on change nothing."""

import ctypes
import types

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from solution import nf4
from solution.body import _hip
from solution.body.attention import cache_attention, varlen_attention


def _fill(out, src):
    """out = src's first elements again and again, past torch."""
    n, step = out.numel() * out.element_size(), min(out.numel(), src.numel()) * src.element_size()
    for at in range(0, n, step):
        ctypes.memmove(out.data_ptr() + at, src.data_ptr(), min(step, n - at))


@pytest.fixture
def stand_ins(monkeypatch):
    monkeypatch.setattr(_hip, "attn_cache", lambda q, k, v, o, *a, **kw: _fill(o, q))
    monkeypatch.setattr(_hip, "attn_win_fwd", lambda q, k, v, o, *a, **kw: _fill(o, q))
    monkeypatch.setattr(_hip, "nf4_matvec", lambda x, items, y, **kw: _fill(y, x))


K = torch.ones(1, 4, 1, 64).half()
LENGTHS = torch.ones(1, dtype=torch.int32)
CU = torch.tensor([0, 1], dtype=torch.int32)
STATE = types.SimpleNamespace(
    shape=(64, 64), absmax=torch.zeros(64, dtype=torch.uint8), code=torch.zeros(16), offset=torch.zeros(()),
    state2=types.SimpleNamespace(absmax=torch.zeros(1), code=torch.zeros(256)))
PACKED = torch.zeros(2048, 1, dtype=torch.uint8)

CALLS = dict(
    cache=(lambda q: cache_attention(q, K, K, LENGTHS), (1, 1, 2, 64)),
    cache_three_dims=(lambda q: cache_attention(q, K, K, LENGTHS, window=2), (1, 2, 64)),
    window=(lambda q: varlen_attention(q, K[0, :1], K[0, :1], CU, 4, window=2), (1, 2, 64)),
    matvec=(lambda x: nf4.nf4_matvec(x, PACKED, None, STATE), (2, 64)))
call = pytest.mark.parametrize("name", CALLS)


@call
def test_trace_runs_the_operator_again(stand_ins, name):
    f, shape = CALLS[name]
    a, b = (torch.randn(shape).half() for _ in range(2))
    traced = torch.jit.trace(f, (a,), check_trace=False)
    for x in (a, b, a):
        assert torch.equal(traced(x), f(x)) and torch.equal(f(x), x)


@call
def test_tangents_are_refused(stand_ins, name):
    f, shape = CALLS[name]
    x = torch.randn(shape).half()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((_hip.EsepError, NotImplementedError)):
            f(dual)
        assert torch.equal(f(x), x)  # without one


def test_a_tangent_of_the_cache_is_refused(stand_ins):
    q = torch.randn(1, 1, 2, 64).half()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(K, torch.ones_like(K))
        for k, v in ((dual, K), (K, dual)):
            with pytest.raises(_hip.EsepError, match="no gradient"):
                cache_attention(q, k, v, LENGTHS)


@call
def test_proxy_graphs_are_refused(stand_ins, name):
    f, shape = CALLS[name]
    with pytest.raises(_hip.EsepError, match="proxy"):
        make_fx(f)(torch.randn(shape).half())


@call
def test_modes_and_compilers_that_leave_the_call_alone(stand_ins, name):
    f, shape = CALLS[name]
    x = torch.randn(shape).half()
    with FlopCounterMode(display=False):
        assert torch.equal(f(x), x)
    assert torch.equal(torch.compile(f, backend="eager")(x), x)
    with torch.inference_mode():
        assert torch.equal(f(x), x)
