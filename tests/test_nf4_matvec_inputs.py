"""What nf4_matvec hands to its kernel, without a GPU: rows that the matrix-core kernel can read, whatever views
x comes as; the gradient of a bias in the bias' own shape."""

import pytest
import torch

from solution import nf4
from solution.body import _hip
from test_nf4_matvec_args import _state

N, K = 32, 128


@pytest.fixture
def handed(monkeypatch):
    seen = []
    monkeypatch.setattr(_hip, "nf4_matvec", lambda x, items, y, **kw: seen.append(x))
    return seen


def _call(x, bias=None):
    return nf4.nf4_matvec(x, torch.zeros(N * K // 2, 1, dtype=torch.uint8), bias, _state(N, K))


def _views():
    base = torch.arange(8 * 2 * K).remainder(97).half()
    wide = base.view(8, 2 * K)
    yield "dense", base[:4 * K].view(4, K), False
    yield "column block", wide[:, K:], False
    yield "one row of many", wide[3:4, :K], False
    yield "expanded", base[:K].expand(4, K), True
    yield "overlapping", base.as_strided((4, K), (8, 1)), True
    yield "odd address", base[1:1 + 4 * K].view(4, K), True
    yield "odd row stride", base.as_strided((4, K), (K + 1, 1)), True
    yield "one row at an odd address", base[3:3 + K].view(1, K), True
    yield "columns apart", wide[:4, ::2], True
    yield "transposed", base[:4 * K].view(K, 4).t(), True


@pytest.mark.parametrize("what,x,copied", list(_views()), ids=[v[0] for v in _views()])
def test_rows_that_the_kernel_reads(handed, what, x, copied):
    y = _call(x)
    (got,) = handed
    assert y.shape == (len(x), N) and torch.equal(got, x)
    assert (got.data_ptr() != x.data_ptr()) == copied
    ld = _hip._rows_ld(got, K)  # refuses rows that overlap
    assert got.data_ptr() % 16 == 0 and ld % 8 == 0


def test_expanded_leading_dimensions(handed):
    x = torch.randn(K).half().expand(2, 3, K)
    assert _call(x).shape == (2, 3, N)
    assert torch.equal(handed[0], x.reshape(6, K)) and _hip._rows_ld(handed[0], K) == K


@pytest.mark.parametrize("shape", [(N,), (1, N), (N, 1)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_a_bias_gets_a_gradient_of_its_shape(handed, shape, dtype):
    x = torch.randn(3, K).half()
    bias = torch.zeros(shape, dtype=dtype).requires_grad_()
    dy = torch.arange(3 * N).view(3, N).half()
    (g,) = torch.autograd.grad(_call(x, bias), bias, dy)
    assert g.shape == shape and g.dtype == dtype and torch.equal(g.reshape(-1), dy.sum(0).to(dtype))
