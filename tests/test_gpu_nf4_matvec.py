"""Products of a few rows with NF4 weights (esep_nf4_matvec, nf4_matvec, nf4_matvec_multi) against float64.

Bound per element: the codes are rounded to x's type and the result once more, u half a step of the type:
u (sum |x| |W| + |y|); products, scales and sums in 32 bits add less than (K + 80) 2^-24 of sum |x| |W| (a sum of K
terms in any order, and the scale's two roundings) and of the bias."""

import types

import numpy as np
import pytest
import torch

from _util import DEV, gen
from oracle import nf4_ref

pytestmark = pytest.mark.gpu


def _weight(N, K, seed, scale=0.05):
    """A packed weight and its quant state on the GPU, and W in float64 from the format's definition."""
    rng = np.random.default_rng(seed)
    packed, absmax, absmax2, code2, offset = nf4_ref.quantize_nf4(
        (rng.standard_normal(N * K) * scale).astype(np.float32))
    w = nf4_ref.dequantize_nf4(packed, absmax, absmax2, code2, offset, out_dtype=np.float32)

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)

    st = types.SimpleNamespace(
        quant_type="nf4", blocksize=64, nested=True, shape=(N, K), absmax=dev(absmax),
        code=dev(nf4_ref.NF4), offset=torch.tensor(float(offset), device=DEV),
        state2=types.SimpleNamespace(absmax=dev(absmax2), code=dev(code2), blocksize=256))
    return dev(packed).view(-1, 1), st, torch.from_numpy(w.astype(np.float64)).view(N, K).to(DEV)


def _check(y, x, w, bias, what):
    u = torch.finfo(y.dtype).eps / 2
    x, K = x.to(y.dtype).double(), x.shape[-1]
    ref = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if bias is not None:
        ref = ref + bias.to(y.dtype).double()
        mag = mag + bias.to(y.dtype).double().abs()
    tol = u * (mag + ref.abs()) + (K + 80) * 2.0 ** -24 * mag + torch.finfo(y.dtype).smallest_normal
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(((y.double() - ref).abs() / tol).max()))


SIZES = [(1, 64), (16, 64), (17, 128), (40, 192), (256, 1536), (1536, 896), (1000, 960), (4864, 896),
         (33, 8960), (2112, 64), (64, 18944),
         (4112, 4160)]  # two tiles to a block, 8 and 9 rows of x in LDS


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_matvec_vs_float64(size, dtype):
    from solution import nf4

    N, K = SIZES[size]
    packed, st, w = _weight(N, K, size)
    g = gen(size)
    for M in (1, 2, 7, 8, 9, 16):
        x = torch.randn(M, K, generator=g).to(dtype).to(DEV)
        bias = torch.randn(N, generator=g).to(dtype).to(DEV) if M % 2 else None
        y = nf4.nf4_matvec(x, packed, bias, st)
        assert y.dtype == dtype and y.shape == (M, N)
        _check(y, x, w, bias, (SIZES[size], M))
        assert torch.equal(y, nf4.nf4_matvec(x, packed, bias, st))
        # a row's bits do not depend on the rows beside it up to 8, nor above
        if M in (8, 16):
            lone = x[:1].repeat(1, 1) if M == 8 else torch.cat([x[:1], x[5:6].expand(8, K)])
            assert torch.equal(nf4.nf4_matvec(lone, packed, bias, st)[0], y[0])


@pytest.mark.parametrize("N,K", [(64, 65), (64, 1), (128, 7), (192, 100), (32, 898), (64, 31)])
def test_rows_that_share_scale_blocks(N, K):
    """K no multiple of 64 (a row starts within a block, within a byte when K is odd)."""
    from solution import nf4

    packed, st, w = _weight(N, K, N + K)
    for dtype, M in ((torch.float16, 1), (torch.bfloat16, 16)):
        x = torch.randn(M, K, generator=gen(K)).to(dtype).to(DEV)
        bias = torch.randn(N, generator=gen(N)).to(dtype).to(DEV)
        _check(nf4.nf4_matvec(x, packed, bias, st), x, w, bias, (N, K))


@pytest.mark.parametrize("outs,K", [((1536, 256, 256), 1536), ((130, 1, 7, 16, 33, 64, 2, 5), 128),
                                    ((8960, 8960), 256), ((48, 16), 100)])
@pytest.mark.parametrize("M", [1, 5, 12])
def test_several_weights(outs, K, M):
    """Side by side in one launch, each with tables of its own; some with a bias."""
    from solution import nf4

    ws = [_weight(n, K, 10 * i + n, scale=0.02 * (i + 1)) for i, n in enumerate(outs)]
    for i, (_, st, w) in enumerate(ws):  # a code table of each weight's own
        if i % 2:
            st.code = st.code * 2
            w *= 2
    x = torch.randn(M, 1, K, generator=gen(M)).half().to(DEV)
    biases = [torch.randn(n, generator=gen(n)).half().to(DEV) if i != 1 else None
              for i, n in enumerate(outs)]
    y = nf4.nf4_matvec_multi(x, [p for p, _, _ in ws], [s for _, s, _ in ws], biases)
    assert y.shape == (M, 1, sum(outs))
    for part, (p, st, w), b in zip(y.split(outs, -1), ws, biases):
        _check(part[:, 0], x[:, 0], w, b, outs)
        if K % 64 == 0:
            assert part.is_cuda and torch.isfinite(part).all()


def test_agrees_with_nf4_linear():
    """Within both forms' bounds of the same definition."""
    from solution import nf4

    packed, st, w = _weight(512, 1024, 3)
    x = torch.randn(4, 1024, generator=gen(4)).half().to(DEV)
    _check(nf4.nf4_matvec(x, packed, None, st), x, w, None, "matvec")
    _check(nf4.nf4_linear(x, packed, None, st), x, w, None, "linear")


def test_strided_and_unaligned_inputs():
    from solution import nf4

    N, K = 80, 256
    packed, st, w = _weight(N, K, 5)
    wide = torch.randn(3, 2 * K, generator=gen(5)).half().to(DEV)
    x = wide[:, K:]
    want = nf4.nf4_matvec(x.contiguous(), packed, None, st)
    assert torch.equal(nf4.nf4_matvec(x, packed, None, st), want)
    assert torch.equal(nf4.nf4_matvec(x.t().contiguous().t(), packed, None, st), want)
    odd = torch.empty(3, K + 1, device=DEV).half()[:, 1:]
    odd.copy_(x)
    _check(nf4.nf4_matvec(odd, packed, None, st), x, w, None, "x at an odd address")
    buf = torch.empty(packed.numel() + 3, dtype=torch.uint8, device=DEV)[3:]
    buf.copy_(packed.view(-1))
    _check(nf4.nf4_matvec(x, buf, None, st), x, w, None, "packed at an odd address")
    assert torch.equal(nf4.nf4_matvec(x.float(), packed, None, st), want)  # computes in fp16
    bias = torch.randn(N, generator=gen(6)).to(DEV)
    _check(nf4.nf4_matvec(x, packed, bias, st), x, w, bias, "fp32 bias")


def test_infinities_stay_in_their_rows():
    from solution import nf4

    packed, st, w = _weight(48, 320, 7)
    x = torch.randn(9, 320, generator=gen(7)).half().to(DEV)
    want = nf4.nf4_matvec(x, packed, None, st)
    bad = x.clone()
    bad[3, 5], bad[8, 300] = float("inf"), float("nan")
    got = nf4.nf4_matvec(bad, packed, None, st)
    keep = [0, 1, 2, 4, 5, 6, 7]
    assert torch.equal(got[keep], want[keep])
    assert got[8].isnan().all() and not got[3].isfinite().any()


def test_empty():
    from solution import nf4

    packed, st, _ = _weight(48, 64, 8)
    assert nf4.nf4_matvec(torch.empty(0, 64, device=DEV).half(), packed, None, st).shape == (0, 48)


def test_gradients():
    """dx and the biases' gradients: dx is the product with the weight in x's type (each of its N terms rounded
    once, the result once), checked against float64 and against a difference of the float64 operator."""
    from solution import nf4

    outs, K, M = (96, 40), 192, 5
    ws = [_weight(n, K, n) for n in outs]
    w = torch.cat([x[2] for x in ws])
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        g = gen(9)
        x = torch.randn(M, K, generator=g).to(dtype).to(DEV).requires_grad_()
        bs = [torch.randn(n, generator=g).to(DEV).requires_grad_() for n in outs]
        y = nf4.nf4_matvec_multi(x, [p for p, _, _ in ws], [s for _, s, _ in ws], bs)
        dy = torch.randn(M, sum(outs), generator=g).to(y.dtype).to(DEV)
        dx, db0, db1 = torch.autograd.grad(y, [x, *bs], dy)
        assert dx.dtype == dtype and db0.dtype == torch.float32
        u = torch.finfo(y.dtype).eps / 2
        ref, mag = dy.double() @ w, dy.double().abs() @ w.abs()
        assert ((dx.double() - ref).abs() <= u * (mag + ref.abs()) + 2.0 ** -15 * mag).all()
        want = dy.double().sum(0)
        got = torch.cat([db0, db1]).double()
        assert ((got - want).abs() <= 1e-5 * dy.double().abs().sum(0)).all()
        step = torch.randn(M, K, generator=g).to(DEV).double()
        slope = ((x.detach().double() + step) @ w.t() * dy.double()).sum() - (
            x.detach().double() @ w.t() * dy.double()).sum()  # linear: any step
        along = (dx.double() * step).sum()
        assert (along - slope).abs() <= ((u * (mag + ref.abs()) + 2.0 ** -15 * mag) * step.abs()).sum()
        lone = nf4.nf4_matvec(x, ws[0][0], None, ws[0][1])
        assert torch.autograd.grad(lone, x, dy[:, :96].contiguous())[0].shape == x.shape


def test_graph_replays():
    from solution import nf4

    ws = [_weight(n, 512, n) for n in (256, 80)]
    args = [p for p, _, _ in ws], [s for _, s, _ in ws]
    x = torch.randn(2, 512, generator=gen(1)).half().to(DEV)
    nf4.nf4_matvec_multi(x, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = nf4.nf4_matvec_multi(x, *args)
    for seed in (2, 3, 4):
        x.copy_(torch.randn(x.shape, generator=gen(seed)))
        graph.replay()
        want = nf4.nf4_matvec_multi(x, *args)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
