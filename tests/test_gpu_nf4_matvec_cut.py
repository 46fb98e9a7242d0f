"""nf4_matvec where a wavefront's run crosses tiles and where blocks run in several rounds (the sizes and why are in
test_nf4_matvec_cut.py), against float64 with the bounds of test_gpu_nf4_matvec.py. The weights are random bytes, decoded
here by the format's definition."""

import types

import pytest
import torch

from _util import DEV, gen
from oracle import nf4_ref
from test_gpu_nf4_matvec import _check
from test_nf4_matvec_cut import CROSSING

pytestmark = pytest.mark.gpu


def _weight(N, K, seed):
    """A packed weight of random codes and scales, its quant state and W in float64."""
    g = torch.Generator(DEV).manual_seed(seed)
    nb = N * K // 64
    packed = torch.randint(0, 256, (N * K // 2,), generator=g, device=DEV, dtype=torch.uint8)
    absmax = torch.randint(0, 256, (nb,), generator=g, device=DEV, dtype=torch.uint8)
    absmax2 = 0.5 + torch.rand(-(-nb // 256), generator=g, device=DEV)
    code2 = torch.randn(256, generator=g, device=DEV)
    code, off = torch.from_numpy(nf4_ref.NF4).to(DEV), torch.tensor(0.3, device=DEV)
    st = types.SimpleNamespace(
        quant_type="nf4", blocksize=64, nested=True, shape=(N, K), absmax=absmax, code=code, offset=off,
        state2=types.SimpleNamespace(absmax=absmax2, code=code2, blocksize=256))
    c = code.double()
    w = torch.stack((c[(packed >> 4).long()], c[(packed & 15).long()]), 1).view(nb, 64)
    scale = code2.double()[absmax.long()] * absmax2.double().repeat_interleave(256)[:nb] + off.double()
    return packed.view(-1, 1), st, (w * scale[:, None]).view(N, K)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(CROSSING)))
def test_runs_across_tiles(case, dtype):
    from solution import nf4

    outs, K, rows = CROSSING[case]
    ws = [_weight(n, K, 100 * case + i) for i, n in enumerate(outs)]
    for M in rows:
        x = torch.randn(M, K, generator=gen(M)).to(dtype).to(DEV)
        biases = [torch.randn(n, generator=gen(n)).to(dtype).to(DEV) for n in outs]
        y = nf4.nf4_matvec_multi(x, [p for p, _, _ in ws], [s for _, s, _ in ws], biases)
        for part, (_, _, w), b in zip(y.split(outs, -1), ws, biases):
            _check(part, x, w, b, (CROSSING[case], M))


@pytest.mark.parametrize("N,K", [(4096, 3584), (1536, 8960)])
def test_views_of_x(N, K):
    """Expanded rows, odd addresses and odd row strides have the dense rows' bits."""
    from solution import nf4

    packed, st, w = _weight(N, K, 7)
    base = torch.randn(5 * (K + 1), generator=gen(7)).half().to(DEV)
    views = [base[:K].expand(4, K), base[1:1 + 4 * K].view(4, K), base.as_strided((4, K), (K + 1, 1)),
             base[3:3 + K].view(1, K), base.as_strided((4, K), (8, 1))]
    for x in views:
        y = nf4.nf4_matvec(x, packed, None, st)
        assert torch.equal(y, nf4.nf4_matvec(x.contiguous().clone(), packed, None, st))
    _check(nf4.nf4_matvec(views[0], packed, None, st), views[0].contiguous(), w, None, "expanded")
