"""Products of a few rows with NF4 weights without a GPU: what is refused."""

import ctypes
import re
import types
from pathlib import Path

import pytest
import torch

from solution import nf4
from solution.body import _hip


class _Weight(ctypes.Structure):
    """esep_nf4_matvec_weight (include/esep_body.h)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("packed", "absmax", "absmax2", "code2", "offset", "nf4", "bias")]
    _fields_ += [("N", ctypes.c_int64)]


def _call(n=1, K=64, dt=1, M=1, ldx=64, ldy=64, x=16, y=16, weights=True, **kw):
    arr = (_Weight * 9)()
    for i in range(9):
        f = dict(packed=16, absmax=16, absmax2=16, code2=16, offset=16, nf4=16, bias=None, N=16)
        if i == 0:
            f.update(kw)
        arr[i] = _Weight(*f.values())
    p = ctypes.addressof(arr) if weights else None
    return _hip.lib().esep_nf4_matvec(p, n, x, ldx, y, ldy, M, K, dt, None)


def test_refusals():
    err = _hip.lib().esep_last_error
    assert _call(dt=0) == -1 and b"dtype" in err()
    assert _call(n=0) == -1 and _call(n=9) == -1 and _call(weights=False) == -1
    assert _call(M=17) == -2 and _call(M=-1) == -2 and b"M=-1" in err()
    assert _call(K=0) == -2 and _call(K=(1 << 24) + 1) == -2
    assert _call(N=-1) == -2 and _call(N=3, K=32) == -2 and b"multiple of 64" in err()
    for name in ("packed", "absmax", "absmax2", "code2", "offset", "nf4"):
        assert _call(**{name: None}) == -1, name
    assert _call(ldx=63) == -2 and _call(n=5, ldy=79) == -2 and b"row strides" in err()
    assert _call(x=None) == -1 and _call(y=None) == -1
    assert _call(M=0) == 0 and _call(N=0) == 0


def test_row_limit_is_the_header_s():
    text = (Path(__file__).resolve().parents[1] / "include" / "esep_body.h").read_text()
    assert int(re.search(r"#define ESEP_NF4_MATVEC_ROWS (\d+)", text).group(1)) == nf4.MATVEC_ROWS


def _state(N, K):
    nb = N * K // 64
    return types.SimpleNamespace(
        shape=(N, K), absmax=torch.zeros(nb, dtype=torch.uint8), code=torch.zeros(16),
        offset=torch.zeros(()), state2=types.SimpleNamespace(absmax=torch.zeros(-(-nb // 256)),
                                                             code=torch.zeros(256)))


def test_public_entries_refuse():
    st, packed = _state(32, 64), torch.zeros(1024, 1, dtype=torch.uint8)
    x = torch.zeros(1, 64, dtype=torch.float16)
    with pytest.raises(_hip.EsepError, match="nf4_linear"):
        nf4.nf4_matvec(x.expand(17, 64), packed, None, st)
    with pytest.raises(_hip.EsepError, match="columns"):
        nf4.nf4_matvec(x[:, :32], packed, None, st)
    with pytest.raises(_hip.EsepError, match="float64"):
        nf4.nf4_matvec(x.double(), packed, None, st)
    for n in (0, 9):
        with pytest.raises(_hip.EsepError, match="weights"):
            nf4.nf4_matvec_multi(x, [packed] * n, [st] * n)
    with pytest.raises(_hip.EsepError, match="weights"):
        nf4.nf4_matvec_multi(x, [packed], [st], [None, None])
    with pytest.raises(_hip.EsepError, match="device"):
        nf4.nf4_matvec(x, packed, None, st)
