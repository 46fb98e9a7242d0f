"""Windowed attention without a GPU: what is refused, the workspace, the oracle's mask."""

import numpy as np
import pytest
import torch

from oracle import attention_ref
from solution.body import _hip
from solution.body.attention import varlen_attention


def _fwd(**kw):
    a = dict(q=16, q_rs=256, k=16, k_rs=128, v=16, v_rs=128, o=16, o_rs=256, low=None, lse=None, dt=1, T=10, HQ=4,
             HK=2, D=64, cu=16, n_seq=1, max_seqlen=10, scale=0.1, window=4, sinks=1, zero_rest=0, stream=None)
    a.update(kw)
    return _hip.lib().esep_attn_win_fwd(*a.values())


def _bwd(**kw):
    a = dict(q=16, q_rs=256, k=16, k_rs=128, v=16, v_rs=128, o=16, o_rs=256, low=16, dout=16, do_rs=256, lse=16,
             ws=16, dq=16, dq_rs=256, dk=16, dk_rs=128, dv=16, dv_rs=128, dt=1, T=10, HQ=4, HK=2, D=64,
             cu=16, n_seq=1, max_seqlen=10, scale=0.1, window=4, sinks=1, stream=None)
    a.update(kw)
    return _hip.lib().esep_attn_win_bwd(*a.values())


@pytest.mark.parametrize("call", [_fwd, _bwd])
def test_refusals(call):
    err = _hip.lib().esep_last_error
    assert call(window=0) == -2 and b"window=0" in err()
    assert call(sinks=-1) == -2 and b"sinks=-1" in err()
    assert call(dt=0) == -1
    assert call(D=96) == -2
    assert call(HQ=3) == -2
    assert call(T=-1) == -2
    assert call(q_rs=255) == -2 and b"token stride" in err()
    assert call(k_rs=(1 << 22) + 8) == -2
    assert call(q=None) == -1 and call(cu=None) == -1
    assert call(v=8) == -3 and call(k_rs=129) == -3
    assert call(low=8) == -3 and b"o_low" in err()
    assert call(scale=0.0) == -1
    assert call(T=0) == 0 and call(n_seq=0) == 0


def test_backward_refusals():
    assert _bwd(lse=None) == -1 and _bwd(ws=None) == -1 and _bwd(ws=8) == -3
    # more sink rows than a launch of their sums takes
    assert _bwd(T=1 << 30, max_seqlen=1 << 30, window=1, sinks=1 << 20) == -2
    assert b"sinks" in _hip.lib().esep_last_error()


def test_workspace():
    ws = _hip.attn_win_bwd_workspace
    base = ws(5000, 4, 2, 64, 5000, 100, 0)  # no sinks
    # delta, and dK / dV partials of two blocks per kv head or none
    assert base in (5000 * 4, 5000 * 4 + 2 * 2 * 5000 * 2 * 64)
    assert ws(5000, 4, 2, 64, 612, 100, 4) == base  # no sequence long enough for far queries
    assert ws(5000, 4, 2, 64, 613, 100, 4) > base
    assert ws(5000, 4, 2, 64, 700, 100, 599) > ws(5000, 4, 2, 64, 700, 100, 4)
    assert ws(0, 4, 2, 64, 1, 1, 0) == 0
    # a window and sinks that leave nothing out: the causal backward's
    for window, sinks in ((700, 0), (1 << 30, 5), (100, 600)):
        assert ws(5000, 4, 2, 64, 700, window, sinks) == _hip.attn_bwd_workspace(5000, 4, 2, 64)


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(window=2.5), dict(window=True),
                                dict(window=4, sinks=-1), dict(window=1 << 31), dict(sinks=0.5)])
def test_public_entry_refuses(kw):
    q, k = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(4, 1, 64, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(_hip.EsepError, match="window|sinks"):
        varlen_attention(q, k, k, cu, 4, **kw)


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(4, 1, 64, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(_hip.EsepError, match="device"):
        varlen_attention(q, k, k, cu, 4, window=2)


def test_oracle_mask():
    seen = attention_ref.visible(6, window=2, sinks=1)
    want = np.array([[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0],
                     [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]], dtype=bool)
    assert np.array_equal(seen, want)


def test_oracle_gradients_against_differences():
    g = np.random.default_rng(0)
    cu = np.array([0, 5, 5, 14], dtype=np.int32)
    q, do = g.standard_normal((2, 14, 4, 3))
    k, v = g.standard_normal((2, 14, 2, 3))
    args = (cu, 0.4, 3, 2)
    grads = attention_ref.attn_bwd(q, k, v, do, *args)
    for i in range(3):
        step = g.standard_normal((q, k, v)[i].shape)
        vals = []
        for eps in (1e-5, -1e-5):
            xs = [q, k, v]
            xs[i] = xs[i] + eps * step
            vals.append((attention_ref.attn_fwd(*xs, *args)[0] * do).sum())
        assert abs((vals[0] - vals[1]) / 2e-5 - (grads[i] * step).sum()) < 1e-7


def test_oracle_window_of_everything_is_causal():
    g = np.random.default_rng(1)
    q, k, v = g.standard_normal((3, 9, 2, 4))
    cu = np.array([0, 9], dtype=np.int32)
    a, b = attention_ref.attn_fwd(q, k, v, cu, 0.5), attention_ref.attn_fwd(q, k, v, cu, 0.5, 9, 0)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
