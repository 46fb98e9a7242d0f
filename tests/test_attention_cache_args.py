"""Attention over a cache without a GPU: what is refused, the workspace."""

import ctypes

import pytest
import torch

from solution.body import _hip
from solution.body.attention import cache_attention

_S3 = ctypes.c_int64 * 3


def _call(**kw):
    a = dict(q=16, qs=_S3(256, 256, 64), k=16, ks=_S3(1280, 128, 64), v=16, vs=_S3(1280, 128, 64), o=16,
             len=16, ws=16, dt=1, B=1, n=1, S=10, HQ=4, HK=2, D=64, scale=0.1, window=0, sinks=0,
             stream=None)
    a.update(kw)
    return _hip.lib().esep_attn_cache(*a.values())


def test_refusals():
    err = _hip.lib().esep_last_error
    assert _call(dt=0) == -1 and _call(D=96) == -2
    assert _call(HQ=3) == -2 and _call(B=-1) == -2 and _call(S=(1 << 30) + 1) == -2
    assert _call(B=1 << 20, n=8) == -2 and b"bad sizes" in err()
    assert _call(B=1 << 19, S=1 << 30) == -2 and b"too many" in err()
    assert _call(window=-1) == -2 and _call(sinks=-1) == -2
    assert _call(scale=0.0) == -1
    for name in ("q", "o", "len", "ws", "k", "v", "qs", "ks", "vs"):
        assert _call(**{name: None}) == -1, name
    for name in ("q", "k", "v", "o", "ws"):
        assert _call(**{name: 8}) == -3, name
    assert _call(ks=_S3(1280, 129, 64)) == -3 and b"multiples of 8" in err()
    assert _call(qs=_S3(-8, 256, 64)) == -3
    assert _call(vs=_S3(0, (1 << 22) + 8, 64)) == -2 and b"token stride" in err()
    assert _call(B=0) == 0 and _call(n=0) == 0


def test_workspace():
    ws = _hip.attn_cache_workspace
    # two numbers per group, then a partial per wavefront and per group, of each query row a maximum, a sum
    # and D values
    assert ws(1, 1, 64, 4, 2, 64) == 4 + (4 + 2) * 2 * 66  # a wavefront to a tile
    assert ws(1, 1, 32768, 12, 2, 128) == 4 + (512 + 2) * 6 * 130  # four tiles to each
    assert ws(64, 1, 32768, 12, 2, 128) == 256 + (1024 + 128) * 6 * 130  # four wavefronts to a CU
    assert ws(1, 16, 64, 14, 2, 64) == 16 + (24 + 8) * 32 * 66  # 112 query rows in 4 tiles
    assert ws(1, 1, 32768, 12, 2, 128, 64, 4) < ws(1, 1, 32768, 12, 2, 128)
    assert ws(0, 1, 1, 1, 1, 64) == 0


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=1.5), dict(sinks=-1)])
def test_public_entry_refuses(kw):
    q, k = torch.zeros(1, 1, 2, 64).half(), torch.zeros(1, 4, 1, 64).half()
    with pytest.raises(_hip.EsepError, match="window|sinks"):
        cache_attention(q, k, k, torch.ones(1, dtype=torch.int32), **kw)


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(1, 1, 2, 64).half(), torch.zeros(1, 4, 1, 64).half()
    with pytest.raises(_hip.EsepError, match="device"):
        cache_attention(q, k, k, torch.ones(1, dtype=torch.int32))
