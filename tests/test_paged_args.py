"""Paged caches and beam selection without a GPU: what is refused, the workspaces, torch's recorders."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from solution.body import _hip, paged
from solution.head import beam_select

_S2, _S3, _S4 = ctypes.c_int64 * 2, ctypes.c_int64 * 3, ctypes.c_int64 * 4


def _err():
    return _hip.lib().esep_last_error()


def _tables(**kw):
    a = dict(tables=16, ld=4, lengths=16, add=16, free=16, taken=16, slots=16, pos=16, cu=16, lengths_out=16,
             taken_out=16, B=2, M=4, F=8, page=16, total=2, stream=None)
    a.update(kw)
    return _hip.lib().esep_page_tables(*a.values())


def test_tables_refusals():
    for kw in (dict(B=-1), dict(M=-1), dict(F=-1), dict(page=0), dict(total=-1), dict(M=1 << 20, page=1 << 11)):
        assert _tables(**kw) == -2 and b"bad sizes" in _err(), kw
    assert _tables(ld=3) == -2 and b"overlap" in _err()
    for name in ("tables", "lengths", "add", "free", "taken", "slots", "pos", "cu", "lengths_out", "taken_out"):
        assert _tables(**{name: None}) == -1, name


def _store(**kw):
    a = dict(k=16, ks=_S2(128, 64), v=16, vs=_S2(128, 64), kp=16, kps=_S3(2048, 128, 64), vp=16,
             vps=_S3(2048, 128, 64), slots=16, T=2, N=3, page=16, HK=2, D=64, stream=None)
    a.update(kw)
    return _hip.lib().esep_page_store(*a.values())


def test_store_refusals():
    for kw in (dict(T=-1), dict(T=1 << 31)):
        assert _store(**kw) == -2 and b"number of tokens" in _err(), kw
    for kw in (dict(N=-1), dict(page=0), dict(HK=0), dict(D=4), dict(D=60), dict(N=1 << 20, page=1 << 11)):
        assert _store(**kw) == -2 and b"bad sizes" in _err(), kw
    for name in ("k", "v", "ks", "vs", "kp", "vp", "kps", "vps", "slots"):
        assert _store(**{name: None}) == -1, name
    for name in ("k", "v", "kp", "vp"):
        assert _store(**{name: 8}) == -3, name
    assert _store(ks=_S2(129, 64)) == -3 and _store(vps=_S3(2048, 130, 64)) == -3
    assert _store(T=0) == 0 and _store(N=0) == 0


def _reorder(**kw):
    a = dict(parents=16, kp=16, kps=_S4(0, 2048, 128, 64), vp=16, vps=_S4(0, 2048, 128, 64), tables=16, ld=4, lengths=16,
             start=None, R=1, W=2, M=4, L=1, N=3, page=7, HK=2, D=64, stream=None)
    a.update(kw)
    return _hip.lib().esep_beam_reorder(*a.values())


def test_reorder_refusals():
    for kw in (dict(R=-1), dict(R=65536), dict(W=0), dict(W=33), dict(M=-1), dict(L=-1), dict(L=32768),
               dict(R=60000, L=200)):
        assert _reorder(**kw) == -2 and b"bad sizes R" in _err(), kw
    assert _reorder(M=1 << 28) == -2 and b"too long" in _err()
    assert _reorder(ld=-1) == -2 and b"negative" in _err()
    for name in ("parents", "kp", "vp", "kps", "vps", "tables", "lengths"):
        assert _reorder(**{name: None}) == -1, name
    assert _reorder(kp=8) == -3 and _reorder(vps=_S4(0, 2048, 128, 66)) == -3
    assert _reorder(R=0) == 0 and _reorder(L=0) == 0 and _reorder(N=0) == 0


def _attn(**kw):
    a = dict(q=16, qs=_S3(256, 256, 64), k=16, ks=_S3(2048, 128, 64), v=16, vs=_S3(2048, 128, 64), o=16, tables=16,
             ld=4000, lengths=16, shared=None, ws=16, dt=1, B=2, n=1, M=4000, N=9, page=16, HQ=4, HK=2, D=64, scale=0.1,
             window=0, sinks=0, beams=1, stream=None)
    a.update(kw)
    return _hip.lib().esep_attn_paged(*a.values())


def test_attention_refusals():
    assert _attn(dt=0) == -1 and _attn(D=96) == -2 and _attn(scale=0.0) == -1
    for page in (0, 8, 24, 100):
        assert _attn(page=page) == -2 and b"power of two" in _err()
    assert _attn(window=-1) == -2 and _attn(sinks=-1) == -2
    for kw in (dict(HQ=3), dict(B=-1), dict(N=-1), dict(M=-1), dict(M=1 << 27), dict(B=1 << 20, n=8), dict(beams=3),
               dict(beams=0), dict(B=1 << 19, M=1 << 26)):
        assert _attn(**kw) == -2 and b"bad sizes" in _err(), kw
    assert _attn(shared=16, beams=2, window=5) == -1 and b"window" in _err()
    for name in ("q", "o", "tables", "lengths", "ws", "k", "v", "qs", "ks", "vs"):
        assert _attn(**{name: None}) == -1, name
    for name in ("q", "o", "ws", "k", "v"):
        assert _attn(**{name: 8}) == -3, name
    assert _attn(ks=_S3(2048, 129, 64)) == -3 and _attn(qs=_S3(-8, 256, 64)) == -3
    assert _attn(vs=_S3(2048, (1 << 22) + 8, 64)) == -2 and b"token stride" in _err()
    assert _attn(ld=-1) == -2 and b"negative" in _err()
    assert _attn(B=0) == 0 and _attn(n=0) == 0


def test_attention_workspace():
    ws = _hip.attn_paged_workspace
    # two numbers per group, then a partial per wavefront and per group, of each query row a maximum, a sum and D values:
    # 1025 tiles, four to a wavefront, of each of two kv heads
    assert ws(1, 1, 2048, 16, 4, 2, 64) == 4 + (512 + 2) * 2 * 66
    # two beams: their 4 rows together over up to 1024 tiles of shared tokens, and each on its own
    assert ws(2, 1, 2048, 16, 4, 2, 64, beams=2, shared=True) == 12 + (1537 + 6) * 4 * 66
    # short rows in one launch: none
    assert ws(1, 1, 44, 16, 12, 2, 128) == 0 and ws(1, 1, 64, 16, 12, 2, 128) > 0
    assert ws(64, 1, 64, 16, 28, 4, 128) == 0  # one round of large blocks, or
    assert ws(65, 1, 64, 16, 28, 4, 128) == 0 and ws(129, 1, 64, 16, 28, 4, 64) == 0  # of smaller ones
    assert ws(1000, 1, 20, 16, 28, 4, 64) == 0 and ws(1000, 1, 256, 16, 28, 4, 64) > 0  # several rounds
    assert ws(8, 1, 2048, 16, 12, 2, 128) > 0 and ws(8, 1, 2048, 16, 12, 2, 128, 300, 4) == 0  # a window keeps them short
    assert ws(8, 1, 16, 16, 12, 2, 128, beams=4, shared=True) == 0
    assert ws(0, 1, 1, 16, 1, 1, 64) == 0 and ws(1, 1, 1, 24, 1, 1, 64) == 0


def _select(**kw):
    a = dict(logits=16, ld_r=40, ld_w=10, scores=16, ws=16, o=16, p=16, t=16, dt=0, R=1, W=4, V=10, keep=4, stream=None)
    a.update(kw)
    return _hip.lib().esep_beam_select(*a.values())


def test_select_refusals():
    assert _select(dt=3) == -1 and b"dtype" in _err()
    for kw in (dict(R=-1), dict(W=0), dict(W=65), dict(V=0), dict(V=(1 << 24) + 1), dict(keep=0), dict(keep=65, V=100),
               dict(keep=41), dict(R=16385)):
        assert _select(**kw) == -2 and b"bad sizes" in _err(), kw
    assert _select(R=16000, V=1 << 24) == -2 and b"too many" in _err()
    assert _select(ld_w=-1) == -2
    for name in ("logits", "scores", "ws", "o", "p", "t"):
        assert _select(**{name: None}) == -1, name
    assert _select(ws=12) == -3
    assert _select(R=0) == 0


def test_select_workspace():
    ws = _hip.beam_select_workspace
    assert ws(1, 4, 151936, 8) == 8 * 4 * 75 * 9   # pieces of 2048
    assert ws(24, 5, 151936, 5) == 8 * 120 * 19 * 6  # of 8192
    assert ws(1, 1, 1, 1) == 16 and ws(1, 65, 10, 1) == 0


I1 = torch.ones(1, dtype=torch.int32)
TAB = torch.zeros(1, 2, dtype=torch.int32)
K = torch.zeros(3, 16, 1, 64).half()


@pytest.mark.parametrize("kw", [dict(page=0), dict(page=1.5), dict(total=-1), dict(total=None)])
def test_tables_entry_refuses(kw):
    a = dict(page=16, total=1)
    a.update(kw)
    with pytest.raises(_hip.EsepError, match="page|total"):
        paged.block_tables(TAB, I1, I1, I1, I1, **a)


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=1.5), dict(sinks=-1), dict(beams=0), dict(beams=1.5)])
def test_attention_entry_refuses(kw):
    with pytest.raises(_hip.EsepError, match="window|sinks|beams"):
        paged.paged_attention(torch.zeros(1, 1, 2, 64).half(), K, K, TAB, I1, **kw)


@pytest.mark.parametrize("keep", [0, 1.5, 65, 9])
def test_select_entry_refuses(keep):
    with pytest.raises(_hip.EsepError, match="keep"):
        beam_select(torch.zeros(1, 2, 4), torch.zeros(1, 2), keep)


CALLS = dict(
    tables=lambda x: paged.block_tables(TAB, I1, I1, I1, I1, 16, 1),
    store=lambda x: paged.paged_store(x, x, K, K, I1),
    attention=lambda x: paged.paged_attention(x, K, K, TAB, I1),
    select=lambda x: beam_select(x, torch.zeros(1, 1)),
    reorder=lambda x: paged.beam_reorder(torch.zeros(1, 1, dtype=torch.int32), x, x, TAB, I1))
SHAPES = dict(tables=(1,), store=(1, 1, 64), attention=(1, 1, 64), select=(1, 1, 64), reorder=(3, 16, 1, 64))
call = pytest.mark.parametrize("name", CALLS)


@call
def test_cpu_tensors_are_refused(name):
    with pytest.raises(_hip.EsepError, match="device"):
        CALLS[name](torch.zeros(SHAPES[name]).half())


@call
def test_recorders_are_refused(name):
    x = torch.zeros(SHAPES[name]).half()
    with pytest.raises(_hip.EsepError, match="record"):
        torch.jit.trace(CALLS[name], (x,), check_trace=False)
    with pytest.raises(_hip.EsepError, match="proxy"):
        make_fx(CALLS[name])(x)
    if name == "tables":  # whole numbers only: nothing below reaches it
        return
    with pytest.raises(_hip.EsepError, match="record"):
        torch.func.vmap(CALLS[name])(x[None])
    with pytest.raises(_hip.EsepError, match="no gradient"):
        CALLS[name](x.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(_hip.EsepError, match="device"):
        CALLS[name](x.clone().requires_grad_())
    with forward_ad.dual_level(), pytest.raises(_hip.EsepError, match="no gradient"):
        CALLS[name](forward_ad.make_dual(x, x))


class _Stand(torch.Tensor):
    pass


def test_other_classes_are_refused():
    x = torch.zeros(1, 1, 64).half().as_subclass(_Stand)
    with pytest.raises(_hip.EsepError, match="plain"):
        CALLS["attention"](x)


def _off_device(monkeypatch):
    """The checks behind the device's."""
    def passed(dev):
        raise AssertionError("not refused")

    monkeypatch.setattr(_hip, "_dev", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_hip, "_on", passed)


def test_shapes_and_types_are_refused(monkeypatch):
    _off_device(monkeypatch)
    E = _hip.EsepError
    q, two = torch.zeros(1, 1, 2, 64).half(), torch.ones(2, dtype=torch.int32)

    def tables(*a, total=1):
        return paged.block_tables(*a, 16, total)

    with pytest.raises(E, match="tables must be"):
        tables(TAB.long(), I1, I1, I1, I1)
    with pytest.raises(E, match="unit stride"):
        tables(torch.zeros(1, 4, dtype=torch.int32)[:, ::2], I1, I1, I1, I1)
    with pytest.raises(E, match="lengths"):
        tables(TAB, I1.long(), I1, I1, I1)
    with pytest.raises(E, match="lengths"):
        tables(TAB, I1[0], I1, I1, I1)
    with pytest.raises(E, match="lengths"):
        tables(TAB, two, two, I1, I1)
    with pytest.raises(E, match="new"):
        tables(TAB, I1, two, I1, I1)
    with pytest.raises(E, match="taken"):
        tables(TAB, I1, I1, I1, two)
    with pytest.raises(E, match="free"):
        tables(TAB, I1, I1, torch.ones(4, dtype=torch.int32)[::2], I1)
    k = torch.zeros(1, 1, 64).half()
    with pytest.raises(E, match="one shape"):
        paged.paged_store(k, k, K, K[:2], I1)
    with pytest.raises(E, match="one shape"):
        paged.paged_store(k, k, K.float(), K.float(), I1)
    with pytest.raises(E, match="must be"):
        paged.paged_store(k.bfloat16(), k, K, K, I1)
    with pytest.raises(E, match="must be"):
        paged.paged_store(k, k[:, :, :32], K, K, I1)
    with pytest.raises(E, match="slots"):
        paged.paged_store(k, k, K, K, I1.long())
    with pytest.raises(E, match="overlap"):
        paged.paged_store(k, k, K[:1].expand(3, -1, -1, -1), K, I1)
    with pytest.raises(E, match="unit stride on the head dim"):
        paged.paged_store(k, k, K, torch.zeros(3, 16, 1, 128).half()[..., ::2], I1)
    with pytest.raises(E, match="tables must be"):
        paged.paged_attention(q, K, K, torch.zeros(2, 2, dtype=torch.int32), I1)
    with pytest.raises(E, match="lengths"):
        paged.paged_attention(q, K, K, TAB, two)
    with pytest.raises(E, match="must be torch.float16"):
        paged.paged_attention(q.bfloat16(), K, K, TAB, I1)
    with pytest.raises(E, match="multiple of 2 beams"):
        paged.paged_attention(q, K, K, TAB, I1, beams=2, shared=I1)
    with pytest.raises(E, match="N, P, HK, D"):
        paged.paged_attention(q, K[None], K[None], TAB, I1)
    with pytest.raises(E, match="logits must be"):
        beam_select(torch.zeros(2, 4), torch.zeros(1, 2))
    with pytest.raises(E, match="scores"):
        beam_select(torch.zeros(1, 2, 4), torch.zeros(2))
    with pytest.raises(E, match="scores"):
        beam_select(torch.zeros(1, 2, 4), torch.zeros(1, 2).half())
    with pytest.raises(E, match="parents"):
        paged.beam_reorder(torch.zeros(1, 1), K, K, TAB, I1)
    with pytest.raises(E, match="tables must be"):
        paged.beam_reorder(torch.zeros(1, 2, dtype=torch.int32), K, K, TAB, I1)
    with pytest.raises(E, match="overlap"):
        paged.beam_reorder(torch.zeros(1, 1, dtype=torch.int32), K.expand(2, 3, 16, 1, 64), K.expand(2, 3, 16, 1, 64),
                           TAB, I1)
