"""The serving operators together: a decoder layer on 4-bit weights answering token by token (few-row NF4
products, norm, RoPE, cache attention with a window and sinks, SwiGLU), eager and captured, and the windowed
training form on the same sequences, against one float64 layer over the whole sequences.

Bound: the layer's output is residual + attention + MLP terms, each behind a chain of at most nine values rounded
to fp16 (weights' codes, norm, q / k / v, rotated q / k, probabilities, attention, the projections, SwiGLU). A
rounding is u = 2^-11 of its value at most; through a product of random vectors its share of the norm is
kept, through the two norms and the softmax (scores of deviation about 1) it grows by less than 2 each. The
2-norm of the error is held under 9 * 4 u of the reference's, per token."""

import types

import numpy as np
import pytest
import torch

from _util import DEV, gen
from test_gpu_nf4_matvec import _weight

pytestmark = pytest.mark.gpu

H, INNER, HQ, HK, D, EPS, WINDOW, SINKS = 256, 512, 4, 2, 64, 1e-6, 24, 3
U = 2.0 ** -11


def _layer():
    g, s = gen(40), types.SimpleNamespace()
    sizes = dict(q=(HQ * D, H), k=(HK * D, H), v=(HK * D, H), o=(H, HQ * D), gate=(INNER, H),
                 up=(INNER, H), down=(H, INNER))
    for i, (name, (n, k)) in enumerate(sizes.items()):
        setattr(s, name, _weight(n, k, i, scale=k ** -0.5))
    s.bias = {n: (0.1 * torch.randn(sizes[n][0], generator=g)).half().to(DEV) for n in "qkv"}
    s.w1, s.w2 = ((1 + 0.1 * torch.randn(H, generator=g)).to(DEV) for _ in range(2))
    s.inv = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return s


def _norm64(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()


def _rope64(x, pos, inv):
    ang = pos.double()[:, None] * inv.to(x.device)[None]
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _reference(s, r):
    """The layer's residual stream of one sequence in float64."""
    n = r.shape[0]
    r = r.double()
    pos = torch.arange(n, device=r.device)
    y = _norm64(r, s.w1)
    q, k, v = (y @ getattr(s, m)[2].t() + s.bias[m].double() for m in "qkv")
    q, k = (_rope64(t.view(n, -1, D), pos, s.inv) for t in (q, k))
    v = v.view(n, HK, D)
    seen = (pos[None] <= pos[:, None]) & ((pos[:, None] - pos[None] < WINDOW) | (pos[None] < SINKS))
    o = torch.empty_like(q)
    for h in range(HQ):
        kh = h // (HQ // HK)
        p = torch.softmax((q[:, h] @ k[:, kh].t() * D ** -0.5).masked_fill(~seen, -torch.inf), 1)
        o[:, h] = p @ v[:, kh]
    r = r + o.reshape(n, -1) @ s.o[2].t()
    y = _norm64(r, s.w2)
    a, b = y @ s.gate[2].t(), y @ s.up[2].t()
    return r + (a * torch.sigmoid(a) * b) @ s.down[2].t()


def _half(s, r, product, product_multi, attend):
    """The layer on r [T, H] fp32 through the framework; attend(y's q, k, v [T, heads, D]) -> [T, HQ * D]."""
    from solution.body import norm_rope
    from solution.swiglu import swiglu

    _, y = norm_rope.add_rmsnorm(r, None, s.w1, EPS, torch.float16)
    ws = [getattr(s, m) for m in "qkv"]
    qkv = product_multi(y, [w[0] for w in ws], [w[1] for w in ws], [s.bias[m] for m in "qkv"])
    q, k, v = (t.view(r.shape[0], -1, D) for t in qkv.split([HQ * D, HK * D, HK * D], -1))
    o = product(attend(q, k, v), s.o[0], None, s.o[1])
    r, y = norm_rope.add_rmsnorm(r, o, s.w2, EPS, torch.float16)
    gu = product_multi(y, [s.gate[0], s.up[0]], [s.gate[1], s.up[1]], None)
    h = swiglu(gu[..., :INNER].contiguous(), gu[..., INNER:].contiguous())
    return r + product(h, s.down[0], None, s.down[1]).float()


def _check(got, ref, what):
    err = (got.double() - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert (err < 36 * U).all(), (what, float(err.max() / U))


def _sequences():
    g = gen(41)
    lens = [60, 1, 33]
    return lens, [torch.randn(n + 4, H, generator=g).to(DEV) for n in lens]


def _decoder(s, lens):
    """(step(r [B, H], k_cache, v_cache, lengths) -> r', caches): one token a row, its k and v stored."""
    from solution import nf4
    from solution.body import norm_rope
    from solution.body.attention import cache_attention

    inv = s.inv.float().to(DEV)
    kc, vc = (torch.full((len(lens), HK, 80, D), float("nan"), device=DEV).half() for _ in range(2))
    rows = torch.arange(len(lens), device=DEV)

    def step(r, lengths):
        pos = (lengths - 1).long()

        def attend(q, k, v):
            q, k = norm_rope.rope(q, k, pos, inv)
            kc[rows, :, pos], vc[rows, :, pos] = k, v
            return cache_attention(q, kc.transpose(1, 2), vc.transpose(1, 2), lengths, window=WINDOW,
                                   sinks=SINKS).reshape(r.shape[0], -1)

        return _half(s, r, nf4.nf4_matvec, nf4.nf4_matvec_multi, attend)

    return step, kc, vc


@torch.no_grad()
def test_answering_token_by_token():
    s = _layer()
    lens, rs = _sequences()
    refs = [_reference(s, r) for r in rs]
    step, kc, vc = _decoder(s, lens)
    lengths = torch.zeros(3, dtype=torch.int32, device=DEV)
    for t in range(max(lens)):  # the prompts, a token at a time; a row that is done repeats its last
        at = [min(t, n - 1) for n in lens]
        lengths.copy_(torch.tensor(at) + 1)
        out = step(torch.stack([r[a] for r, a in zip(rs, at)]), lengths)
        _check(out, torch.stack([f[a] for f, a in zip(refs, at)]), t)
    # the answers: captured once, replayed
    x = torch.empty(3, H, device=DEV)
    lengths.copy_(torch.tensor(lens) + 1)
    x.copy_(torch.stack([r[n] for r, n in zip(rs, lens)]))
    step(x, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, lengths)
    for t in range(4):
        lengths.copy_(torch.tensor(lens) + 1 + t)
        x.copy_(torch.stack([r[n + t] for r, n in zip(rs, lens)]))
        graph.replay()
        eager = step(x, lengths)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        _check(out, torch.stack([f[n + t] for f, n in zip(refs, lens)]), ("answer", t))


def test_training_form_of_the_same_layer():
    """The whole sequences packed through the windowed attention and nf4_linear: the same layer, and its
    gradient reaches the input."""
    from solution import nf4
    from solution.body import norm_rope
    from solution.body.attention import varlen_attention

    s = _layer()
    lens, rs = _sequences()
    full = [n + 4 for n in lens]
    cu = torch.tensor([0, *np.cumsum(full)], dtype=torch.int32, device=DEV)
    inv = s.inv.float().to(DEV)

    def attend(q, k, v):
        q, k = norm_rope.rope(q, k, None, inv, cu_seqlens=cu)
        return varlen_attention(q, k, v, cu, max(full), window=WINDOW, sinks=SINKS).reshape(q.shape[0], -1)

    def multi(x, ws, states, biases):
        biases = biases or [None] * len(ws)
        return torch.cat([nf4.nf4_linear(x, w, b, st) for w, st, b in zip(ws, states, biases)], -1)

    r = torch.cat(rs).requires_grad_()
    out = _half(s, r, nf4.nf4_linear, multi, attend)
    _check(out.detach(), torch.cat([_reference(s, x) for x in rs]), "training")
    r64 = [x.double().requires_grad_() for x in rs]
    g = torch.randn(out.shape, generator=gen(42)).to(DEV)
    (got,) = torch.autograd.grad(out, r, g)
    want = torch.autograd.grad([_reference(s, x) for x in r64], r64, list(g.double().split(full)))
    _check(got, torch.cat(want), "gradient")
