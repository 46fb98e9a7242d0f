"""Varlen causal attention with grouped kv heads on the HIP kernels (esep_attn_fwd /
esep_attn_bwd): the consumer of the RoPE output in the packed decoder. It replaces the
reference's per-row loop over torch's scaled_dot_product_attention (solution/body/packed.py:
404-436) with one launch over all rows: q [T, HQ, D] and k, v [T, HK, D] in the packed token
layout, sequences delimited by cu_seqlens, query head h reading kv head h // (HQ // HK).

Forward saves (q, k, v, o, lse); the backward recomputes the probabilities from lse. Both
directions are deterministic (no atomics). fp16 and bf16, D in {64, 128}; other inputs are
rejected (EsepError), never silently computed another way.
"""

import torch

from . import _hip


def cu_seqlens_from_lengths(lengths, device):
    """int32 [len(lengths) + 1] prefix sums of host sequence lengths, on `device`."""
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + int(n))
    return torch.tensor(cu, dtype=torch.int32, device=device)


def supported(q, k, v, dropout=0.0):
    """Whether varlen_attention takes these inputs ([T, H, D] or [1, T, H, D] views)."""
    if dropout != 0.0 or not q.is_cuda:
        return False
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        return False
    D = q.shape[-1]
    return D in (64, 128) and q.shape[-2] % k.shape[-2] == 0 and k.shape == v.shape


def _heads_packed(t):
    rs, hs, ds = t.stride()
    if ds != 1 or hs != t.shape[2] or rs % 8 or t.data_ptr() % 16:
        t = _copy(t)
    return t


def _copy(t):
    """A dense copy at an address of its own (contiguous() gives a dense tensor back at its odd address)."""
    return t.clone(memory_format=torch.contiguous_format)


class VarlenAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, max_seqlen, scale):
        q, k, v = _heads_packed(q), _heads_packed(k), _heads_packed(v)
        T, HQ, D = q.shape
        o = torch.empty_like(q)
        lse = torch.empty((HQ, T), device=q.device, dtype=torch.float32)
        _hip.attn_fwd(q, k, v, o, cu_seqlens, max_seqlen, scale, lse=lse)
        ctx.save_for_backward(q, k, v, o, lse, cu_seqlens)
        ctx.max_seqlen, ctx.scale = int(max_seqlen), float(scale)
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, cu = ctx.saved_tensors
        do = _heads_packed(do)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        _hip.attn_bwd(q, k, v, o, do, lse, dq, dk, dv, cu, ctx.max_seqlen, ctx.scale)
        return dq, dk, dv, None, None, None


class WindowAttention(torch.autograd.Function):
    """VarlenAttention through a window: apply(q, k, v, cu_seqlens, max_seqlen, scale, window, sinks).
    Saved beside VarlenAttention's: what the rounding of o dropped, so that dq and dk do not carry it. The
    output and the gradients of tokens behind the last sequence are 0."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, max_seqlen, scale, window, sinks):
        q, k, v = _heads_packed(q), _heads_packed(k), _heads_packed(v)
        T, HQ, D = q.shape
        some = cu_seqlens.numel() > 1 and max_seqlen > 0  # else nothing is launched
        new = torch.empty if some else torch.zeros
        o = new((T, HQ, D), device=q.device, dtype=q.dtype)
        low = lse = None
        if any(ctx.needs_input_grad):
            # what the backward would refuse is refused here already: 2^24 sink rows or 2^36 floats of their partials
            # (esep_attn_win_bwd), which no smaller product reaches
            if sinks * HQ * T >= 1 << 31:
                _hip.attn_win_bwd_workspace(T, HQ, k.shape[1], D, max_seqlen, window, sinks,
                                            cu_seqlens.numel() - 1)
            low = torch.empty_like(o)
            lse = torch.empty((HQ, T), device=q.device, dtype=torch.float32)
        _hip.attn_win_fwd(q, k, v, o, cu_seqlens, max_seqlen, scale, window, sinks, lse=lse, o_low=low,
                          zero_rest=True)
        ctx.save_for_backward(q, k, v, o, low, lse, cu_seqlens)
        ctx.args = max_seqlen, scale, window, sinks
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, low, lse, cu = ctx.saved_tensors
        q, k, v, o, do = (_heads_packed(t) for t in (q, k, v, o, do))
        new = torch.empty if cu.numel() > 1 and ctx.args[0] > 0 else torch.zeros
        dq, dk, dv = (new(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
        low = low if _hip.dense16(low) else low.contiguous().clone()
        _hip.attn_win_bwd(q, k, v, o, do, lse.contiguous(), dq, dk, dv, cu.contiguous(), *ctx.args,
                          o_low=low)
        return dq, dk, dv, None, None, None, None, None


def _whole(name, value, least):
    if type(value) is int and least <= value <= 0x7FFFFFFF:
        return value
    try:
        n = int(value)
        whole = not isinstance(value, bool) and bool(n == value) and least <= n <= 0x7FFFFFFF
    except (TypeError, ValueError, OverflowError, RuntimeError):  # no number, NaN, an infinity, a tensor of many
        whole = False
    if not whole:
        raise _hip.EsepError(f"{name} must be a whole number of at least {least}, got {value!r}")
    return n


def _bound(max_seqlen, T):
    """A bound on the lengths that fits 32 bits: past those, the number of tokens says as much."""
    n = int(max_seqlen)
    if n < 0:
        raise _hip.EsepError(f"max_seqlen must be 0 or more, got {max_seqlen!r}")
    return n if n <= 0x7FFFFFFF - _ROUND else T


_ROUND = 1024  # the launches round it up to a block's tokens


def varlen_attention(q, k, v, cu_seqlens, max_seqlen, scale=None, window=None, sinks=0):
    """Causal attention within each sequence of the packed tokens. q [T, HQ, D] (or
    [1, T, HQ, D]), k, v [T, HK, D]; cu_seqlens int32 [n_seq + 1] on q's device; max_seqlen an
    int >= every sequence length, cu_seqlens from 0 on and not falling. Returns o [T, HQ, D] in q's dtype.

    Scores, softmax sums and the gradients' sums are fp32; the probabilities and, in the backward, the scores'
    gradients are rounded to q's dtype before the products with v, dO, k and q. An infinity or a NaN reaches queries
    of its own sequence only, but there also some that do not see its token.

    window (None: no bound): query i of a sequence sees key j <= i only if i - j < window (the last
    `window` tokens, its own among them, as HF's sliding_window) or j < sinks (the sequence's
    first tokens, which stay visible; without a window they always are). With a window, tokens behind the
    last sequence get an output and gradients of 0, and dq and dk do not carry the rounding of o (which keeps one
    more tensor of o's size until the backward). Where window + sinks reach max_seqlen it is the causal kernels
    that run. The backward's scratch memory grows with the sinks (esep_attn_win_bwd); what it would refuse, a forward
    with gradients refuses."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if q.dim() == 4:  # [1, T, H, D] views: the Function works on [T, H, D]
        q, k, v = q.squeeze(0), k.squeeze(0), v.squeeze(0)
    max_seqlen, sinks = _bound(max_seqlen, q.shape[0]), _whole("sinks", sinks, 0)
    if window is not None:
        window = _whole("window", window, 1)
        _hip.refuse_proxies("varlen_attention")
        return WindowAttention.apply(q, k, v, cu_seqlens, max_seqlen, float(scale), window, sinks)
    return VarlenAttention.apply(q, k, v, cu_seqlens, max_seqlen, float(scale))


_NO_GRADIENT = ("cache_attention has no gradient: call it under torch.no_grad(), or on detached tensors "
                "(varlen_attention is the form for training)")


class CacheAttention(torch.autograd.Function):
    """cache_attention where torch looks on: one node of a trace, which runs it again, and tangents are refused
    (the kernel fills its buffer behind torch's back)."""

    @staticmethod
    def forward(ctx, q, k_cache, v_cache, lengths, scale, window, sinks):
        return _cache(q, k_cache, v_cache, lengths, scale, window, sinks)

    @staticmethod
    def backward(ctx, do):
        raise _hip.EsepError(_NO_GRADIENT)

    @staticmethod
    def jvp(ctx, *tangents):
        raise _hip.EsepError(_NO_GRADIENT)


def cache_attention(q, k_cache, v_cache, lengths, scale=None, window=None, sinks=0):
    """Attention of each row's newest tokens over its cache: decoding (one new token a row), or a few new
    tokens at once. q [B, n, HQ, D] (or [B, HQ, D]: n = 1), the queries of the n newest tokens; k_cache, v_cache
    [B, S, HK, D] views (HF's [B, HK, S, D] cache transposed, say) at 16-byte addresses, with a dense head dim and
    batch, token and head strides of any multiples of 8 elements (tokens up to 2^22 apart), in which the new tokens
    are stored already; lengths int32 [B] on the same device: the tokens in each
    row's cache, the new ones the last of them. Query head h reads kv head h // (HQ // HK). fp16 and bf16, D
    in {64, 128}.

    Query t of a row sits at position p = lengths - n + t and sees key j <= p, through a window only if p - j <
    window or j < sinks, as in varlen_attention. What a cache holds past a row's length is never read; a query
    at a position below 0 (a row shorter than n) gets 0. Lengths past S count as S. Scores and sums are fp32, the
    probabilities are rounded to q's dtype before the product with v. An infinity or a NaN reaches queries of its
    own row only, but with several new tokens also some that do not see it.

    For answering only: there is no gradient, so inputs that record one in grad mode, or carry a forward-mode
    tangent, are refused. The scratch memory is of the caller's stream and, under capture, of the graph. A
    traced module (torch.jit.trace) calls it again. Returns o, of q's shape and dtype, dense."""
    sinks = _whole("sinks", sinks, 0)
    if window is not None:
        window = _whole("window", window, 1)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if _hip.recorded(q, k_cache, v_cache):  # (lengths are whole numbers)
        if (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad) and torch.is_grad_enabled():
            raise _hip.EsepError(_NO_GRADIENT)
        _hip.refuse_proxies("cache_attention")
        return CacheAttention.apply(q, k_cache, v_cache, lengths, scale, window, sinks)
    return _cache(q, k_cache, v_cache, lengths, scale, window, sinks)


def _cache(q, k_cache, v_cache, lengths, scale, window, sinks):
    q4 = q.unsqueeze(1) if q.dim() == 3 else q
    if q4.dim() == 4 and _unaligned(q4):
        q4 = _copy(q4)
    o = torch.empty(q4.shape, device=q.device, dtype=q.dtype)
    _hip.attn_cache(q4, k_cache, v_cache, o, lengths, scale, window, sinks)
    return o.squeeze(1) if q.dim() == 3 else o


def _unaligned(q):
    """The kernel reads q in 16-byte pieces."""
    b, n, h, d = q.stride()
    return d != 1 or q.data_ptr() % 16 != 0 or b % 8 != 0 or n % 8 != 0 or h % 8 != 0
