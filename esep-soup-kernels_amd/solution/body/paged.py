"""Paged key-value caches for answering, on the HIP kernels: which page and place each new token gets (block_tables), the
store of its key and value there (paged_store), attention over the pages (paged_attention, cache_attention's form
for them), and beams whose pages follow their parents (beam_reorder). No reference counterpart: the reference
trains, and calls with a cache run the original forward (solution/body/packed.py:736-771).

A pool of N pages holds P tokens each, k_pages and v_pages [N, P, HK, D] of fp16 or bf16, one pair to a layer (or one
allocation [L, N, P, HK, D] whose layers are its slices). Row b's token t lies in page tables[b, t // P] at place
t % P; tables int32 [B, M], so that a row has room for M * P tokens. The numbers of free pages lie in a list `free`,
of which the first `taken` are in use. A step, all of it on the device and fit for a HIP graph:

    plan = block_tables(tables, lengths, new, free, taken, page, total, update=True)
    q, k = rope(q, k, plan.positions, inv_freq)
    paged_store(k, v, k_pages, v_pages, plan.slots)
    o = paged_attention(q, k_pages, v_pages, tables, plan.lengths)

Pages go back by the host, between steps. Of the list, used = min(taken, F) entries are in use (taken also counts the
pages that were not there). A row that is done: its n numbers of 0 or more among tables[b, :ceil(lengths[b] / P)] to
free[used - n:used], taken = used - n, lengths[b] = 0; pages that rows share go back once, with the last of them.

Where taken was more than F, rows have gone short: one that did has -1 among those entries, and holds its tokens before
the first such page, j, only. A page is taken for its first token and for no later one (what lies in it for the
earlier ones would be another row's). So the row goes on once its numbers behind j have gone back as well and lengths[b] =
j * P: its tokens from there on are given anew. Left as it is, it gets slots again from its next page on, and
nothing sees the keys of the page that is missing.
"""

from typing import NamedTuple

import torch

from . import _hip
from .attention import _copy, _unaligned, _whole


class PagePlan(NamedTuple):
    """What block_tables returns (int32): slots [total] and positions [total] of the new tokens, the rows' one behind
    another; cu_seqlens [B + 1], their offsets; lengths [B] with them; taken [1], the pages in use."""

    slots: torch.Tensor
    positions: torch.Tensor
    cu_seqlens: torch.Tensor
    lengths: torch.Tensor
    taken: torch.Tensor


def block_tables(tables, lengths, new, free, taken, page, total, update=False):
    """Pages and places for new[b] more tokens of each row b of lengths[b] tokens (both int32 [B]; negative: 0), as a
    PagePlan. A page that a row begins is taken from free (int32 [F]), row by row from entry taken (int32 [1]) on,
    and written into tables (int32 [B, M], in place). page: tokens to a page. total: the sum of new, which the
    host knows; with fewer new tokens the slots behind them are -1 (paged_store leaves those out), and tokens past
    `total` are not added.

    A token whose row is full (M * page tokens, which the new lengths never pass) or for which no free page is left
    gets slot -1; in the latter case the table's entry is -1 (paged_attention sees none of that page's keys) and the
    new `taken` is more than F: the pages that were not there count, as do the tokens in the new lengths, and the
    module's text says how rows go on. With update, lengths and taken are changed in place, else they are left
    and the same call can be made again, with more pages in the list, say."""
    page, total = _whole("page", page, 1), _whole("total", total, 0)
    _hip.refuse_recorded("block_tables", tables)
    return PagePlan(*_hip.page_tables(tables, lengths, new, free, taken, page, total, update))


def paged_store(k, v, k_pages, v_pages, slots):
    """Stores the keys and values of T tokens, k and v [T, HK, D] (slices of a fused projection, say), in the pages
    [N, P, HK, D] at slots (int32 [T], block_tables'): place slot % P of page slot // P. Slots below 0 or past the pool
    are left out. Slots are one token's each: two tokens with the same one leave pieces of either there. D a multiple of 8;
    the pages at 16-byte addresses with strides of multiples of 8 elements."""
    _hip.refuse_recorded("paged_store", k, v, k_pages, v_pages)
    if k.dim() == 3 and v.dim() == 3:
        k, v = _copy(k) if _odd(k) else k, _copy(v) if _odd(v) else v
    _hip.page_store(k, v, k_pages, v_pages, slots)


def _odd(t):
    """The kernel reads k and v in 16-byte pieces."""
    ts, hs, ds = t.stride()
    return ds != 1 or ts % 8 != 0 or hs % 8 != 0 or t.data_ptr() % 16 != 0


def paged_attention(q, k_pages, v_pages, tables, lengths, scale=None, window=None, sinks=0, beams=1, shared=None):
    """cache_attention over pages: q [B, n, HQ, D] (or [B, HQ, D]: n = 1), the queries of each row's n newest tokens,
    which are stored already; k_pages, v_pages [N, P, HK, D] views at 16-byte addresses with a dense head dim and
    strides of multiples of 8 elements (tokens up to 2^22 apart; [N, HK, P, D] pages transposed, say), P a power of
    two of at least 16; tables int32 [B, M]; lengths int32 [B], the tokens in each row's pages, the new ones the
    last of them. fp16 and bf16, D in {64, 128}; query head h reads kv head h // (HQ // HK).

    Query t of a row sits at position p = lengths - n + t and sees key j <= p, through a window only if p - j < window or
    j < sinks. What lies in the pages past a row's length, before its window or in pages of other rows is never
    read. Keys of a page outside the pool (an entry of -1) are not seen. A query that sees none gets 0, as one at a
    position below 0 does. Lengths past M * P count as that. Rounding and infinities are cache_attention's. The tables' width is
    all that the host knows of the lengths: where rows are short, tables[:, :m] that just holds them takes one
    launch that suits them (300 rows of 60 tokens 7 us instead of 22); where few are long and the rest short, wide ones
    take the launches that share the long rows out (one of 2500 tokens among 256 of up to 100 26 us instead of 86).

    beams, shared (int32 [B // beams]): rows r * beams .. + beams - 1 hold their first shared[r] tokens in the same
    pages (a request's beams over its prompt). The pages are then read once for all of them instead of once for
    each (without a window; with one it makes no difference). The result is that of the rows on their own up to the order of
    the sums.

    For answering only: no gradient (inputs that record one, traces and transforms are refused). Returns o, of q's
    shape and dtype, dense."""
    sinks, beams = _whole("sinks", sinks, 0), _whole("beams", beams, 1)
    if window is not None:
        window = _whole("window", window, 1)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    _hip.refuse_recorded("paged_attention", q, k_pages, v_pages)
    if beams == 1 or window is not None:
        shared = None
    q4 = q.unsqueeze(1) if q.dim() == 3 else q
    if q4.dim() == 4 and _unaligned(q4):
        q4 = _copy(q4)
    o = torch.empty_like(q4, memory_format=torch.contiguous_format)
    _hip.attn_paged(q4, k_pages, v_pages, o, tables, lengths, scale, window, sinks, beams, shared)
    return o.squeeze(1) if q.dim() == 3 else o


def beam_reorder(parents, k_pages, v_pages, tables, lengths, start=None):
    """The beams' states follow their parents, in place: tokens start[r] .. lengths[r] - 1 (int32 [R]; start None: 0)
    of beam w of request r become what its beam parents[r, w] (int32 [R, W], head.beam_select's) held before the call. Row
    r * W + w of tables (int32 [R * W, M]) names the beam's pages; k_pages and v_pages [N, P, HK, D] of one layer, or [L,
    N, P, HK, D] of all of them, any P. A contiguous cache [B, S, HK, D] is one of B pages with a table of its row numbers.

    The beams of a request are equally long. Beams that are their own parent, or name one outside [0, W), are left
    alone, as are pages that a beam shares with its parent (the prompt's) and -1 entries; every other page in that
    range is one beam's own. Up to 32 beams. (lengths and start at a stride, as block_tables' lengths[::W], are copied
    first, one more launch.)"""
    _hip.refuse_recorded("beam_reorder", k_pages, v_pages, parents)
    if k_pages.dim() == 4 and v_pages.dim() == 4:
        k_pages, v_pages = k_pages.unsqueeze(0), v_pages.unsqueeze(0)
    start = start if start is None else start.contiguous()
    _hip.beam_reorder(parents.contiguous(), k_pages, v_pages, tables, lengths.contiguous(), start)
