"""Attention of the newest tokens over pages (esep_attn_paged, paged_attention) against float64.

Bound per element, as in test_gpu_attention_cache.py: with u half a step of the stored type, u (sum p |v| + |o|) +
4e-5 of the same for the 32-bit arithmetic, and in fp16 2^-25 sum |v| for probabilities held as subnormals. (Parts of
a cut group, and of shared and own tokens, add in 32 bits.)"""

import random

import pytest
import torch

from _util import DEV, gen
from test_gpu_attention_cache import _check, _reference

pytestmark = pytest.mark.gpu


def _i(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _scatter(k, v, lengths, P, rng, layout="nphd", shared=None, beams=1, fill=float("nan"), extra=2):
    """Contiguous k, v [B, S, HK, D] in pages in a random order; what no row holds is `fill`. Returns (k pages, v pages,
    tables). With shared, the rows of a request name its first row's pages for those tokens."""
    B, S, HK, D = k.shape
    held = [-(-min(max(n, 0), S) // P) for n in lengths]
    M = max(-(-S // P), 1)
    ids = list(range(sum(held) + extra))
    rng.shuffle(ids)
    shape = (len(ids), HK, P, D) if layout == "nhpd" else (len(ids), P, HK, D)
    pages = [torch.full(shape, fill, device=DEV, dtype=k.dtype) for _ in range(2)]
    if layout == "nhpd":
        pages = [t.transpose(1, 2) for t in pages]
    tables = [[-1] * M for _ in range(B)]
    for b in range(B):
        for j in range(held[b]):
            if shared is not None and b % beams and (j + 1) * P <= shared[b // beams]:
                tables[b][j] = tables[b // beams * beams][j]
                continue
            tables[b][j] = ids.pop()
            n = min(P, min(lengths[b], S) - j * P)
            for t, src in zip(pages, (k, v)):
                t[tables[b][j], :n] = src[b, j * P:j * P + n]
    return *pages, _i(tables)


def _wide(tables, page, tokens=1 << 15):
    """The same tables with room for `tokens`: rows that may be long are walked in cut runs and joined, where short ones
    take one launch."""
    out = torch.full((tables.shape[0], max(tokens // page, tables.shape[1])), -1, dtype=torch.int32, device=DEV)
    out[:, :tables.shape[1]] = tables
    return out


def _inputs(B, n, S, HQ, HK, D, dtype, seed):
    g = gen(seed)
    q = torch.randn(B, n, HQ, D, generator=g).to(dtype).to(DEV)
    return q, *(torch.randn(B, S, HK, D, generator=g).to(dtype).to(DEV) for _ in range(2))


def _sub(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


# (lengths, n, S, HQ, HK, D, page, window, sinks, layout)
CASES = [
    ([1], 1, 16, 2, 2, 64, 16, None, 0, "nphd"),
    ([1, 0, 17], 1, 48, 12, 2, 128, 16, None, 0, "nhpd"),
    ([31, 32, 33, 64, 65, 0, 500], 1, 512, 12, 2, 128, 32, None, 0, "nphd"),
    ([700], 1, 1024, 14, 2, 64, 16, None, 0, "nphd"),
    ([9000, 3, 4000], 1, 9008, 28, 4, 128, 16, None, 0, "nhpd"),
    ([2000, 150, 60], 1, 2048, 12, 2, 128, 64, 100, 4, "nphd"),
    ([2000, 150, 60], 1, 2048, 8, 8, 64, 16, 1, 0, "nhpd"),
    ([2000, 999], 1, 2048, 8, 8, 64, 128, 33, 70, "nphd"),
    ([2000, 45, 130], 1, 2048, 6, 2, 128, 16, 40, 9, "nphd"),  # sinks and window within one tile
    ([300, 5, 77], 5, 320, 12, 2, 128, 32, None, 0, "nhpd"),
    ([300, 40, 17], 17, 336, 14, 2, 64, 16, 25, 3, "nphd"),    # 119 query rows
    ([1200, 64], 64, 1216, 4, 1, 128, 64, 300, 40, "nphd"),    # 256 query rows
    ([3, 0, 7], 7, 16, 4, 2, 64, 16, None, 0, "nphd"),         # rows shorter than the new tokens
    ([50], 1, 64, 64, 1, 128, 64, None, 0, "nhpd"),            # 64 query heads on one kv head
    ([5000] * 3, 1, 8192, 6, 3, 128, 4096, 4096, 4096, "nphd"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_paged_vs_float64(case, dtype):
    """What lies past a row's length, before its window or in other pages is NaN."""
    from solution.body.paged import paged_attention

    lengths, n, S, HQ, HK, D, page, window, sinks, layout = CASES[case]
    q, k, v = _inputs(len(lengths), n, S, HQ, HK, D, dtype, case)
    for b, length in enumerate(lengths):
        if window is not None and length - n + 1 - window > sinks:
            k[b, sinks:length - n + 1 - window] = float("inf")
            v[b, sinks:length - n + 1 - window] = float("nan")
    kp, vp, tables = _scatter(k, v, lengths, page, random.Random(case), layout)
    o = paged_attention(q, kp, vp, tables, _i(lengths), window=window, sinks=sinks)
    clean = [t.nan_to_num(0.0, 0.0, 0.0) for t in (k, v)]
    ref, tol = _reference(q, *clean, lengths, D ** -0.5, window, sinks, torch.finfo(dtype).eps / 2, _sub(dtype))
    _check(o, ref, tol, CASES[case])
    # the same bits twice, from a table whose rows are further apart
    wide = _wide(tables, page)
    part = wide[:, :tables.shape[1]]
    assert torch.equal(o, paged_attention(q, kp, vp, part, _i(lengths), window=window, sinks=sinks))
    # rows that may be long
    o = paged_attention(q, kp, vp, wide, _i(lengths), window=window, sinks=sinks)
    _check(o, ref, tol, ("wide", CASES[case]))
    assert torch.equal(o, paged_attention(q, kp, vp, wide, _i(lengths), window=window, sinks=sinks))


# (lengths of each request's beams, beams, shared, n, HQ, HK, D, page)
SHARED = [
    ([40, 40], 2, [32], 1, 4, 2, 64, 16),
    ([700] * 4 + [90] * 4, 4, [640, 64], 1, 28, 4, 128, 16),
    ([5000] * 3 + [33] * 3 + [0] * 3, 3, [4096, 16, 0], 1, 12, 2, 128, 32),
    ([200, 190, 180, 260], 2, [160, 176], 5, 14, 2, 64, 16),      # uneven beams, several new tokens
    ([900] * 8, 8, [896], 1, 28, 4, 128, 64),                     # 56 query rows in two tiles
    ([130] * 2 + [64] * 2, 2, [1 << 20, -7], 1, 8, 8, 64, 128),   # what no row has, and less than none
    ([100] * 6, 2, [96, 96, 96], 70, 2, 1, 128, 32),              # shared past what the first new token sees
    ([3] * 2, 2, [2], 7, 4, 2, 64, 16),                           # rows shorter than the new tokens
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(SHARED)))
def test_shared_pages(case, dtype):
    """Beams over a common prompt, walked together and each on its own."""
    from solution.body.paged import paged_attention

    lengths, W, shared, n, HQ, HK, D, page = SHARED[case]
    B, S = len(lengths), -(-max(lengths) // page) * page
    q, k, v = _inputs(B, n, S, HQ, HK, D, dtype, case)
    for b in range(B):  # the shared tokens are the first beam's
        s = max(0, min(shared[b // W], S))
        k[b, :s], v[b, :s] = k[b // W * W, :s].clone(), v[b // W * W, :s].clone()
    kp, vp, tables = _scatter(k, v, lengths, page, random.Random(case), shared=shared, beams=W)
    ref, tol = _reference(q, k, v, lengths, D ** -0.5, None, 0, torch.finfo(dtype).eps / 2, _sub(dtype))
    for t in (tables, _wide(tables, page)):
        o = paged_attention(q, kp, vp, t, _i(lengths), beams=W, shared=_i(shared))
        _check(o, ref, tol, ("shared", SHARED[case]))
        assert torch.equal(o, paged_attention(q, kp, vp, t, _i(lengths), beams=W, shared=_i(shared)))
        own = paged_attention(q, kp, vp, t, _i(lengths))
        _check(own, ref, tol, ("own", SHARED[case]))
    # through a window the pages are read row by row
    assert torch.equal(paged_attention(q, kp, vp, tables, _i(lengths), window=50, beams=W, shared=_i(shared)),
                       paged_attention(q, kp, vp, tables, _i(lengths), window=50))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("rows", [64, 65, 200, 300, 1100])
def test_many_rows(rows, wide):
    """More rows than a wavefront has lanes, of all lengths, empty ones among them; also as beams of nothing in common."""
    from solution.body.paged import paged_attention

    rng = random.Random(rows)
    lengths = [rng.randrange(90) for _ in range(rows)]
    lengths[rows // 3] = 600
    q, k, v = _inputs(rows, 1, 608, 4, 2, 64, torch.float16, 5)
    kp, vp, tables = _scatter(k, v, lengths, 16, rng)
    tables = _wide(tables, 16) if wide else tables
    ref, tol = _reference(q, k, v, lengths, 0.125, None, 0, 2.0 ** -11, 2.0 ** -25)
    _check(paged_attention(q, kp, vp, tables, _i(lengths)), ref, tol, rows)
    if rows % 5 == 0:
        none = _i([0] * (rows // 5))
        _check(paged_attention(q, kp, vp, tables, _i(lengths), beams=5, shared=none), ref, tol, rows)


@pytest.mark.parametrize("wide", [False, True])
def test_more_groups_than_wavefronts(wide):
    """9600 (row, kv head) groups of one to three tiles: a wavefront walks several."""
    from solution.body.paged import paged_attention

    rng = random.Random(1)
    lengths = [rng.randrange(96) for _ in range(1200)]
    q, k, v = _inputs(1200, 1, 96, 8, 8, 64, torch.bfloat16, 6)
    kp, vp, tables = _scatter(k, v, lengths, 32, rng)
    tables = _wide(tables, 32) if wide else tables
    ref, tol = _reference(q, k, v, lengths, 0.125, None, 0, 2.0 ** -8, 0.0)
    _check(paged_attention(q, kp, vp, tables, _i(lengths)), ref, tol, "groups")


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("beams", [1, 3])
@pytest.mark.parametrize("D", [64, 128])
def test_more_rows_than_wavefronts(D, beams, wide):
    """Rows of one or two parts, joined several to a block, their number no multiple of those."""
    from solution.body.paged import paged_attention

    rng = random.Random(D)
    rows, HQ, HK = 699, 3, 3
    lengths = [rng.choice([0, 1, 31, 65, 40 + rng.randrange(200)]) for _ in range(rows // beams) for _ in range(beams)]
    shared = [rng.choice([0, n // 16 * 16]) for n in lengths[::beams]]
    q, k, v = _inputs(rows, 1, 240, HQ, HK, D, torch.float16, 6)
    for b in range(rows):
        s = shared[b // beams]
        k[b, :s], v[b, :s] = k[b // beams * beams, :s].clone(), v[b // beams * beams, :s].clone()
    kp, vp, tables = _scatter(k, v, lengths, 16, rng, shared=shared if beams > 1 else None, beams=beams)
    tables = _wide(tables, 16) if wide else tables
    ref, tol = _reference(q, k, v, lengths, D ** -0.5, None, 0, 2.0 ** -11, 2.0 ** -25)
    o = paged_attention(q, kp, vp, tables, _i(lengths), beams=beams, shared=_i(shared))
    _check(o, ref, tol, "rows")


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
@pytest.mark.parametrize("B,n,HQ,HK,D", [(100, 20, 12, 2, 128), (60, 11, 12, 2, 128), (150, 9, 14, 2, 64),
                                         (300, 9, 14, 2, 64)])
def test_many_rows_of_several_query_tiles(B, n, HQ, HK, D, window, sinks):
    """Blocks of one and two wavefronts, a query tile of a kv head each; empty rows and rows shorter than n among them."""
    from solution.body.paged import paged_attention

    rng = random.Random(B)
    lengths = [rng.choice([0, 1, n - 1, n, 33, 40 + rng.randrange(110)]) for _ in range(B)]
    q, k, v = _inputs(B, n, 160, HQ, HK, D, torch.float16, 8)
    kp, vp, tables = _scatter(k, v, lengths, 16, rng)
    ref, tol = _reference(q, k, v, lengths, D ** -0.5, window, sinks, 2.0 ** -11, 2.0 ** -25)
    _check(paged_attention(q, kp, vp, tables, _i(lengths), window=window, sinks=sinks), ref, tol, "tiles")


def test_long_runs():
    """A wavefront's run is longer than the 32 tiles whose pages it reads at once."""
    from solution.body.paged import paged_attention

    rng, lengths = random.Random(2), [30011, 17, 25000] + [20000] * 9
    q, k, v = _inputs(12, 1, 30016, 8, 8, 64, torch.bfloat16, 7)
    kp, vp, tables = _scatter(k, v, lengths, 16, rng, "nhpd")
    o = paged_attention(q, kp, vp, tables, _i(lengths))
    ref, tol = _reference(q, k, v, lengths, 0.125, None, 0, 2.0 ** -8, 0.0)
    _check(o, ref, tol, "long runs")


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("n,window", [(1, None), (3, None), (2, 70), (60, None)])
def test_missing_pages_are_not_seen(page, n, window, wide):
    """Entries of -1 and past the pool: as if their keys were masked; a row of nothing else gets 0."""
    from solution.body.paged import paged_attention

    lengths, S = [200, 130, 90, 64], 256
    q, k, v = _inputs(4, n, S, 6, 2, 128, torch.float16, 8)
    kp, vp, tables = _scatter(k, v, lengths, page, random.Random(page))
    holes = [(0, 0, -1), (0, 2, 1 << 30), (1, 1, kp.shape[0]), (1, 128 // page, -5)] + [
        (3, j, -1) for j in range(64 // page)]
    hidden = torch.zeros(4, S, dtype=torch.bool, device=DEV)
    for b, j, bad in holes:
        tables[b, j] = bad
        hidden[b, j * page:(j + 1) * page] = True
    o = paged_attention(q, kp, vp, _wide(tables, page) if wide else tables, _i(lengths), window=window)
    for b, length in enumerate(lengths):
        pos = torch.arange(length - n, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)[None]
        seen = (j <= pos) & ~hidden[b, :length]
        if window is not None:
            seen &= pos - j < window
        for h in range(6):
            K, V = k[b, :length, h // 3].double(), v[b, :length, h // 3].double()
            sc = (128 ** -0.5 * q[b, :, h].double() @ K.t()).masked_fill(~seen, -torch.inf)
            p = torch.softmax(sc, 1).nan_to_num(0.0)
            want = p @ V
            tol = (2.0 ** -11 + 4e-5) * (p @ V.abs() + want.abs()) + 2.0 ** -25 * (seen.double() @ V.abs())
            _check(o[b, :, h], want, tol, (b, h))
    assert not o[3].any()


def test_missing_shared_pages_are_not_seen():
    from solution.body.paged import paged_attention

    q, k, v = _inputs(4, 1, 256, 12, 2, 128, torch.bfloat16, 9)
    k[1:], v[1:] = k[:1], v[:1]
    lengths = _i([250] * 4)
    kp, vp, tables = _scatter(k, v, [250] * 4, 32, random.Random(0), shared=[224], beams=4)
    tables[:, 3] = -1
    tables = _wide(tables, 32)
    ref = paged_attention(q, kp, vp, tables, lengths)
    o = paged_attention(q, kp, vp, tables, lengths, beams=4, shared=_i([224]))
    keep = torch.cat([torch.arange(96), torch.arange(128, 250)]).to(DEV)
    want, tol = _reference(q, k[:, keep], v[:, keep], [218] * 4, 128 ** -0.5, None, 0, 2.0 ** -8, 0.0)
    _check(o, want, tol, "shared")
    _check(ref, want, tol, "own")


def test_lengths_past_the_table_count_as_its_size():
    from solution.body.paged import paged_attention

    q, k, v = _inputs(3, 2, 48, 4, 2, 64, torch.bfloat16, 8)
    kp, vp, tables = _scatter(k, v, [48] * 3, 16, random.Random(3))
    got, want = (paged_attention(q, kp, vp, tables, _i(n)) for n in ([60, 1 << 30, -4], [48, 48, 0]))
    assert torch.equal(got, want) and not got[2].any()


def test_no_pages_and_no_rows():
    from solution.body.paged import paged_attention

    q, k, v = _inputs(2, 1, 16, 4, 2, 64, torch.float16, 9)
    kp, vp, tables = _scatter(k, v, [16, 16], 16, random.Random(4))
    assert not paged_attention(q, kp, vp, tables[:, :0], _i([5, 5])).any()  # no room at all
    for t in (tables, _wide(tables, 16)):
        assert not paged_attention(q, kp[:0], vp[:0], t, _i([5, 5])).any()  # an empty pool
        assert not paged_attention(q, kp, vp, t, _i([0, -3])).any()
    assert paged_attention(q[:0], kp, vp, tables[:0], _i([])).shape == (0, 1, 4, 64)


def test_agrees_with_the_contiguous_form():
    """Up to the order of the sums: each within its bound of float64."""
    from solution.body.attention import cache_attention
    from solution.body.paged import paged_attention

    lengths = [3000, 77, 1500]
    q, k, v = _inputs(3, 1, 3008, 12, 2, 128, torch.bfloat16, 10)
    kp, vp, tables = _scatter(k, v, lengths, 16, random.Random(5))
    ref, tol = _reference(q, k, v, lengths, 128 ** -0.5, 200, 4, 2.0 ** -8, 0.0)
    for t in (tables, _wide(tables, 16)):
        _check(paged_attention(q, kp, vp, t, _i(lengths), window=200, sinks=4), ref, tol, "pages")
    _check(cache_attention(q, k, v, _i(lengths), window=200, sinks=4), ref, tol, "cache")


@pytest.mark.parametrize("wide", [False, True])
def test_one_table_for_all_rows(wide):
    """Rows over the same pages, their table expanded."""
    from solution.body.paged import paged_attention

    q, k, v = _inputs(5, 1, 96, 6, 2, 64, torch.bfloat16, 10)
    kp, vp, tables = _scatter(k[:1], v[:1], [96], 16, random.Random(8))
    tables = _wide(tables, 16) if wide else tables
    lens = _i([96, 1, 0, 50, 64])
    got = paged_attention(q, kp, vp, tables.expand(5, -1), lens)
    assert torch.equal(got, paged_attention(q, kp, vp, tables.expand(5, -1).contiguous(), lens))
    shared = paged_attention(q, kp, vp, tables.expand(5, -1), lens, beams=5, shared=_i([96]))
    ref, tol = _reference(q, k[:1].expand(5, -1, -1, -1), v[:1].expand(5, -1, -1, -1), lens.tolist(), 0.125, None, 0,
                          2.0 ** -8, 0.0)
    _check(got, ref, tol, "expanded")
    _check(shared, ref, tol, "expanded, shared")


def test_strides_and_three_dims():
    """q as a slice of the fused q / k / v output and at an odd address, k and v pages of one allocation; [B, HQ, D]."""
    from solution.body.paged import paged_attention

    B, HQ, HK, D, lengths = 3, 6, 2, 64, [90, 17, 64]
    q, k, v = _inputs(B, 1, 96, HQ, HK, D, torch.float16, 10)
    kp, vp, tables = _scatter(k, v, lengths, 16, random.Random(6), fill=0.0)
    lens = _i(lengths)
    want = paged_attention(q, kp, vp, tables, lens)
    both = torch.stack((kp, vp), 3)  # [N, P, HK, 2, D]
    fused = torch.randn(B, 1, (HQ + 2 * HK) * D, device=DEV).half()
    fused[..., :HQ * D] = q.reshape(B, 1, -1)
    qv = fused[..., :HQ * D].view(B, 1, HQ, D)
    assert torch.equal(paged_attention(qv, both[..., 0, :], both[..., 1, :], tables, lens), want)
    assert torch.equal(paged_attention(qv[:, 0], kp, vp, tables, lens), want[:, 0])
    odd = torch.empty(B, 1, HQ, D + 1, device=DEV).half()[..., 1:]
    odd.copy_(q)
    assert torch.equal(paged_attention(odd, kp, vp, tables, lens), want)


def test_pages_past_32_bit_offsets():
    """Pages more than 2^32 bytes into the pool."""
    from solution.body.paged import paged_attention

    N, P, HK, D = 4100, 1024, 4, 128  # 4.3 GB each
    kp, vp = (torch.zeros(N, P, HK, D, device=DEV, dtype=torch.float16) for _ in range(2))
    q, k, v = _inputs(2, 1, 2048, 4, HK, D, torch.float16, 11)
    ids = [[N - 1, 7], [2050, N - 2]]
    for b in range(2):
        for j in range(2):
            kp[ids[b][j]], vp[ids[b][j]] = k[b, j * P:(j + 1) * P], v[b, j * P:(j + 1) * P]
    o = paged_attention(q, kp, vp, _i(ids), _i([2048, 2000]))
    ref, tol = _reference(q, k, v, [2048, 2000], D ** -0.5, None, 0, 2.0 ** -11, 2.0 ** -25)
    _check(o, ref, tol, "far pages")


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("beams", [1, 2])
def test_graph_replays_follow_the_lengths(beams, wide):
    """A captured step replayed while the rows grow: lengths and tables are read on the device."""
    from solution.body.paged import paged_attention

    q, k, v = _inputs(4, 1, 640, 12, 2, 128, torch.bfloat16, 12)
    kp, vp, tables = _scatter(k, v, [640] * 4, 16, random.Random(7))
    tables = _wide(tables, 16) if wide else tables
    shared = _i([0, 0]) if beams == 2 else None
    lens = _i([10, 300, 1, 64])

    def step():
        return paged_attention(q, kp, vp, tables, lens, beams=beams, shared=shared)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(1, 5):
        lens.add_(70)
        q.copy_(torch.randn(q.shape, generator=gen(i)))
        tables.copy_(tables.roll(1, 0) if beams == 1 else tables)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_two_streams_at_once():
    """Two calls in flight: their scratch memory is their own."""
    from solution.body.paged import paged_attention

    sets = []
    for i, (lengths, n, beams, shared) in enumerate((([3000, 1, 2999, 64], 1, 1, None), ([2500, 2500], 3, 2, [2048]))):
        q, k, v = _inputs(len(lengths), n, 3008, 12, 2, 128, torch.bfloat16, 13 + i)
        if shared:
            k[1], v[1] = k[0], v[0]
        kp, vp, tables = _scatter(k, v, lengths, 16, random.Random(i), shared=shared, beams=beams)
        tables = _wide(tables, 16)
        sets.append((q, kp, vp, tables, _i(lengths), None, None, 0, beams, shared and _i(shared)))
    want = [paged_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(5):
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(paged_attention(*s))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])
