"""Block tables and slots, the store of new keys and values, and the beams' reordering (block_tables, paged_store,
beam_reorder) against their definitions, a token at a time on the host: whole numbers and copies, compared bit for bit."""

import random

import pytest
import torch

from _util import DEV, gen

pytestmark = pytest.mark.gpu


def _i(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ----------------------------------------------------------------------------------------
# block tables
# ----------------------------------------------------------------------------------------
def _tables_ref(tables, lengths, new, free, taken, page, total):
    tables, slots, positions, cu, out = [list(r) for r in tables], [], [], [0], []
    M = len(tables[0]) if tables else 0
    cap, taken = M * page, max(taken, 0)
    for row, n0, n in zip(tables, lengths, new):
        n0, n = min(max(n0, 0), cap), min(max(n, 0), total - len(slots))
        for t in range(n0, n0 + n):
            j = t // page
            if t < cap and t % page == 0:
                row[j] = max(free[taken], -1) if taken < len(free) else -1
                taken += 1
            slots.append(row[j] * page + t % page if t < cap and row[j] >= 0 else -1)
            positions.append(t)
        cu.append(len(slots))
        out.append(min(n0 + n, cap))
    pad = total - len(slots)
    return tables, slots + [-1] * pad, positions + [0] * pad, cu, out, [taken]


def _tables_case(rng, B, M, page, most, spare=0, odd=False):
    lengths = [rng.randint(0, M * page) for _ in range(B)]
    new = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(B)]
    if odd:
        for b in range(0, B, 5):
            lengths[b], new[b] = rng.choice([(-3, 2), (M * page + 9, 4), (5, -7), (0, 0)])
    held = [-(-min(max(n, 0), M * page) // page) for n in lengths]
    ids = list(range(sum(held) + sum(-(-max(n, 0) // page) + 1 for n in new) + spare))
    rng.shuffle(ids)
    it = iter(ids)
    tables = [[next(it) for _ in range(h)] + [-9] * (M - h) for h in held]
    taken = rng.randint(0, 5)
    return tables, lengths, new, [-5] * taken + list(it), taken


def _run_tables(tables, lengths, new, free, taken, page, total, update=False, ld=None):
    from solution.body.paged import block_tables

    B, M = len(tables), len(tables[0]) if tables else 0
    wide = torch.full((B, ld or M), 77, dtype=torch.int32, device=DEV)
    t = wide[:, :M]
    if B:
        t.copy_(_i(tables))
    ln, tk = _i(lengths), _i([taken])
    p = block_tables(t, ln, _i(new), _i(free), tk, page, total, update=update)
    if not update:
        assert ln.tolist() == lengths and tk.tolist() == [taken]
    assert (wide[:, M:] == 77).all()
    return t.tolist(), *(x.tolist() for x in (p.slots, p.positions, p.cu_seqlens, p.lengths, p.taken))


@pytest.mark.parametrize("update", [False, True])
@pytest.mark.parametrize("B,M,page,most", [(1, 1, 1, 1), (1, 9, 16, 40), (64, 5, 16, 1), (255, 3, 32, 20),
                                           (256, 7, 16, 30), (257, 4, 128, 300), (700, 6, 7, 25), (3, 400, 16, 5000)])
def test_tables(B, M, page, most, update):
    rng = random.Random(B * 31 + M)
    for odd in (False, True):
        case = _tables_case(rng, B, M, page, most, odd=odd)
        total = sum(max(n, 0) for n in case[2])
        for n in {total, total + 5, total + 3000, max(total - 3, 0), total // 2, 0}:
            want = _tables_ref(*case, page, n)
            assert _run_tables(*case, page, n, update, ld=M + 3) == want, (odd, n, total)


@pytest.mark.parametrize("update", [False, True])
@pytest.mark.parametrize("n", [1, 300])
def test_free_list_runs_out(n, update):
    """Rows that get no page have -1 in the table and in the slots; `taken` says how many were missing. A bad number in the
    list is no page either."""
    page, M = 16, 40
    tables, lengths, new = [[3] + [0] * (M - 1), [-1] * M, [-1] * M], [10, 0, 0], [n, n, 3 * n]
    for free in ([], [7], [-2, 9, 1 << 30], [8, 9, 10, 11]):
        case = tables, lengths, new, free, 0
        want = _tables_ref(*case, page, 5 * n)
        if 1 << 30 in free:  # a slot that 32 bits do not hold
            want = (want[0], [s if s < 1 << 31 else -1 for s in want[1]], *want[2:])
        assert _run_tables(*case, page, 5 * n, update) == want


def test_no_rows():
    assert _run_tables([], [], [], [4], 0, 16, 3) == ([], [-1] * 3, [0] * 3, [0], [], [0])


def test_step_by_step_in_a_graph():
    """A captured step whose lengths, tables and pages in use go on from replay to replay."""
    from solution.body.paged import block_tables

    B, M, page = 5, 6, 16
    lengths0, free0 = [0, 15, 16, 31, 90], list(range(100, 140))
    held = [-(-n // page) for n in lengths0]
    tables0 = [[50 + 10 * b + j for j in range(h)] + [-1] * (M - h) for b, h in enumerate(held)]
    tables, lengths, free, taken, new = _i(tables0), _i(lengths0), _i(free0), _i([0]), _i([1, 1, 1, 0, 2])
    block_tables(tables, lengths, new, free, taken, page, 6)  # changes the tables alone, to what the next call finds
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = block_tables(tables, lengths, new, free, taken, page, 6, update=True)
    state = tables0, lengths0, 0
    for _ in range(20):
        graph.replay()
        torch.cuda.synchronize()
        t, slots, pos, cu, lens, tk = _tables_ref(state[0], state[1], new.tolist(), free0, state[2], page, 6)
        assert tables.tolist() == t and lengths.tolist() == lens and taken.tolist() == tk
        assert plan.slots.tolist() == slots and plan.positions.tolist() == pos and plan.cu_seqlens.tolist() == cu
        assert plan.lengths is lengths and plan.taken is taken
        state = t, lens, tk[0]


# ----------------------------------------------------------------------------------------
# the store
# ----------------------------------------------------------------------------------------
def _pages(shape, dtype, seed, layout="nphd"):
    t = torch.randn(shape, generator=gen(seed)).to(dtype).to(DEV)
    if layout == "nhpd":
        t = t.transpose(-2, -3).contiguous().transpose(-2, -3)
    return t


def _store_ref(k, pages, slots):
    out, P = pages.clone(), pages.shape[1]
    for t, s in enumerate(slots):
        if 0 <= s < out.shape[0] * P:
            out[s // P, s % P] = k[t]
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,N,P,HK,D,layout", [(1, 1, 16, 1, 64, "nphd"), (37, 9, 16, 2, 128, "nhpd"),
                                               (5, 3, 7, 3, 8, "nphd"), (100, 40, 5, 12, 128, "nphd"),
                                               (9, 4, 16, 40, 256, "nhpd"), (1000, 70, 16, 4, 64, "nhpd")])
def test_store(T, N, P, HK, D, layout, dtype):
    from solution.body.paged import paged_store

    rng = random.Random(T)
    slots = rng.sample(range(N * P), min(T, N * P)) + [-1] * (T - min(T, N * P))
    rng.shuffle(slots)
    for at, bad in zip(rng.sample(range(T), T // 4), [-1, N * P, -(1 << 31), (1 << 31) - 1] * T):
        slots[at] = bad
    kp, vp = _pages((N, P, HK, D), dtype, 1, layout), _pages((N, P, HK, D), dtype, 2, layout)
    fused = torch.randn(T, 3 * HK, D, generator=gen(3)).to(dtype).to(DEV)
    odd = torch.randn(T, HK, D + 1, generator=gen(4)).to(dtype).to(DEV)[..., 1:]
    for k, v in ((fused[:, HK:2 * HK], fused[:, 2 * HK:]), (odd, fused[:, :HK])):
        want = _store_ref(k, kp, slots), _store_ref(v, vp, slots)
        paged_store(k, v, kp, vp, _i(slots))
        assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_store_nothing():
    from solution.body.paged import paged_store

    kp, vp = _pages((2, 16, 1, 64), torch.float16, 1), _pages((2, 16, 1, 64), torch.float16, 2)
    want = kp.clone()
    paged_store(kp[0, :0], vp[0, :0], kp, vp, _i([]))
    paged_store(kp[0, :1].clone(), vp[0, :1], kp[:0], vp[:0], _i([0]))
    assert torch.equal(kp, want)


def test_store_past_32_bits():
    """Pages whose end lies past 2^32 bytes."""
    from solution.body.paged import paged_store

    N, P, HK, D = 4100, 1024, 4, 128  # 4.3 GB each
    kp, vp = (torch.zeros(N, P, HK, D, dtype=torch.float16, device=DEV) for _ in range(2))
    k, v = _pages((3, HK, D), torch.float16, 1), _pages((3, HK, D), torch.float16, 2)
    slots = [N * P - 1, 5, (N // 2) * P + 3]
    paged_store(k, v, kp, vp, _i(slots))
    for pages, x in ((kp, k), (vp, v)):
        flat = pages.view(N * P, HK, D)
        for t, s in enumerate(slots):
            assert torch.equal(flat[s], x[t])
            flat[s] = 0
        assert not pages.view(torch.int64).any()


# ----------------------------------------------------------------------------------------
# the beams' reordering
# ----------------------------------------------------------------------------------------
def _reorder_ref(parents, pages, tables, lengths, start):
    out, (L, N, P) = pages.clone(), pages.shape[:3]
    W = len(parents[0]) if parents else 0
    for r, row in enumerate(parents):
        end = min(lengths[r], len(tables[0]) * P)
        for w, parent in enumerate(row):
            if parent == w or not 0 <= parent < W:
                continue
            for t in range(max(start[r], 0) if start else 0, end):
                src, dst = tables[r * W + parent][t // P], tables[r * W + w][t // P]
                if src != dst and 0 <= src < N and 0 <= dst < N:
                    out[:, dst, t % P] = pages[:, src, t % P]
    return out


def _parents(rng, R, W, how):
    if how == "swap":
        return [rng.sample(range(W), W) for _ in range(R)]
    if how == "one":
        return [[rng.randrange(W)] * W for _ in range(R)]
    if how == "none":
        return [list(range(W)) for _ in range(R)]
    return [[rng.choice([rng.randrange(W), rng.randrange(W), w, -1, W, 1 << 30]) for w in range(W)] for _ in range(R)]


@pytest.mark.parametrize("how", ["swap", "one", "none", "any"])
@pytest.mark.parametrize("R,W,L,P,HK,D,top,dtype", [
    (1, 2, 1, 16, 1, 64, 1, torch.float16), (3, 4, 2, 16, 2, 128, 90, torch.bfloat16),
    (2, 5, 3, 7, 3, 64, 40, torch.float16), (4, 8, 1, 32, 4, 128, 100, torch.bfloat16),
    (2, 16, 2, 16, 2, 64, 50, torch.float16), (1, 32, 1, 16, 5, 64, 33, torch.bfloat16),
    (2, 3, 1, 64, 20, 256, 70, torch.float16), (1, 1, 1, 16, 1, 64, 20, torch.float16),
    (2, 3, 1, 100, 4, 128, 270, torch.bfloat16), (1, 4, 2, 333, 1, 64, 600, torch.float16)])
def test_reorder(R, W, L, P, HK, D, top, dtype, how):
    from solution.body.paged import beam_reorder

    rng = random.Random(R * 100 + W)
    M = -(-top // P) + 1
    lengths = [rng.randint(0, top) for _ in range(R)]
    lengths[0] = top
    start = [rng.randint(0, top) for _ in range(R)]
    start[0] = rng.choice([0, min(3, top - 1)])
    ids = list(range(R * W * M + 2))
    rng.shuffle(ids)
    tables = [[ids.pop() for _ in range(M)] for _ in range(R * W)]
    for row in tables[:W]:  # the first request's first page is shared by its beams
        row[0] = tables[0][0]
    if W > 2:  # and a page of another is missing, or out of the pool
        tables[-1][0], tables[-2][-1] = -1, R * W * M + 2
    parents = _parents(rng, R, W, how)
    layout = "nhpd" if R == 2 else "nphd"
    kp, vp = (_pages((L, R * W * M + 2, P, HK, D), dtype, s, layout) for s in (1, 2))
    for st in (start, None):
        want = [_reorder_ref(parents, t, tables, lengths, st) for t in (kp, vp)]
        beam_reorder(_i(parents), kp, vp, _i(tables), _i(lengths), None if st is None else _i(st))
        assert torch.equal(kp, want[0]) and torch.equal(vp, want[1]), st
    if L == 1:  # one layer's pages
        want = [_reorder_ref(parents, t, tables, lengths, start)[0] for t in (kp, vp)]
        beam_reorder(_i(parents), kp[0], vp[0], _i(tables), _i(lengths), _i(start))
        assert torch.equal(kp[0], want[0]) and torch.equal(vp[0], want[1])


def test_reorder_of_contiguous_caches():
    """HF's [B, HK, S, D] caches as pages of a row each; a length past them counts as theirs, a strided one is taken."""
    from solution.body.paged import beam_reorder

    R, W, HK, S, D = 2, 3, 2, 45, 64
    kc, vc = (torch.randn(R * W, HK, S, D, generator=gen(s)).half().to(DEV) for s in (1, 2))
    parents = torch.tensor([[2, 0, 1], [1, 1, 0]])
    lengths = torch.tensor([[40, 0], [50, 0]], dtype=torch.int32, device=DEV)[:, 0]
    rows = torch.arange(R * W, device=DEV, dtype=torch.int32)[:, None]
    want = []
    for t in (kc, vc):
        x = t.view(R, W, HK, S, D).clone()
        for r, n in enumerate((40, S)):
            x[r, :, :, 4:n] = x[r, parents[r].to(DEV)][:, :, 4:n]
        want.append(x.view(t.shape))
    beam_reorder(_i(parents.tolist()), kc.transpose(1, 2), vc.transpose(1, 2), rows, lengths, _i([4, 4]))
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_reorder_nothing():
    from solution.body.paged import beam_reorder

    kp = _pages((2, 16, 1, 64), torch.float16, 1)
    vp, want = kp.clone(), kp.clone()
    none = torch.zeros(0, 2, dtype=torch.int32, device=DEV)
    beam_reorder(none, kp, vp, none, _i([]))
    beam_reorder(_i([[1, 0]]), kp, vp, _i([[0], [1]]), _i([0]))
    beam_reorder(_i([[1, 0]]), kp, vp, _i([[0], [1]]), _i([9]), _i([9]))
    beam_reorder(_i([[1, 0]]), kp, vp, _i([[0], [1]]), _i([-5]), _i([-9]))
    assert torch.equal(kp, want) and torch.equal(vp, want)


# ----------------------------------------------------------------------------------------
# what is changed behind torch's back
# ----------------------------------------------------------------------------------------
def test_saved_tensors_that_change_are_noticed():
    """A backward pass that saved the pages, tables or lengths does not run over what took their place."""
    from solution.body.paged import beam_reorder, block_tables, paged_store

    dt = torch.bfloat16
    tables, lengths, taken = _i([[0, 1], [2, 3]]), _i([16, 16]), _i([0])

    def refuses(t, change):
        out = (torch.ones(t.shape, device=DEV, dtype=dt, requires_grad=True) * t).sum()
        change()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()

    pages = [_pages((4, 16, 1, 64), dt, i) for i in range(2)]
    k = torch.zeros(1, 1, 64, device=DEV, dtype=dt)
    parents = _i([[1, 0]])
    for t in pages:
        refuses(t, lambda: paged_store(k, k, *pages, _i([3])))
        refuses(t, lambda: beam_reorder(parents, *pages, tables, _i([20])))
    versions = [t._version for t in (tables, lengths, taken)]
    block_tables(tables, lengths, _i([1, 1]), _i([5, 6]), taken, 16, 2)
    assert [t._version for t in (tables, lengths, taken)] == [versions[0] + 1, *versions[1:]]
    block_tables(tables, lengths, _i([1, 1]), _i([5, 6]), taken, 16, 2, update=True)
    assert [t._version for t in (tables, lengths, taken)] == [versions[0] + 2, versions[1] + 1, versions[2] + 1]
