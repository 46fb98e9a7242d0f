"""A pool that runs out: what rows hold then, and how they go on by the recipe in solution/body/paged.py. Each token's keys
are its row and position, so that what the pages hold for a row can be read back through its table."""

import random

import pytest
import torch

from _util import DEV

pytestmark = pytest.mark.gpu

D = 8


def _i(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class _Pool:
    def __init__(self, B, M, page, F, seed):
        self.B, self.M, self.P, self.F = B, M, page, F
        self.rng = random.Random(seed)
        ids = list(range(F + 3))
        self.rng.shuffle(ids)
        self.free, self.taken = _i(ids[:F]), _i([0])
        self.tables = torch.full((B, M), -1, dtype=torch.int32, device=DEV)
        self.lengths = _i([0] * B)
        self.kp = torch.full((F + 3, page, 1, D), -1.0, device=DEV, dtype=torch.float16)
        self.vp = self.kp.clone()

    def add(self, new, total=None):
        """Places new[b] tokens for each row and stores them; returns the slots."""
        from solution.body.paged import block_tables, paged_store

        total = sum(new) if total is None else total
        before = self.lengths.tolist()
        plan = block_tables(self.tables, self.lengths, _i(new), self.free, self.taken, self.P, total, update=True)
        k = torch.zeros(total, 1, D, device=DEV, dtype=torch.float16)
        rows = [b for b, n in enumerate(new) for _ in range(n)][:total]
        k[:len(rows), 0, 0] = torch.tensor(rows, device=DEV).half()
        k[:len(rows), 0, 1] = plan.positions[:len(rows)].half()
        paged_store(k, -k, self.kp, self.vp, plan.slots)
        want = [t for b, n in enumerate(new) for t in range(before[b], before[b] + n)][:total]
        assert plan.positions.tolist() == want
        return plan.slots.tolist()

    def held(self, b):
        """The row's entries, and the first missing page (None: none is)."""
        n = -(-self.lengths[b].item() // self.P)
        row = self.tables[b, :n].tolist()
        return row, next((j for j, page in enumerate(row) if page < 0), None)

    def give_back(self, numbers):
        used = min(self.taken.item(), self.F)
        n = len(numbers)
        self.free[used - n:used] = _i(numbers)
        self.taken[0] = used - n

    def done(self, b):
        self.give_back([page for page in self.held(b)[0] if page >= 0])
        self.lengths[b] = 0

    def set_back(self):
        """Rows that went short, to the tokens that they hold."""
        short = []
        for b in range(self.B):
            row, j = self.held(b)
            if j is not None:
                self.give_back([page for page in row[j:] if page >= 0])
                self.lengths[b] = j * self.P
                short.append(b)
        return short

    def check(self):
        """Every row's tokens are where its table says, each page is one row's or free."""
        owned = []
        for b in range(self.B):
            row, j = self.held(b)
            assert j is None, (b, row)
            owned += row
            n = self.lengths[b].item()
            if n == 0:
                continue
            for pages, sign in ((self.kp, 1), (self.vp, -1)):
                got = pages[torch.tensor(row, device=DEV)].reshape(-1, D)[:n].float() * sign
                assert (got[:, 0] == b).all() and (got[:, 1] == torch.arange(n, device=DEV)).all(), b
        taken = self.taken.item()
        assert 0 <= taken <= self.F and len(owned) == taken
        everything = owned + self.free[taken:].tolist()
        assert len(set(everything)) == len(everything) == self.F


@pytest.mark.parametrize("B,M,page,F,most", [(3, 8, 16, 9, 40), (5, 40, 4, 30, 30), (1, 6, 16, 2, 30),
                                             (300, 4, 16, 310, 9), (4, 30, 7, 25, 60)])
def test_rows_go_on_after_a_shortage(B, M, page, F, most):
    """Rounds of growth until pages are missing; then some rows are done, the short ones set back, and their tokens given anew."""
    p, shortages = _Pool(B, M, page, F, B), 0
    for _ in range(12):
        room = [M * page - n for n in p.lengths.tolist()]
        p.add([min(r, p.rng.randint(0, most)) for r in room])
        if p.taken.item() > F:
            shortages += 1
            short = p.set_back()
            assert short
            p.check()
            for b in p.rng.sample(range(B), (B + 1) // 2):
                p.done(b)
            p.check()
            # the ones that went short go on in a page of their own, up to what the pool has left
            left, new = F - p.taken.item(), [0] * B
            for b in short:
                n = min(page + 1, M * page - p.lengths[b].item())
                need = -(-(p.lengths[b].item() + n) // page) - -(-p.lengths[b].item() // page)
                if need <= left:
                    new[b], left = n, left - need
            assert all(s >= 0 for s in p.add(new))
        p.check()
    assert shortages >= 2


def test_a_row_left_short():
    """Without a set-back: the missing page's later tokens get none either, whatever has come back; the next page does. Nothing
    but the row's own tokens is ever seen."""
    from solution.body.paged import paged_attention

    P = 16
    p = _Pool(2, 4, P, 3, 0)
    assert all(s >= 0 for s in p.add([40, 0]))           # all three pages
    assert p.add([0, 10]) == [-1] * 10                   # none for the second row
    assert p.taken.item() == 4 and p.tables[1, 0].item() == -1
    p.done(0)
    assert p.taken.item() == 0
    slots = p.add([0, 10])                               # six in the missing page, four in the next
    assert slots[:6] == [-1] * 6 and all(s >= 0 for s in slots[6:]) and p.taken.item() == 1
    assert p.tables[1, :2].tolist() == [-1, p.free[0].item()]
    # the four tokens are all that attention sees: equal scores, values -1 and -position
    kp, vp = (torch.full((6, P, 1, 64), float("nan"), device=DEV, dtype=torch.float16) for _ in range(2))
    page = p.tables[1, 1].item()
    kp[page, :4], vp[page, :4] = 1.0, torch.arange(4, device=DEV).half()[:, None, None]
    q = torch.ones(1, 1, 64, device=DEV, dtype=torch.float16)
    o = paged_attention(q, kp, vp, p.tables[1:], p.lengths[1:])
    assert torch.equal(o, torch.full_like(o, 1.5))


def test_the_same_call_again_with_more_pages():
    """update=False: what found too few pages is called again once the list has more."""
    from solution.body.paged import block_tables

    P, tables, lengths, new, taken = 16, torch.full((3, 3), -1, dtype=torch.int32, device=DEV), _i([0, 0, 0]), _i([20, 3, 33]), _i([0])
    short = block_tables(tables, lengths, new, _i([7, 5]), taken, P, 56)
    assert short.taken.item() == 6 and tables.tolist() == [[7, 5, -1], [-1] * 3, [-1] * 3]
    plan = block_tables(tables, lengths, new, _i([7, 5, 1, 0, 9, 4, 2]), taken, P, 56)
    assert plan.taken.item() == 6 and tables.tolist() == [[7, 5, -1], [1, -1, -1], [0, 9, 4]]
    assert min(plan.slots.tolist()) >= 0 and plan.lengths.tolist() == [20, 3, 33]
