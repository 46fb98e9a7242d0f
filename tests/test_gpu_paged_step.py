"""The serving operators over pages together: a decoder layer on 4-bit weights that answers with beams. The prompts
are packed, stored in pages that block_tables deals out, and forked into beams that share their full pages; then step by
step, eager and as one replayed graph: pages for the new tokens, the layer (few-row NF4 products, RoPE, store, paged
attention with the shared prompt), logits, selection, and the beams' pages following their parents.

Each beam's layer output is compared with a float64 layer over the beam's whole history, within the bound that
test_gpu_decode_step.py derives for this layer; the choices with float64 of the same logits."""

import pytest
import torch

from _util import DEV, gen
from test_gpu_beam_select import _check as _check_choice
from test_gpu_decode_step import D, H, HK, HQ, _check, _half, _layer, _rope64
from test_gpu_decode_step import _reference as _windowed_reference

pytestmark = pytest.mark.gpu

V, PAGE, BEAMS, STEPS = 517, 16, 3, 20
LENS = [37, 16, 5]


def _reference(s, r, monkeypatch):
    """The layer over one sequence in float64, every earlier token seen."""
    import test_gpu_decode_step as module

    monkeypatch.setattr(module, "WINDOW", 1 << 20)
    return _windowed_reference(s, r)


class _Answers:
    """Rows of pages, their lengths and tables, and a step."""

    def __init__(self, s, emb, head, R, W, M, n_pages):
        self.s, self.emb, self.head, self.W = s, emb, head, W
        self.inv = s.inv.float().to(DEV)
        self.kp, self.vp = (torch.full((n_pages, PAGE, HK, D), float("nan"), device=DEV).half() for _ in range(2))
        self.tables = torch.full((R * W, M), -1, dtype=torch.int32, device=DEV)
        order = torch.randperm(n_pages, generator=gen(3)).int()
        self.free, self.taken = order.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        self.lengths = torch.zeros(R * W, dtype=torch.int32, device=DEV)
        self.one = torch.ones(R * W, dtype=torch.int32, device=DEV)
        self.tokens = torch.zeros(R, W, dtype=torch.int32, device=DEV)
        self.scores = torch.full((R, W), float("-inf"), device=DEV)
        self.scores[:, 0] = 0

    def state(self):
        return [self.kp, self.vp, self.tables, self.taken, self.lengths, self.tokens, self.scores]

    def prompts(self, tokens):
        """The first beam of each request takes the prompt; the others share its full pages."""
        from solution import nf4
        from solution.body import norm_rope
        from solution.body.attention import varlen_attention
        from solution.body.paged import beam_reorder, block_tables, paged_store

        lens = torch.tensor([len(t) for t in tokens], dtype=torch.int32, device=DEV)
        first = self.tables[::self.W].clone()
        plan = block_tables(first, torch.zeros_like(lens), lens, self.free, self.taken, PAGE, int(lens.sum()))
        self.taken.copy_(plan.taken)

        def attend(q, k, v):
            q, k = norm_rope.rope(q, k, plan.positions, self.inv)
            paged_store(k, v, self.kp, self.vp, plan.slots)
            return varlen_attention(q, k, v, plan.cu_seqlens, int(lens.max())).reshape(q.shape[0], -1)

        def multi(x, ws, states, biases):
            biases = biases or [None] * len(ws)
            return torch.cat([nf4.nf4_linear(x, w, b, st) for w, st, b in zip(ws, states, biases)], -1)

        out = _half(self.s, self.emb[torch.cat(tokens)], nf4.nf4_linear, multi, attend)
        # the fork: the other beams' rows begin behind the full pages and take a page for the rest, which the first's fills
        self.shared = lens // PAGE * PAGE
        full = (torch.arange(self.tables.shape[1], device=DEV)[None] < (self.shared // PAGE)[:, None])
        for w in range(self.W):
            self.tables[w::self.W] = first if w == 0 else torch.where(full, first, -1)
        row = torch.arange(self.lengths.numel(), device=DEV)
        held, want = self.shared.repeat_interleave(self.W), lens.repeat_interleave(self.W)
        self.lengths.copy_(torch.where(row % self.W == 0, want, held))
        rest = int((want - self.lengths).sum())
        plan = block_tables(self.tables, self.lengths, want - self.lengths, self.free, self.taken, PAGE, rest, update=True)
        beam_reorder(torch.zeros_like(self.tokens), self.kp, self.vp, self.tables, lens, self.shared)
        self.start = lens
        return out

    def choose(self, logits):
        from solution.head import beam_select

        scores, parents, tokens = beam_select(logits, self.scores)
        self.scores.copy_(scores)
        self.tokens.copy_(tokens)
        return scores, parents, tokens

    def step(self):
        """One more token of every beam; returns (layer output, logits, plan's slots, choice)."""
        from solution import nf4
        from solution.body import norm_rope
        from solution.body.paged import beam_reorder, block_tables, paged_attention, paged_store

        W, n = self.W, self.lengths.numel()
        plan = block_tables(self.tables, self.lengths, self.one, self.free, self.taken, PAGE, n, update=True)

        def attend(q, k, v):
            q, k = norm_rope.rope(q, k, plan.positions, self.inv)
            paged_store(k, v, self.kp, self.vp, plan.slots)
            return paged_attention(q, self.kp, self.vp, self.tables, plan.lengths, beams=W,
                                   shared=self.shared).reshape(n, -1)

        r = self.emb.index_select(0, self.tokens.view(-1))
        out = _half(self.s, r, nf4.nf4_matvec, nf4.nf4_matvec_multi, attend)
        logits = (out @ self.head).half().view(-1, W, V)
        before = self.scores.clone()
        choice = self.choose(logits)
        beam_reorder(choice[1], self.kp, self.vp, self.tables, plan.lengths[::W], self.start)
        return out, logits, before, *choice


@torch.no_grad()
def test_answering_with_beams(monkeypatch):
    s, g = _layer(), gen(50)
    emb, head = torch.randn(V, H, generator=g).to(DEV), (0.05 * torch.randn(H, V, generator=g)).to(DEV)
    prompts = [torch.randint(0, V, (n,), generator=g).to(DEV) for n in LENS]
    R, M = len(LENS), 5
    a = _Answers(s, emb, head, R, BEAMS, M, 60)
    out = a.prompts(prompts)
    _check(out, torch.cat([_reference(s, emb[p], monkeypatch) for p in prompts]), "prompts")
    last = torch.tensor(LENS, device=DEV).cumsum(0) - 1
    logits = (out[last] @ head).half()[:, None].expand(R, BEAMS, V)
    before = a.scores.clone()
    choice = a.choose(logits)
    _check_choice(choice, logits, before, BEAMS)
    assert not choice[1].any()  # one beam was alive
    history = [[prompts[r].tolist() for _ in range(BEAMS)] for r in range(R)]

    def follow(parents, tokens):
        for r in range(R):
            history[r] = [history[r][p] + [t] for p, t in zip(parents[r].tolist(), tokens[r].tolist())]

    def check(outs, i):
        out, logits, before, *choice = outs
        ref = [_reference(s, emb[torch.tensor(h, device=DEV)], monkeypatch)[-1] for rows in history for h in rows]
        _check(out, torch.stack(ref), i)
        _check_choice(choice, logits, before, BEAMS)
        follow(*choice[1:])

    follow(*choice[1:])
    moved = 0
    for i in range(STEPS):
        outs = a.step()
        moved += int((outs[4].cpu() != torch.arange(BEAMS)).sum())
        check(outs, i)
    assert moved > STEPS  # beams do change places
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    saved = [t.clone() for t in a.state()]
    with torch.cuda.graph(graph):
        outs = a.step()
    for i in range(6):
        for t, x in zip(a.state(), saved):
            t.copy_(x)
        want = a.step()
        after = [t.clone() for t in a.state()]
        for t, x in zip(a.state(), saved):
            t.copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y)
        for t, x in zip(a.state(), after):
            assert torch.equal(t.nan_to_num(7.0), x.nan_to_num(7.0))
        saved = after
        check(outs, ("replay", i))
    assert a.lengths.view(R, BEAMS)[:, 0].tolist() == [n + STEPS + 6 for n in LENS] and int(a.taken) <= 60
