"""The measured work of answering over a paged key-value cache: block tables and slots from the rows' lengths, the
store of new keys and values, attention of the newest tokens over the pages, and beam search's selection over the
vocabulary with the reordering of the beams' states.

A case names a `kind` and its sizes. `listed()` holds one fixed set, `draw()` gives more of the same ranges,
`prepare()` builds the inputs on the GPU, `run()` is one pass (in plain torch operations, or with `own` through
this framework's entry points), `work()` the bytes and operations that the pass cannot do without, `exact()` the
same outputs from the definitions in float64. Passes can be repeated on one state: the pages and tables that a pass
writes take the same values again.
"""

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ----------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------
def listed():
    return [
        # one more token for each of a batch of answers, 16 tokens to a page: latency, once a step
        dict(name="tables_step", kind="tables", rows=64, step=True, longest=8192, page=16),
        # a queue of prompts admitted at once
        dict(name="tables_prompts", kind="tables", rows=300, step=False, longest=2047, page=32),
        # the new token of 32 answers, once a layer and step: latency
        dict(name="store_step", kind="store", tokens=32, padded=3, hk=2, dim=128, page=16, layout="nphd",
             dtype="fp16"),
        # a packed batch of prompts of a 3584-wide model
        dict(name="store_prompts", kind="store", tokens=32771, padded=0, hk=4, dim=128, page=64, layout="nhpd",
             dtype="bf16"),
        # one answer being decoded over a short prompt: latency
        dict(name="paged_one", kind="paged", requests=1, beams=1, new=1, longest=700, grown=0, hq=12, hk=2, dim=128,
             page=16, window=0, sinks=0, layout="nphd", dtype="fp16"),
        # a batch of answers over ragged prompts
        dict(name="paged_batch", kind="paged", requests=48, beams=1, new=1, longest=8192, grown=0, hq=28, hk=4,
             dim=128, page=64, window=0, sinks=0, layout="nphd", dtype="bf16"),
        # short follow-ups through a window with sinks, 64-wide heads, odd lengths
        dict(name="paged_window", kind="paged", requests=7, beams=1, new=5, longest=9001, grown=0, hq=14, hk=2,
             dim=64, page=32, window=1500, sinks=5, layout="nhpd", dtype="fp16"),
        # beam search over long prompts: the beams of a request share its prompt's pages
        dict(name="paged_beams", kind="paged", requests=8, beams=4, new=1, longest=8000, grown=130, hq=28, hk=4,
             dim=128, page=16, window=0, sinks=0, layout="nphd", dtype="bf16"),
        # the next tokens of one request's four beams: latency
        dict(name="select_step", kind="select", requests=1, beams=4, vocab=151936, keep=8, first=False,
             dtype="bf16"),
        # of 24 requests' five, at their first step (one beam alive each), unrounded logits
        dict(name="select_batch", kind="select", requests=24, beams=5, vocab=151936, keep=5, first=True,
             dtype="fp32"),
        # one request's four beams of up to 61 new tokens, all layers at once: latency
        dict(name="reorder_step", kind="reorder", layers=28, requests=1, beams=4, start=303, grown=61, hk=2, dim=128,
             page=16, dtype="fp16"),
        # twelve requests' eight beams of long answers
        dict(name="reorder_batch", kind="reorder", layers=28, requests=12, beams=8, start=1000, grown=391, hk=4,
             dim=128, page=64, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (query heads, kv heads, head dim)
_HEADS = [(14, 2, 64), (16, 2, 128), (12, 2, 128), (28, 4, 128), (8, 8, 64), (12, 12, 128)]
_PAGES = [16, 32, 64, 128]
_VOCABS = [1000, 32000, 50001, 128000, 151936]


def draw(rng):
    kind = rng.choice(["tables", "store", "paged", "paged", "select", "reorder"])
    hq, hk, dim = rng.choice(_HEADS)
    page, dtype = rng.choice(_PAGES), rng.choice(["fp16", "bf16"])
    layout = rng.choice(["nphd", "nhpd"])
    if kind == "tables":
        rows = _log_int(rng, 1, 512)
        return dict(kind=kind, rows=rows, step=rng.random() < 0.5,
                    longest=_log_int(rng, 8, max(16, min(32768, 524288 // rows))), page=page)
    if kind == "store":
        tokens = _log_int(rng, 1, 32768)
        return dict(kind=kind, tokens=tokens, padded=rng.choice([0, rng.randint(0, tokens // 2)]), hk=hk, dim=dim,
                    page=page, layout=layout, dtype=dtype)
    if kind == "paged":
        longest = _log_int(rng, 16, 32768)
        rows = _log_int(rng, 1, max(2, min(64, 262144 // longest)))
        beams = rng.choice([1, 1, rng.randint(2, 8)])
        window = rng.choice([0, _log_int(rng, 16, 8192)]) if beams == 1 else 0
        return dict(kind=kind, requests=max(1, rows // beams), beams=beams,
                    new=rng.choice([1, 1, 1, rng.randint(2, 24)]), longest=longest,
                    grown=_log_int(rng, 24, 500) if beams > 1 else 0, hq=hq, hk=hk, dim=dim, page=page,
                    window=window, sinks=rng.choice([0, 4, rng.randint(1, 100)]) if window else 0, layout=layout,
                    dtype=dtype)
    if kind == "select":
        vocab, beams = rng.choice(_VOCABS), _log_int(rng, 1, 16)
        return dict(kind=kind, requests=_log_int(rng, 1, max(1, min(64, 18000000 // (vocab * beams)))), beams=beams,
                    vocab=vocab, keep=beams * rng.choice([1, 2]), first=rng.random() < 0.25,
                    dtype=rng.choice(["fp16", "bf16", "fp32"]))
    beams = rng.randint(2, 8)
    return dict(kind=kind, layers=rng.choice([1, 24, 28]), requests=_log_int(rng, 1, 12), beams=beams,
                start=_log_int(rng, 1, 2000), grown=_log_int(rng, 1, 390), hk=min(hk, 4), dim=dim, page=page,
                dtype=dtype)


def _tables_lengths(case):
    """(tokens in each row before, new ones): a step adds one token to rows of all lengths; prompts find empty
    rows, and every seventh a row that goes on."""
    rng = random.Random(case["rows"] * 1009 + case["longest"])
    B, top = case["rows"], case["longest"]
    if case["step"]:
        return [rng.randint(max(0, top // 8 - 1), top - 1) for _ in range(B)], [1] * B
    old = [rng.randint(1, top) if b % 7 == 3 else 0 for b in range(B)]
    return old, [rng.randint(max(1, top // 8), top) for _ in range(B)]


def _paged_lengths(case):
    """(lengths of the rows, tokens that the beams of each request share): the first request's row is the longest,
    the others between a quarter of it and all of it; beams of a request have grown alike."""
    rng = random.Random(case["longest"] * 1009 + case["requests"] * 31 + case["new"])
    new, W, page = case["new"], case["beams"], case["page"]
    top = max(case["longest"], new)
    low = max(new, top // 4)
    prompts = [top] + [rng.randint(low, top) for _ in range(case["requests"] - 1)]
    lens = [p + (max(case["grown"], new) if W > 1 else 0) for p in prompts for _ in range(W)]
    return lens, [p // page * page if W > 1 else 0 for p in prompts]


def _parents(case):
    """Each request's surviving beams stay where they are; the places of the others are taken by copies of them."""
    rng = random.Random(case["requests"] * 1009 + case["beams"] * 31 + case["grown"])
    W, out = case["beams"], []
    for _ in range(case["requests"]):
        alive = sorted(rng.sample(range(W), rng.randint(1, max(1, W - 1))))
        out.append([w if w in alive else rng.choice(alive) for w in range(W)])
    return out


# ----------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------
class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))
        self.host = random.Random(int(seed))

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        t = torch.randn(*shape, device="cuda", generator=self.g, dtype=dtype)
        return t if scale == 1.0 else t.mul_(scale)

    def order(self, n):
        ids = list(range(n))
        self.host.shuffle(ids)
        return ids


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(d, case, n, dtype, lead=()):
    """Pages that hold what was there before."""
    shape = (n, case["page"], case["hk"], case["dim"])
    if case.get("layout") == "nhpd":
        return d.normal(*lead, n, case["hk"], case["page"], case["dim"], dtype=dtype).transpose(-2, -3)
    return d.normal(*lead, *shape, dtype=dtype)


def _prepare_tables(case, d):
    P = case["page"]
    old, new = _tables_lengths(case)
    M = -(-2 * case["longest"] // P)
    held = [-(-n // P) for n in old]
    need = sum(-(-(a + b) // P) for a, b in zip(old, new))
    ids = d.order(need + 100)
    tables = [ids[sum(held[:b]):sum(held[:b + 1])] + [-1] * (M - held[b]) for b in range(case["rows"])]
    free = [-1] * 7 + ids[sum(held):]  # seven entries are taken already
    return dict(tables=_ints(tables), lengths=_ints(old), new=_ints(new), free=_ints(free), taken=_ints([7]),
                total=sum(new), page=P)


def _prepare_store(case, d):
    T, P, dt = case["tokens"], case["page"], DTYPES[case["dtype"]]
    n = -(-T // P) + 4
    slots = d.order(n * P)[:T]
    for i in d.order(T)[:case["padded"]]:
        slots[i] = -1
    qkv = d.normal(T, 4 * case["hk"], case["dim"], dtype=dt)  # k and v as slices of a fused projection
    return dict(k=qkv[:, 2 * case["hk"]:3 * case["hk"]], v=qkv[:, 3 * case["hk"]:], k_pages=_pages(d, case, n, dt),
                v_pages=_pages(d, case, n, dt), slots=_ints(slots))


def _prepare_paged(case, d):
    P, dt, W = case["page"], DTYPES[case["dtype"]], case["beams"]
    lens, shared = _paged_lengths(case)
    ids = d.order(sum(-(-n // P) for n in lens) + 3)
    n_pages, tables, width = len(ids), [], max(-(-n // P) for n in lens) + 1
    for b, n in enumerate(lens):
        row = tables[b // W * W][:shared[b // W] // P] if b % W else []
        while len(row) < -(-n // P):
            row.append(ids.pop())
        tables.append(row + [-1] * (width - len(row)))
    return dict(q=d.normal(len(lens), case["new"], case["hq"], case["dim"], dtype=dt),
                k_pages=_pages(d, case, n_pages, dt), v_pages=_pages(d, case, n_pages, dt), tables=_ints(tables),
                lengths=_ints(lens), shared=_ints(shared), lens=lens)


def _prepare_select(case, d):
    R, W, V = case["requests"], case["beams"], case["vocab"]
    logits = d.normal(R, W, V, scale=2.5).to(DTYPES[case["dtype"]])
    logits[..., V - V // 500:] = -math.inf  # entries that no token has
    scores = -5.0 * d.normal(R, W).abs()
    if case["first"]:
        scores[:, 0], scores[:, 1:] = 0.0, -math.inf
    return dict(logits=logits, scores=scores)


def _prepare_reorder(case, d):
    P, W, dt = case["page"], case["beams"], DTYPES[case["dtype"]]
    lens = [case["start"] + max(1, case["grown"] - 3 * r) for r in range(case["requests"])]
    first = case["start"] // P  # the page that the beams' own tokens begin in is each beam's own
    own_pages = [-(-n // P) - first for n in lens]
    ids = d.order(case["requests"] * first + W * sum(own_pages))
    n_pages, tables = len(ids), []
    width = max(-(-n // P) for n in lens)
    for r, n in enumerate(own_pages):
        prompt = [ids.pop() for _ in range(first)]
        for _ in range(W):
            row = prompt + [ids.pop() for _ in range(n)]
            tables.append(row + [-1] * (width - len(row)))
    return dict(k_pages=_pages(d, case, n_pages, dt, (case["layers"],)),
                v_pages=_pages(d, case, n_pages, dt, (case["layers"],)), tables=_ints(tables), lens=lens,
                lengths=_ints(lens), start=_ints([case["start"]] * len(lens)), parents=_ints(_parents(case)))


_PREPARE = dict(tables=_prepare_tables, store=_prepare_store, paged=_prepare_paged, select=_prepare_select,
                reorder=_prepare_reorder)


def prepare(case, seed):
    s = _PREPARE[case["kind"]](case, _Draw(seed))
    s["case"] = case
    if own:
        s["paged"], s["head"] = _entries()  # as a program imports them
    return s


# ----------------------------------------------------------------------------------------
# one pass through the framework
# ----------------------------------------------------------------------------------------
def _entries():
    root = str(Path(__file__).resolve().parents[1] / "esep-soup-kernels_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from solution import head
    from solution.body import paged

    return paged, head


def _own_tables(s):
    p = s["paged"].block_tables(s["tables"], s["lengths"], s["new"], s["free"], s["taken"], s["page"], s["total"])
    return p.slots, p.positions, p.cu_seqlens, p.lengths, p.taken, s["tables"]


def _own_store(s):
    s["paged"].paged_store(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"])
    return s["k_pages"], s["v_pages"]


def _own_paged(s):
    c = s["case"]
    return s["paged"].paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"],
                                      window=c["window"] or None, sinks=c["sinks"], beams=c["beams"],
                                      shared=s["shared"] if c["beams"] > 1 else None)


def _own_select(s):
    return s["head"].beam_select(s["logits"], s["scores"], s["case"]["keep"])


def _own_reorder(s):
    s["paged"].beam_reorder(s["parents"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"], s["start"])
    return s["k_pages"], s["v_pages"]


# ----------------------------------------------------------------------------------------
# one pass in plain torch operations
# ----------------------------------------------------------------------------------------
def _plain_tables(s):
    P, total, tables, free = s["page"], s["total"], s["tables"], s["free"].long()
    B, M = tables.shape
    before, new = s["lengths"].long(), s["new"].long()
    after = (before + new).clamp(max=M * P)
    held, need = (before + P - 1) // P, (after + P - 1) // P
    take = need - held
    first = s["taken"] + take.cumsum(0) - take
    col = torch.arange(M, device="cuda")[None]
    at = first[:, None] + col - held[:, None]
    page = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    tables.copy_(torch.where((col >= held[:, None]) & (col < need[:, None]), page, tables))
    ends = new.cumsum(0)
    i = torch.arange(total, device="cuda")
    row = torch.repeat_interleave(torch.arange(B, device="cuda"), new, output_size=total)
    pos = before[row] + i - (ends - new)[row]
    page = tables[row, (pos // P).clamp(max=M - 1)].long()
    slots = torch.where((pos < M * P) & (page >= 0), page * P + pos % P, -1)
    cu = torch.cat([ends.new_zeros(1), ends])
    return (slots.int(), pos.int(), cu.int(), after.int(), (s["taken"] + take.sum()).int(), tables)


def _plain_store(s):
    P = s["k_pages"].shape[1]
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    for new, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        pages[slots // P, slots % P] = new[live]
    return s["k_pages"], s["v_pages"]


def _seen(pos_q, pos_k, window, sinks):
    i, j = pos_q[:, None], pos_k[None, :]
    seen = j <= i
    if window:
        seen = seen & ((i - j < window) | (j < sinks))
    return seen


def _plain_paged(s):
    c = s["case"]
    group, n, P = c["hq"] // c["hk"], c["new"], c["page"]
    out = torch.empty_like(s["q"])
    for b, length in enumerate(s["lens"]):
        ids = s["tables"][b, :-(-length // P)].long()
        q = s["q"][b].float().view(n, c["hk"], group, c["dim"]).permute(1, 2, 0, 3)  # [hk, group, n, dim]
        k, v = (s[x][ids].reshape(-1, c["hk"], c["dim"])[:length].float().transpose(0, 1).contiguous()
                for x in ("k_pages", "v_pages"))  # [hk, length, dim]
        seen = _seen(torch.arange(length - n, length, device=q.device), torch.arange(length, device=q.device),
                     c["window"], c["sinks"])
        scores = torch.matmul(q.reshape(c["hk"], group * n, c["dim"]), k.transpose(1, 2).contiguous())
        scores = (scores.view(c["hk"], group, n, length) * c["dim"] ** -0.5).masked_fill(~seen, -math.inf)
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        o = torch.matmul(p.view(c["hk"], group * n, length), v).view(c["hk"], group, n, c["dim"])
        out[b] = o.permute(2, 0, 1, 3).reshape(n, c["hq"], c["dim"]).to(out.dtype)
    return out


def _plain_select(s):
    """The candidates' values in 64 bits: two of them can lie closer than 32 tell apart."""
    R, W, V = s["logits"].shape
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    lse = top.double() + torch.log(torch.exp(x - top).sum(-1, keepdim=True, dtype=torch.float64))
    value = (s["scores"].double()[..., None] + (x.double() - lse)).view(R, W * V)
    value = torch.where(torch.isnan(value), -math.inf, value)
    value, at = torch.sort(value, dim=-1, descending=True, stable=True)
    keep = s["case"]["keep"]
    at = at[:, :keep]
    return value[:, :keep].float(), (at // V).int(), (at % V).int()


def _plain_reorder(s):
    c = s["case"]
    P, W = c["page"], c["beams"]
    tables, parents = s["tables"].long(), s["parents"].long()
    for r, length in enumerate(s["lens"]):
        t = torch.arange(c["start"], length, device="cuda")
        own_rows = tables[r * W:(r + 1) * W]
        to = own_rows[:, t // P]
        for pages in (s["k_pages"], s["v_pages"]):
            pages[:, to, t % P] = pages[:, to[parents[r]], t % P]
    return s["k_pages"], s["v_pages"]


_PLAIN = dict(tables=_plain_tables, store=_plain_store, paged=_plain_paged, select=_plain_select,
              reorder=_plain_reorder)
_OWN = dict(tables=_own_tables, store=_own_store, paged=_own_paged, select=_own_select, reorder=_own_reorder)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ----------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------
def _visible(pos, window, sinks):
    """Keys that the query at this position sees."""
    if not window or pos < window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def _work_tables(c):
    old, new = _tables_lengths(c)
    taken = sum(-(-(a + b) // c["page"]) + -a // c["page"] for a, b in zip(old, new))
    # lengths and new read, new lengths and offsets written; a page's number read and written; the open page of a
    # row that goes on read; a slot and a position written for every token
    going = sum(1 for a in old if a % c["page"])
    return dict(bytes=16 * c["rows"] + 8 * taken + 4 * going + 8 * sum(new) + 12, flops=0)


def _work_paged(c):
    lens, shared = _paged_lengths(c)
    W, n, keys, pairs, entries = c["beams"], c["new"], 0, 0, 0
    for b, length in enumerate(lens):
        skip = shared[b // W] if b % W else 0  # counted with the request's first beam
        first = max(0, length - n - c["window"] + 1) if c["window"] else 0
        keys += length - skip - first + min(first, c["sinks"])
        entries += -(-(length - skip - first + min(first, c["sinks"])) // c["page"])
        pairs += sum(_visible(i, c["window"], c["sinks"]) for i in range(length - n, length))
    return dict(bytes=2 * c["dim"] * (2 * c["hk"] * keys + 2 * len(lens) * n * c["hq"]) + 4 * (entries + len(lens)),
                flops=4 * c["dim"] * c["hq"] * pairs)


def _work_reorder(c):
    moved = 0
    for r, row in enumerate(_parents(c)):
        grown = max(1, c["grown"] - 3 * r)
        to = [w for w, p in enumerate(row) if p != w]
        moved += grown * (len(to) + len({row[w] for w in to}))
    W, R = c["beams"], c["requests"]
    return dict(bytes=moved * c["layers"] * 2 * c["hk"] * c["dim"] * 2 + 4 * R * (W + 2), flops=0)


def work(case):
    c = case
    if c["kind"] == "tables":
        return _work_tables(c)
    if c["kind"] == "store":
        live = c["tokens"] - c["padded"]
        return dict(bytes=4 * c["tokens"] + live * 2 * c["hk"] * c["dim"] * 2 * 2, flops=0)
    if c["kind"] == "paged":
        return _work_paged(c)
    if c["kind"] == "select":
        R, W, V = c["requests"], c["beams"], c["vocab"]
        size = 4 if c["dtype"] == "fp32" else 2
        read = (1 if c["first"] else W) * R * V  # a beam that is out cannot be chosen
        return dict(bytes=read * size + 4 * R * W + 12 * R * c["keep"], flops=4 * read)
    return _work_reorder(c)


# ----------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ----------------------------------------------------------------------------------------
def _exact_tables(s):
    P = s["page"]
    tables, old, new, free = (s[x].tolist() for x in ("tables", "lengths", "new", "free"))
    taken, slots, positions, cu, lengths = s["taken"].item(), [], [], [0], []
    for b, row in enumerate(tables):
        for t in range(old[b], old[b] + new[b]):
            if t % P == 0 and t // P < len(row):
                row[t // P] = free[taken] if taken < len(free) else -1
                taken += 1
            page = row[t // P] if t // P < len(row) else -1
            slots.append(page * P + t % P if page >= 0 else -1)
            positions.append(t)
        cu.append(cu[-1] + new[b])
        lengths.append(min(old[b] + new[b], P * len(row)))
    return tuple(_ints(x) for x in (slots, positions, cu, lengths, [taken], tables))


def _exact_store(s):
    out = []
    at = [(i, slot) for i, slot in enumerate(s["slots"].tolist()) if slot >= 0]
    token, slot = (torch.tensor(x, device="cuda") for x in zip(*at)) if at else (None, None)
    for new, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        flat = pages.contiguous().flatten(0, 1).clone()
        if at:
            flat.index_copy_(0, slot, new.index_select(0, token))
        out.append(flat.view(pages.shape))
    return tuple(out)


def _exact_paged(s):
    c = s["case"]
    q, P = s["q"].double(), c["page"]
    out = torch.zeros_like(q)
    for b, length in enumerate(s["lens"]):
        for t in range(c["new"]):
            pos = length - c["new"] + t
            first = max(0, pos - c["window"] + 1) if c["window"] else 0
            idx = torch.cat([torch.arange(min(c["sinks"], first)), torch.arange(first, pos + 1)]).to(q.device)
            page = s["tables"][b].long()[idx // P]
            K, V = (s[x][page, idx % P].double() for x in ("k_pages", "v_pages"))
            for kh in range(c["hk"]):
                hs = slice(kh * c["hq"] // c["hk"], (kh + 1) * c["hq"] // c["hk"])
                sc = q[b, t, hs] @ K[:, kh].t().contiguous() / math.sqrt(c["dim"])
                out[b, t, hs] = torch.softmax(sc, -1) @ V[:, kh].contiguous()
    return out


def _exact_select(s):
    R, W, V = s["logits"].shape
    keep, out = s["case"]["keep"], ([], [], [])
    for r in range(R):
        value = torch.log_softmax(s["logits"][r].double(), -1) + s["scores"][r].double()[:, None]
        value = value.cpu().numpy().reshape(-1)
        value = np.where(np.isnan(value), -np.inf, value)
        border = np.partition(value, W * V - keep)[W * V - keep]
        above, ties = np.nonzero(value > border)[0], np.nonzero(value == border)[0]
        at = np.concatenate([above, ties[:keep - len(above)]])
        at = at[np.lexsort((at, -value[at]))]
        for x, y in zip(out, (value[at], at // V, at % V)):
            x.append(y)
    scores, parents, tokens = (torch.from_numpy(np.stack(x)).cuda() for x in out)
    return scores, parents.int(), tokens.int()


def _exact_reorder(s):
    """Runs of tokens within a page, beam by beam, out of the old pages."""
    c = s["case"]
    P, W, tables = c["page"], c["beams"], s["tables"].tolist()
    out = [s["k_pages"].clone(), s["v_pages"].clone()]
    for r, row in enumerate(s["parents"].tolist()):
        for w, parent in enumerate(row):
            t = c["start"]
            while t < s["lens"][r]:
                end = min(s["lens"][r], (t // P + 1) * P)
                run_ = slice(t % P, t % P + end - t)
                for new, old in zip(out, (s["k_pages"], s["v_pages"])):
                    new[:, tables[r * W + w][t // P], run_] = old[:, tables[r * W + parent][t // P], run_]
                t = end
    return tuple(out)


def exact(case, seed):
    s = prepare(case, seed)
    return dict(tables=_exact_tables, store=_exact_store, paged=_exact_paged, select=_exact_select,
                reorder=_exact_reorder)[case["kind"]](s)
