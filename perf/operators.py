"""The measured work of three sets of operators: windowed attention with sinks (training), attention of the
newest tokens over a cache (serving), and products of a few rows with 4-bit weights (serving).

A case names a `kind` and its sizes. `listed()` holds one fixed set, `draw()` gives more of the same
ranges, `prepare()` builds the inputs on the GPU, `run()` is one pass (in plain torch operations in 32
bits, or with `own` through this framework's entry points), `work()` the bytes and operations that the
pass cannot do without, `exact()` the same outputs in float64.
"""

import math
import random
import sys
import types
from pathlib import Path

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# The NF4 data type (normal-float 4-bit quantiles).
NF4 = [-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635,
       -0.18477343022823334, -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725,
       0.24611230194568634, 0.33791524171829224, 0.44070982933044434, 0.5626170039176941,
       0.7229568362236023, 1.0]


# ----------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------
def listed():
    return [
        # one short prompt of a fine-tuning step in a sliding-window layer: latency
        dict(name="window_short", kind="window", tokens=200, seqs=1, hq=12, hk=2, dim=128, window=64,
             sinks=4, dtype="fp16"),
        # one training batch, 8 rows of up to 1024 tokens, a plain sliding window
        dict(name="window_rows", kind="window", tokens=5933, seqs=8, hq=12, hk=2, dim=128, window=256,
             sinks=0, dtype="bf16"),
        # a small model with 64-wide heads and longer rows
        dict(name="window_dim64", kind="window", tokens=12011, seqs=9, hq=14, hk=2, dim=64, window=512,
             sinks=16, dtype="bf16"),
        # one long document whose first tokens stay visible
        dict(name="window_long", kind="window", tokens=32768, seqs=1, hq=12, hk=2, dim=128, window=4096,
             sinks=4, dtype="bf16"),
        # a large packed batch of a 3584-wide model
        dict(name="window_packed", kind="window", tokens=65536, seqs=29, hq=28, hk=4, dim=128,
             window=1024, sinks=64, dtype="fp16"),
        # one answer being decoded over a short prompt: latency
        dict(name="cache_one", kind="cache", rows=1, new=1, longest=700, space=1024, hq=12, hk=2, dim=128,
             window=0, sinks=0, layout="bhsd", dtype="fp16"),
        # a batch of answers over ragged prompts
        dict(name="cache_batch", kind="cache", rows=32, new=1, longest=8192, space=8320, hq=28, hk=4,
             dim=128, window=0, sinks=0, layout="bhsd", dtype="bf16"),
        # long answers through a window, the first tokens visible
        dict(name="cache_window", kind="cache", rows=8, new=1, longest=32768, space=32768, hq=12, hk=2,
             dim=128, window=4096, sinks=4, layout="bhsd", dtype="bf16"),
        # a few new tokens at once (a short follow-up), 64-wide heads, token-major cache
        dict(name="cache_chunk", kind="cache", rows=4, new=16, longest=4001, space=4096, hq=14, hk=2,
             dim=64, window=0, sinks=0, layout="bshd", dtype="fp16"),
        # q / k / v of one token from 4-bit weights: latency
        dict(name="nf4_qkv", kind="nf4", rows=1, n_in=1536, outs="1536,256,256", bias=True, dtype="fp16"),
        # gate and up of one token of a 3584-wide model
        dict(name="nf4_gate_up", kind="nf4", rows=1, n_in=3584, outs="18944,18944", bias=False,
             dtype="fp16"),
        # down projection of seven answers decoded side by side
        dict(name="nf4_down", kind="nf4", rows=7, n_in=8960, outs="1536", bias=False, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (query heads, kv heads, head dim)
_HEADS = [(14, 2, 64), (16, 2, 128), (12, 2, 128), (28, 4, 128), (8, 8, 64), (12, 12, 128)]


def draw(rng):
    kind = rng.choice(["window", "cache", "nf4"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "window":
        hq, hk, dim = rng.choice(_HEADS)
        tokens = _log_int(rng, 100, 32768)
        # rows of up to about 8192 tokens
        return dict(kind=kind, tokens=tokens, seqs=max(-(-tokens // 5000), rng.randint(1, 16)), hq=hq,
                    hk=hk, dim=dim, window=_log_int(rng, 16, 4096),
                    sinks=rng.choice([0, 0, 1, 4, 16, 64, rng.randint(1, 200)]), dtype=dtype)
    if kind == "cache":
        hq, hk, dim = rng.choice(_HEADS)
        longest = _log_int(rng, 16, 32768)
        rows = _log_int(rng, 1, max(2, min(64, 262144 // longest)))
        window = rng.choice([0, _log_int(rng, 16, 8192)])
        return dict(kind=kind, rows=rows, new=rng.choice([1, 1, 1, rng.randint(2, 32)]),
                    longest=longest, space=longest + rng.randint(0, 300), hq=hq, hk=hk, dim=dim,
                    window=window, sinks=rng.choice([0, 4, rng.randint(1, 100)]) if window else 0,
                    layout=rng.choice(["bhsd", "bshd"]), dtype=dtype)
    n_in, outs, bias = rng.choice([(896, "896,128,128", True), (896, "4864,4864", False),
                                   (4864, "896", False), (1536, "1536,256,256", True),
                                   (1536, "1536", False), (1536, "8960,8960", False),
                                   (8960, "1536", False), (3584, "3584,512,512", True),
                                   (3584, "18944,18944", False), (18944, "3584", False)])
    return dict(kind=kind, rows=rng.choice([1, 1, rng.randint(2, 16)]), n_in=n_in, outs=outs, bias=bias,
                dtype=dtype)


def _lengths(total, n, seed=5):
    """n ragged lengths of 1 and more that sum to `total`, the same for the same arguments."""
    rng = random.Random(total * 1009 + n * 31 + seed)
    n = min(n, total)
    w = [rng.uniform(0.4, 1.6) for _ in range(n)]
    lens = [max(1, int(total * x / sum(w))) for x in w]
    i = 0
    while sum(lens) != total:
        step = 1 if sum(lens) < total else -1
        if lens[i % n] + step >= 1:
            lens[i % n] += step
        i += 1
    return lens


def _cache_lengths(case):
    """Filled lengths of a cache's rows: the first row is the longest, the others between a quarter of it
    and all of it, none shorter than its new tokens."""
    rng = random.Random(case["longest"] * 1009 + case["rows"] * 31 + case["new"])
    top = max(case["longest"], case["new"])
    low = max(case["new"], top // 4)
    return [top] + [rng.randint(low, top) for _ in range(case["rows"] - 1)]


def _space(case):
    return max(case["space"], case["new"])


# ----------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------
class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        t = torch.randn(*shape, device="cuda", generator=self.g)
        return (t if scale == 1.0 else t * scale).to(dtype)

    def byte(self, n):
        return torch.randint(0, 256, (n,), device="cuda", generator=self.g, dtype=torch.uint8)

    def uniform(self, n):
        return torch.rand(n, device="cuda", generator=self.g)


def _quant_state(d, n_out, n_in):
    """A packed NF4 weight and its quant state: scales of a weight of deviation about n_in ** -0.5 (block
    maxima near 2.5 deviations), stored in 8 bits around their mean."""
    nb = n_out * n_in // 64
    sd = n_in ** -0.5
    i = torch.arange(128, device="cuda", dtype=torch.float32)
    pos = (i / 127.0) ** 2
    second = types.SimpleNamespace(absmax=(0.5 + 0.3 * d.uniform(-(-nb // 256))) * sd,
                                   code=torch.cat([-pos.flip(0), pos]), blocksize=256)
    state = types.SimpleNamespace(quant_type="nf4", blocksize=64, nested=True, shape=(n_out, n_in),
                                  absmax=d.byte(nb), code=torch.tensor(NF4, device="cuda"),
                                  offset=torch.tensor(2.5 * sd, device="cuda"), state2=second)
    return d.byte(n_out * n_in // 2).view(-1, 1), state


def prepare(case, seed):
    d, dt = _Draw(seed), DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] == "window":
        T, hq, hk, dim = (case[k] for k in ("tokens", "hq", "hk", "dim"))
        lens = _lengths(T, case["seqs"])
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s.update(q=d.normal(T, hq, dim, dtype=dt).requires_grad_(own),
                 k=d.normal(T, hk, dim, dtype=dt).requires_grad_(own),
                 v=d.normal(T, hk, dim, dtype=dt).requires_grad_(own), do=d.normal(T, hq, dim, dtype=dt),
                 lens=lens, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    elif case["kind"] == "cache":
        B, n, hq, hk, dim = (case[k] for k in ("rows", "new", "hq", "hk", "dim"))
        S = _space(case)
        lens = _cache_lengths(case)
        s.update(q=d.normal(B, n, hq, dim, dtype=dt), lens=lens,
                 lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
        for name in ("k", "v"):  # rows behind a row's length hold what was there before
            if case["layout"] == "bhsd":
                s[name] = d.normal(B, hk, S, dim, dtype=dt).transpose(1, 2)
            else:
                s[name] = d.normal(B, S, hk, dim, dtype=dt)
    else:
        outs = [int(n) for n in case["outs"].split(",")]
        s.update(x=d.normal(case["rows"], case["n_in"], dtype=dt),
                 weights=[_quant_state(d, n, case["n_in"]) for n in outs],
                 biases=[d.normal(n, dtype=dt) if case["bias"] else None for n in outs])
    if own:
        _entries()  # the framework is imported before the first pass
    return s


# ----------------------------------------------------------------------------------------
# one pass through the framework
# ----------------------------------------------------------------------------------------
def _entries():
    root = str(Path(__file__).resolve().parents[1] / "esep-soup-kernels_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from solution import nf4
    from solution.body import attention

    return attention, nf4


def _own_window(s):
    attention, _ = _entries()
    c = s["case"]
    o = attention.varlen_attention(s["q"], s["k"], s["v"], s["cu"], max(s["lens"]), window=c["window"],
                                   sinks=c["sinks"])
    return o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])


def _own_cache(s):
    attention, _ = _entries()
    c = s["case"]
    return attention.cache_attention(s["q"], s["k"], s["v"], s["lengths"], window=c["window"] or None,
                                     sinks=c["sinks"])


def _own_nf4(s):
    _, nf4 = _entries()
    if len(s["weights"]) == 1:
        packed, state = s["weights"][0]
        return nf4.nf4_matvec(s["x"], packed, s["biases"][0], state)
    return nf4.nf4_matvec_multi(s["x"], [p for p, _ in s["weights"]], [q for _, q in s["weights"]],
                                s["biases"] if s["case"]["bias"] else None)


# ----------------------------------------------------------------------------------------
# one pass in plain torch operations, in 32 bits
# ----------------------------------------------------------------------------------------
def _softmax(scores, seen):
    scores = scores.masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _seen(pos_q, pos_k, window, sinks):
    i, j = pos_q[:, None], pos_k[None, :]
    seen = j <= i
    if window:
        seen = seen & ((i - j < window) | (j < sinks))
    return seen


def _plain_window(s):
    c = s["case"]
    group, scale, dt = c["hq"] // c["hk"], c["dim"] ** -0.5, DTYPES[c["dtype"]]
    q, k, v, do = (s[n].detach().float().transpose(0, 1) for n in ("q", "k", "v", "do"))
    o, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    t0 = 0
    for n in s["lens"]:
        at = slice(t0, t0 + n)
        t0 += n
        pos = torch.arange(n, device=q.device)
        seen = _seen(pos, pos, c["window"], c["sinks"])
        step = max(1, min(group, (1 << 29) // (n * n)))  # heads at a time: scores of up to 2 GiB
        for kh in range(c["hk"]):
            ks, vs = k[kh, at], v[kh, at]
            for h in range(kh * group, (kh + 1) * group, step):
                hs = slice(h, min(h + step, (kh + 1) * group))
                qs, ds = q[hs, at], do[hs, at]
                p = _softmax(scale * torch.matmul(qs, ks.t()), seen)
                out = torch.matmul(p, vs)
                dv[kh, at] += torch.matmul(p.transpose(1, 2), ds).sum(0)
                grad = p * (torch.matmul(ds, vs.t()) - (ds * out).sum(-1, keepdim=True))
                o[hs, at], dq[hs, at] = out, scale * torch.matmul(grad, ks)
                dk[kh, at] += scale * torch.matmul(grad.transpose(1, 2), qs).sum(0)
    return tuple(t.transpose(0, 1).to(dt) for t in (o, dq, dk, dv))


def _plain_cache(s):
    c = s["case"]
    group, n = c["hq"] // c["hk"], c["new"]
    out = torch.empty_like(s["q"])
    for b, length in enumerate(s["lens"]):
        q = s["q"][b].float().view(n, c["hk"], group, c["dim"]).permute(1, 2, 0, 3)  # [hk, group, n, dim]
        k, v = (s[name][b, :length].float().transpose(0, 1) for name in ("k", "v"))  # [hk, length, dim]
        seen = _seen(torch.arange(length - n, length, device=q.device),
                     torch.arange(length, device=q.device), c["window"], c["sinks"])
        scores = torch.matmul(q.reshape(c["hk"], group * n, c["dim"]), k.transpose(1, 2))
        p = _softmax(scores.view(c["hk"], group, n, length) * c["dim"] ** -0.5, seen)
        o = torch.matmul(p.view(c["hk"], group * n, length), v).view(c["hk"], group, n, c["dim"])
        out[b] = o.permute(2, 0, 1, 3).reshape(n, c["hq"], c["dim"]).to(out.dtype)
    return out


def _plain_nf4(s):
    x = s["x"].float()
    parts = []
    for (packed, st), bias in zip(s["weights"], s["biases"]):
        flat = packed.view(-1).int()
        value = st.code[torch.stack((flat >> 4, flat & 15), 1).view(-1, 64)]
        nb = st.absmax.numel()
        second = st.state2.absmax.repeat_interleave(256)[:nb]
        scale = st.state2.code[st.absmax.int()] * second + st.offset
        y = torch.matmul(x, (value * scale[:, None]).view(*st.shape).t())
        parts.append(y if bias is None else y + bias.float())
    return torch.cat(parts, -1).to(s["x"].dtype)


_PLAIN = dict(window=_plain_window, cache=_plain_cache, nf4=_plain_nf4)
_OWN = dict(window=_own_window, cache=_own_cache, nf4=_own_nf4)


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


def work(case):
    if case["kind"] == "window":
        T, hq, hk, dim = (case[k] for k in ("tokens", "hq", "hk", "dim"))
        pairs = sum(_visible(i, case["window"], case["sinks"]) for n in _lengths(T, case["seqs"])
                    for i in range(n))
        # q, do read and o, dq written; k, v read and dk, dv written
        return dict(bytes=2 * T * dim * (4 * hq + 4 * hk), flops=14 * dim * hq * pairs)
    if case["kind"] == "cache":
        B, n, hq, hk, dim = (case[k] for k in ("rows", "new", "hq", "hk", "dim"))
        keys = pairs = 0
        for length in _cache_lengths(case):
            first = max(0, length - n - case["window"] + 1) if case["window"] else 0
            keys += length - first + min(first, case["sinks"])
            pairs += sum(_visible(i, case["window"], case["sinks"]) for i in range(length - n, length))
        return dict(bytes=2 * dim * (2 * hk * keys + 2 * B * n * hq) + 4 * B,
                    flops=4 * dim * hq * pairs)
    outs = [int(n) for n in case["outs"].split(",")]
    K, M = case["n_in"], case["rows"]
    nb = [n * K // 64 for n in outs]
    tables = sum(b + 4 * -(-b // 256) + 4 * (256 + 16 + 1) for b in nb)
    return dict(bytes=sum(n * K // 2 for n in outs) + tables + 2 * M * (K + sum(outs))
                + (2 * sum(outs) if case["bias"] else 0), flops=2 * M * K * sum(outs))


# ----------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------
def _exact_window(s):
    """Query blocks against the keys that they can see, gradients by autograd."""
    c = s["case"]
    q, k, v, do = (s[n].detach().double() for n in ("q", "k", "v", "do"))
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    group, W, S = c["hq"] // c["hk"], c["window"], c["sinks"]
    t0 = 0
    for n in s["lens"]:
        for kh in range(c["hk"]):
            at = (slice(t0, t0 + n), slice(kh * group, (kh + 1) * group))
            qs = q[at].permute(1, 0, 2).clone().requires_grad_()
            ks, vs = (t[t0:t0 + n, kh].clone().requires_grad_() for t in (k, v))
            ds = do[at].permute(1, 0, 2)
            for a in range(0, n, 1024):
                b = min(n, a + 1024)
                first = max(0, a - W + 1)
                idx = torch.cat([torch.arange(min(S, first)), torch.arange(first, b)]).to(q.device)
                i = torch.arange(a, b, device=q.device).view(-1, 1)
                hidden = (idx > i) | ((i - idx >= W) & (idx >= S))
                sc = torch.einsum("gid,jd->gij", qs[:, a:b], ks[idx]) / math.sqrt(c["dim"])
                lse = torch.logsumexp(torch.where(hidden, torch.full_like(sc, -math.inf), sc), -1)
                p = torch.where(hidden, torch.zeros_like(sc), torch.exp(sc - lse[..., None]))
                ob = torch.einsum("gij,jd->gid", p, vs[idx])
                gq, gk, gv = torch.autograd.grad(ob, (qs, ks, vs), ds[:, a:b])
                o[at][a:b] = ob.detach().permute(1, 0, 2)
                dq[at] += gq.permute(1, 0, 2)
                dk[t0:t0 + n, kh] += gk
                dv[t0:t0 + n, kh] += gv
        t0 += n
    return o, dq, dk, dv


def _exact_cache(s):
    c = s["case"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    for b, length in enumerate(s["lens"]):
        for t in range(c["new"]):
            pos = length - c["new"] + t
            first = max(0, pos - c["window"] + 1) if c["window"] else 0
            idx = torch.cat([torch.arange(min(c["sinks"], first)), torch.arange(first, pos + 1)])
            idx = idx.to(q.device)
            for kh in range(c["hk"]):
                hs = slice(kh * c["hq"] // c["hk"], (kh + 1) * c["hq"] // c["hk"])
                sc = q[b, t, hs] @ s["k"][b, idx, kh].double().t() / math.sqrt(c["dim"])
                out[b, t, hs] = torch.softmax(sc, -1) @ s["v"][b, idx, kh].double()
    return out


def _exact_nf4(s):
    x, parts = s["x"].double(), []
    for (packed, st), bias in zip(s["weights"], s["biases"]):
        n, k = st.shape
        second = st.state2
        group = torch.arange(st.absmax.numel(), device=x.device) // second.blocksize
        scale = second.code.double()[st.absmax.long()] * second.absmax.double()[group] + st.offset.double()
        y = torch.zeros(x.shape[0], n, dtype=torch.float64, device=x.device)
        codes = packed.view(n, k // 2).long()
        for parity, codes_p in ((0, codes // 16), (1, codes % 16)):  # even columns are the high halves
            w = st.code.double()[codes_p] * scale.view(n, k // 64).repeat_interleave(32, 1)
            y += x[:, parity::2] @ w.t()
        parts.append(y if bias is None else y + bias.double())
    return torch.cat(parts, -1)


def exact(case, seed):
    s = prepare(case, seed)
    return dict(window=_exact_window, cache=_exact_cache, nf4=_exact_nf4)[case["kind"]](s)
