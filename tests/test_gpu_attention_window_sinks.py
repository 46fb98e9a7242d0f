"""The windowed backward's sink partials on the GPU: far blocks of more than 512 queries, places numbered by the
sequences and by the offsets, nothing read that was not written and nothing written past the workspace. Bounds as
in test_gpu_attention_window.py."""

import pytest
import torch

from _util import DEV
from test_gpu_attention_window import _check, _inputs, _limits, _reference, _run

pytestmark = pytest.mark.gpu

# (lengths, query heads, kv heads, head dim, window, sinks)
CASES = [
    ([6500], 8, 8, 64, 3, 6400),                             # far blocks of 1024 queries, one place
    ([700, 5400, 1, 900], 8, 8, 64, 20, 5300),               # the same among other sequences
    ([40] * 30 + [5200] + [30] * 30, 8, 8, 64, 100, 5000),   # more sequences than offsets: places by offset
    ([1500, 30, 700], 4, 2, 128, 64, 5),
    ([30] * 20 + [1500, 700], 4, 2, 128, 64, 200),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_sink_partials(case):
    from solution.body import _hip

    lengths, HQ, HK, D, window, sinks = CASES[case]
    q, k, v, do, cu = _inputs(lengths, HQ, HK, D, torch.bfloat16, 500 + case)
    ref, tol = _reference(q, k, v, do, lengths, D ** -0.5, window, sinks, *_limits(torch.bfloat16))
    got = _run(q, k, v, do, cu, max(lengths), window=window, sinks=sinks)
    _check(got, ref, tol, CASES[case])

    # a workspace of NaN with a border behind it
    o, lse = torch.empty_like(q), torch.empty((HQ, q.shape[0]), device=DEV)
    low = torch.empty_like(q)
    rest = cu, max(lengths), D ** -0.5, window, sinks
    _hip.attn_win_fwd(q, k, v, o, *rest, lse=lse, o_low=low)
    need = _hip.attn_win_bwd_workspace(q.shape[0], HQ, HK, D, max(lengths), window, sinks, len(lengths))
    ws = torch.full((need + 4096,), float("nan"), device=DEV)
    ws[need:] = 7.0
    grads = [torch.full_like(t, float("nan")) for t in (q, k, v)]
    _hip.attn_win_bwd(q, k, v, o, do, lse, *grads, *rest, o_low=low, workspace=ws)
    for a, b in zip(got, [o, *grads]):
        assert torch.equal(a, b)
    assert (ws[need:] == 7.0).all()
