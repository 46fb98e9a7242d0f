"""The windowed backward's sink partials without a GPU: their size follows the sequences there are, and what the
backward refuses is refused before the forward runs."""

import pytest
import torch

from solution.body import _hip, attention

# (T, query heads, kv heads, D, max_seqlen, window, sinks)
LONG = (131072, 32, 8, 128, 131072, 16, 4096)


def _rows(sizes, n_seq):
    """Floats beside delta and the split's partials."""
    T, HQ, HK, D, longest, window, _ = sizes
    w = _hip.attn_win_bwd_workspace
    return w(*sizes, n_seq) - w(T, HQ, HK, D, longest, window, 0, n_seq)


def test_one_sequence_takes_one_place():
    # near: one place of 4096 rows; far: 4096 blocks of 8 heads x 32 tiles of sink rows make 16 chunks of 8192
    # queries, and the place; K and V, one block to a kv head
    assert _rows(LONG, 1) == (1 + 17) * 2 * 8 * 4096 * 128
    assert _rows(LONG, 29) == (29 + 45) * 2 * 8 * 4096 * 128
    most = 131072 // 528 + 1
    assert _rows(LONG, most) == _rows(LONG, 10 * most) == _rows(LONG, None) == (2 * most + 16) * 2 * 8 * 4096 * 128


def test_few_sinks_keep_blocks_of_512_queries():
    # 65536 tokens, 4 kv heads of one tile of sink rows: 512 blocks, short of two rounds, so two to a kv head
    sizes = (65536, 4, 4, 64, 65536, 1024, 64)
    assert _rows(sizes, 3) == (3 + 128 + 3) * 2 * 4 * 64 * 64


def test_partials_no_card_holds_are_refused():
    w = _hip.attn_win_bwd_workspace
    with pytest.raises(_hip.EsepError, match="sinks"):
        w(262144, 64, 32, 128, 262144, 16, 1024, 300)  # 2^24 rows and more
    assert w(262144, 64, 32, 128, 262144, 16, 1024, 200) > 0
    with pytest.raises(_hip.EsepError, match="sinks"):
        w(1 << 30, 4, 2, 64, 1 << 30, 1, 1 << 20, 1)


def test_the_forward_refuses_what_the_backward_would(monkeypatch):
    ran = []
    monkeypatch.setattr(_hip, "attn_win_fwd", lambda *a, **kw: ran.append(1))
    T, n_seq, sinks = 32768, 64, 16384
    q = torch.zeros(T, 8, 64, dtype=torch.float16)
    cu = torch.arange(n_seq + 1, dtype=torch.int32) * (T // n_seq)
    args = (cu, T)
    with pytest.raises(_hip.EsepError, match="sinks"):
        attention.varlen_attention(q.requires_grad_(), q, q, *args, window=1, sinks=sinks)
    assert not ran
    attention.varlen_attention(q, q, q, *args, window=1, sinks=sinks // 2)  # half the rows
    q = q.detach()
    attention.varlen_attention(q, q, q, *args, window=1, sinks=sinks)  # no gradient is asked for
    assert len(ran) == 2
