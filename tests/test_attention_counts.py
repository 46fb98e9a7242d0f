"""window and sinks that are no whole numbers, without a GPU: refused with the entries' own error."""

import pytest
import torch

from solution.body import _hip, attention

NO_COUNTS = [float("nan"), float("inf"), [1], "3", "three", 1.5, True, object(), torch.tensor([1, 2])]


def _varlen(**kw):
    q, cu = torch.zeros(5, 2, 64).half(), torch.tensor([0, 5], dtype=torch.int32)
    return attention.varlen_attention(q, q, q, cu, 5, **kw)


def _cache(**kw):
    q = torch.zeros(1, 1, 2, 64).half()
    return attention.cache_attention(q, q, q, torch.ones(1, dtype=torch.int32), **kw)


@pytest.mark.parametrize("call", [_varlen, _cache])
@pytest.mark.parametrize("value", NO_COUNTS, ids=[str(i) for i in range(len(NO_COUNTS))])
def test_refused(call, value):
    with pytest.raises(_hip.EsepError, match="window must be a whole number"):
        call(window=value)
    with pytest.raises(_hip.EsepError, match="sinks must be a whole number"):
        call(window=2, sinks=value)


@pytest.mark.parametrize("call", [_varlen, _cache])
def test_no_sinks_is_a_count(call):
    with pytest.raises(_hip.EsepError, match="sinks must be a whole number"):
        call(window=2, sinks=None)
