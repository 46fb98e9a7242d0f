"""Qwen2 with sliding-window layers through the packed decoder, against HF's original forward: hidden
states, loss and every gradient within the tolerances of test_gpu_packed.py, through the kernels and
through torch's operations; what still goes to the original forward."""

import pytest
import torch

from test_gpu_packed import (LENS, VOCAB, _batch, _compare, _config, _counts, _original_forward,
                             _run)

pytestmark = pytest.mark.gpu

WINDOW = 7


def _model(kinds, head_dim=64, window=WINDOW):
    from transformers import Qwen2Config, Qwen2ForCausalLM

    base = _config()
    cfg = Qwen2Config(vocab_size=VOCAB, hidden_size=256, intermediate_size=512,
                      num_hidden_layers=len(kinds), num_attention_heads=4, num_key_value_heads=2,
                      head_dim=head_dim, max_position_embeddings=1024,
                      rms_norm_eps=base.rms_norm_eps, rope_theta=1e6, tie_word_embeddings=True,
                      use_cache=False, use_sliding_window=True, sliding_window=window,
                      max_window_layers=0, layer_types=list(kinds))
    cfg._attn_implementation = "sdpa"
    torch.manual_seed(0)
    return Qwen2ForCausalLM(cfg).cuda().float().train()


MIXED = ("sliding_attention", "full_attention", "sliding_attention")


@pytest.mark.parametrize("kernels", [True, False], ids=["kernels", "torch"])
@pytest.mark.parametrize("left", [False, True], ids=["right_pad", "left_pad"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_window_layers_match_original(left, kernels, dtype):
    from solution.body import _hip, packed, patch

    patch()
    model = _model(MIXED)
    ids, mask, labels = _batch(left)
    with _original_forward():
        ref = _run(model, ids, mask, labels, dtype=dtype)
    with packed.kernels_enabled(kernels), _hip.count_launches() as names:
        new = _run(model, ids, mask, labels, dtype=dtype)
    tol = dict(tol_h=5e-3, tol_loss=1e-3, tol_g=2e-2) if dtype == torch.float16 else \
        dict(tol_h=3e-2, tol_loss=5e-3, tol_g=6e-2)
    _compare(ref, new, mask, **tol)
    c = _counts(names)
    windowed = [names.count(n) for n in ("_attn_win_fwd", "_attn_win_bwd")]
    if kernels:  # two forwards and one backward
        assert windowed == [4, 2] and (c["_attn_fwd"], c["_attn_bwd"]) == (2, 1), names
    else:
        assert not any(c.values()) and windowed == [0, 0]
    # the window matters at these lengths
    for layer in model.model.layers:
        layer.self_attn.sliding_window = None
    with packed.kernels_enabled(False), torch.no_grad():
        model.config.layer_types = ["full_attention"] * 3
        full = model.model(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
    assert (full.float() - new["hidden"]).abs().max() > 0.05 * new["hidden"].abs().max()


def test_rows_with_gaps_take_the_original_forward():
    """A window counts columns: a pad inside a row widens the distance of the tokens around it."""
    from solution.body import _hip, patch

    patch()
    base = _model(MIXED).model
    ids, mask, _ = _batch()
    mask[0, 10:13] = 0
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        with _original_forward():
            want = base(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
        with _hip.count_launches() as names:
            got = base(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
    assert torch.equal(want, got) and not names


def test_a_layer_that_differs_from_the_config_takes_the_original_forward():
    from solution.body import _hip, patch

    patch()
    base = _model(MIXED).model
    base.layers[1].self_attn.sliding_window = 3
    ids, mask, _ = _batch()
    with torch.no_grad(), _hip.count_launches() as names:
        base(input_ids=ids, attention_mask=mask, use_cache=False)
    assert not names


def test_window_past_the_rows_is_full_attention():
    from solution.body import _hip, patch

    patch()
    base = _model(MIXED, window=max(LENS)).model
    ids, mask, _ = _batch()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16), _hip.count_launches() as names:
        base(input_ids=ids, attention_mask=mask, use_cache=False)
    assert names.count("_attn_fwd") == 1 and names.count("_attn_win_fwd") == 2
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        got = base(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
        for layer in base.layers:
            layer.self_attn.sliding_window = None
        base.config.layer_types = ["full_attention"] * 3
        want = base(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
    assert torch.equal(got, want)
