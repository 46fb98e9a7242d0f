"""Beam search's selection over the vocabulary, on the HIP kernels (esep_beam_select): what answering with several
beams does with the head's logits. No reference counterpart (the reference trains)."""

from ..body import _hip
from ..body.attention import _whole

# Most candidates that a call keeps, and beams of a request.
MOST_KEEP = 64


def beam_select(logits, scores, keep=None):
    """The `keep` (None: W) best continuations of each request's W beams: of scores[r, w] + log softmax(logits[r, w])[t]
    over beams w and tokens t the greatest, the greatest first. logits [R, W, V] of fp32, fp16 or bf16 (rows at any
    stride); scores fp32 [R, W], the beams' sums of log probabilities. Returns (scores fp32 [R, keep], parents int32
    [R, keep], tokens int32 [R, keep]); parents are beams of the request (body.paged.beam_reorder's).

    Equal values go to the lowest beam, then the lowest token. A beam whose score is not finite is out (-inf: the
    beams but one at the first step), as is one whose logits hold a NaN, an infinity above 0 or nothing finite; its values
    and those of -inf logits are -inf, and come last, the lowest beam and token first, where fewer than `keep` others
    are left. keep up to 64 and W * V, W up to 64.

    Sums of exponentials are fp32; log softmax, the sum with the score and the comparison of beams are in 64 bits,
    rounded once (to -inf below fp32's range, in their order still). No gradient: logits that record one, traces and
    transforms are refused."""
    if logits.dim() != 3:
        raise _hip.EsepError(f"logits must be [R, W, V], got {list(logits.shape)}")
    R, W, V = logits.shape
    keep = W if keep is None else _whole("keep", keep, 1)
    if keep > min(MOST_KEEP, W * V):
        raise _hip.EsepError(f"keep={keep} of {W} beams over {V} tokens: at most {min(MOST_KEEP, W * V)}")
    _hip.refuse_recorded("beam_select", logits, scores)
    if V > 1 and logits.stride(2) != 1:
        logits = logits.contiguous()
    return _hip.beam_select(logits, scores.contiguous(), keep)
