"""Log probabilities of given tokens, with the entropy and the most likely alternatives of
every row, in one pass over the logits (diff_gpt.py:348-352 gathers the first from a whole
log_softmax).
"""

from typing import NamedTuple

import torch

from diff_gpt import _native


class TokenLogprobs(NamedTuple):
    """Per row: the given token's log probability and the row's entropy in nats, and the
    ``top`` most likely ids in descending order (equal logits by ascending id) with their
    log probabilities.  fp32 (fp64 for fp64 logits); ids int64."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """TokenLogprobs of logits (..., V) and ids (...) int64, with 0 <= top <= min(V, 64).
    An id outside the vocabulary gives NaN; so does a row with NaN, +inf, or -inf alone."""
    V = logits.size(-1)
    lead = logits.shape[:-1]
    if ids.shape != lead:
        raise ValueError(f"token_logprobs: ids {tuple(ids.shape)} for logits {tuple(logits.shape)}")
    if not 0 <= top <= min(V, _native.MAX_TOP):
        raise ValueError(f"token_logprobs: top {top} outside 0 .. min(V, {_native.MAX_TOP})")
    if len(lead) == 1 and logits.stride(1) == 1 and ids.is_contiguous():
        return TokenLogprobs(*_native.new_token_logprobs(logits, ids, top))
    x = logits.reshape(-1, V)
    if V > 1 and x.stride(1) != 1:
        x = x.contiguous()
    lp, entropy, top_lp, top_ids = _native.new_token_logprobs(x, ids.reshape(x.size(0)).contiguous(), top)
    return TokenLogprobs(lp.view(lead), entropy.view(lead), top_lp.view(*lead, top), top_ids.view(*lead, top))
