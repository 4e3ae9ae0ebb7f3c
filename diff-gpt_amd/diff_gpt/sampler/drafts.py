"""Verification of drafted tokens against the target model's probabilities.

Beyond the reference.  A cheaper model proposes a few tokens a row; the target model runs them
all at once and keeps the longest beginning that its own probabilities bear out, then draws
one token more.  What comes out is distributed as if the target model alone had sampled.
Engine.generate_paged speculates this way.
"""

from typing import NamedTuple

import torch

from diff_gpt import _native


class Verified(NamedTuple):
    """Per row of the batch: how many drafts stand; those and the token after them, -1 behind;
    and the target's log probabilities of these tokens (fp32, 0 behind)."""

    accepted: torch.Tensor
    tokens: torch.Tensor
    logprobs: torch.Tensor


def verify_drafts(target: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor | None = None,
                  noise: torch.Tensor | None = None, draft: torch.Tensor | None = None,
                  counts: torch.Tensor | None = None, temperature: float = 1.0) -> Verified:
    """Verified of drafts tokens (B, N) int64, 0 <= N <= 64, counts[b] of them in row b ((B,)
    int32, None: all).  target (B, N + 1, V): the logits behind 0 .. N drafts; draft (B, N, V):
    the logits that the drafts were drawn from (None: each draft was certain, as a greedy
    draft or one that was looked up).  With p and q the softmax of these over the
    temperature, draft x stands iff all before it do and uniforms[b, i] * q(x) < p(x); the token
    after them is the first maximum over V of max(p - q, 0) / noise (p / noise where all
    stand): uniforms (B, N) in [0, 1) and noise (B, V) from Exp(1), fp32.  At temperature 0
    draft x stands iff it is the first maximum of its logits, nothing is drawn, and log
    probabilities are those at temperature 1.  A draft outside the vocabulary does not stand.
    All of it is decided in fp32 with sums in fp64, for fp64 logits in fp64."""
    return Verified(*_native.verify_drafts(target, tokens, uniforms, noise, draft, counts, temperature))
