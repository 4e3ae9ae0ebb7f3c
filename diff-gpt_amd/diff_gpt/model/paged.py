"""A KV cache in pages: rows of different lengths that share one pool, with grouped heads.

Beyond the reference, whose cache has one length for all rows.  The operators below work on
one layer's (P, S, Hkv, D) views of the pool's pages, S a power of two, and a (B, M) int32
table of page ids: position t of row b lies in page table[b, t // S].
"""

import math
from typing import NamedTuple

import torch

from diff_gpt import _native


def append_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, freqs: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, qknorm: bool = True) -> torch.Tensor:
    """RoPE and QK-norm of q (B, N, H, D) and k (B, N, Hkv, D); the new keys and the values v go
    into the pages behind row b's lengths[b] positions.  Returns the queries.  Row b has
    counts[b] of the N tokens ((B,) int32; None: all), the others' queries are zeros and their
    keys go nowhere, like those of tokens that the table has no room for.  Token n stands at position
    positions[b] + n of freqs (Tmax, D / 2, 2) (None: lengths[b] + n); outside of it queries and
    keys are NaN.  Everything is rounded once, as it is stored."""
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _native.paged_append_(q, k, v, freqs, out, k_pages, v_pages, table, lengths, counts, positions, qknorm)
    return out


def attention_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                    lengths: torch.Tensor, counts: torch.Tensor | None = None, scale: float | None = None,
                    weights: torch.Tensor | None = None, longest: int | None = None) -> torch.Tensor:
    """Attention of each row's newest tokens q (B, N, H, D), whose keys and values the pages
    already hold behind its lengths[b] positions: token n < counts[b] sees positions
    0 .. lengths[b] + n, the others get zeros.  Query head h reads key head h // (H / Hkv).
    weights (B, Hkv, M * S or more) fp32, when given: the probabilities that each position gets
    are added to it, over the row's tokens and the group's heads.  scale: 1 / sqrt(D) by default,
    any other acts as its fp32 value, for fp64 tensors too.  longest: about how many positions the
    longest row will hold, which only the split of long rows follows (None: M * S)."""
    y = torch.empty_like(q, memory_format=torch.contiguous_format)
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, q.size(-1)))
    _native.paged_attention_(q, k_pages, v_pages, y, scale, table, lengths, counts, weights, longest)
    return y


class Evicted(NamedTuple):
    """Rows cut to their budget: their lengths (B,) int32, their kept positions' weights, zeros
    behind them, and for each place of each key head the position it came from, -1 behind the
    last, (B, Hkv, keep) int32."""

    lengths: torch.Tensor
    weights: torch.Tensor
    kept: torch.Tensor


def evict_paged(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                weights: torch.Tensor, keep: int, recent: int, to: torch.Tensor) -> Evicted:
    """Each row and key head cut to ``keep`` positions: the ``recent`` last ones and, of those
    before, the ones of the largest weights (equal ones: the earlier; NaN: above all), moved in
    their order into the pages that ``to`` (B, pages) int32 names, none of which any row may
    hold.  A row of no more positions moves as it is.  Keys stay turned by the positions they
    had."""
    B, Hkv, S = table.size(0), k_pages.size(2), k_pages.size(1)
    new = weights.new_empty
    r = Evicted(new(B, dtype=torch.int32), new((B, Hkv, to.size(1) * S), dtype=torch.float32),
                new((B, Hkv, max(0, keep)), dtype=torch.int32))
    _native.paged_evict_(k_pages, v_pages, table, lengths, weights, keep, recent, to, r.lengths, r.weights, r.kept)
    return r
