"""Attention of a few tokens per row over the row's cache: a tree of candidate tokens, or
a decode step's one, with grouped heads and rows of different lengths.

Beyond the reference.  The tokens' keys and values lie in the cache behind the row's
cached positions; each token sees all of those, itself and its ancestors in the tree.
GPT.forward_tree runs candidate continuations through the layers this way (TreeRows).
"""

import math
import operator
from typing import Sequence

import torch

from diff_gpt import _native
from diff_gpt.model.kv_cache import KVCache

# tokens of a tree: one bit each of a 64-bit mask
MAX_TREE = 64


def _check_parents(parents: Sequence[int]) -> list[int]:
    parents = list(map(operator.index, parents))
    if not 1 <= len(parents) <= MAX_TREE:
        raise ValueError(f"a tree has 1 to {MAX_TREE} tokens, got {len(parents)}")
    for n, p in enumerate(parents):
        if not -1 <= p < n:
            raise ValueError(f"token {n}'s parent must be an earlier token or -1 (the cached row), got {p}")
    return parents


def tree_masks(parents: Sequence[int], device: torch.device | str = "cuda") -> torch.Tensor:
    """The (N,) int64 masks of a tree given by each token's parent, an earlier token or -1
    for the cached row: bit m of mask n is set where token m is token n or above it."""
    masks: list[int] = []
    for n, p in enumerate(_check_parents(parents)):
        masks.append((1 << n) | (masks[p] if p >= 0 else 0))
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64).to(device)


def tree_depths(parents: Sequence[int]) -> list[int]:
    """How many tokens lie above each token: its position behind the cached row."""
    depths: list[int] = []
    for p in _check_parents(parents):
        depths.append(depths[p] + 1 if p >= 0 else 0)
    return depths


def attention_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: int | torch.Tensor,
                   masks: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of q (B, N, H, D), N <= 64, over the (B, Tcap, Hkv, D) cache views: row b's
    ``lengths[b]`` cached positions (one int for all rows, or a (B,) int32 tensor, taken as
    0 .. Tcap - N) and the N tokens behind them, of which token n sees those in its mask
    ((N,) or (B, N) int64, tree_masks; None: the tokens before it and itself).  Query head h
    reads key head h // (H / Hkv).  scale: 1 / sqrt(D) by default, any other acts as its fp32
    value, for fp64 tensors too."""
    y = torch.empty_like(q, memory_format=torch.contiguous_format)
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, q.size(-1)))
    _native.attention_tree_(q, k_cache, v_cache, y, scale, lengths, masks)
    return y


class TreeRows:
    """A tree of tokens behind every row of a cache on its way through the layers: rows
    (B, N, C), token n at the position of its depth, its keys and values in the cache's
    n-th place behind the cached positions."""

    __slots__ = ("cache", "depths", "masks", "start")

    def __init__(self, parents: Sequence[int], cache: KVCache, device: torch.device | str) -> None:
        self.cache = cache
        self.depths = tree_depths(parents)
        self.masks = tree_masks(parents, device)
        self.start = cache.get_pos()

    def freqs(self, table: torch.Tensor) -> torch.Tensor:
        """The tokens' (1, N, 1, D/2, 2) slice of the RoPE table."""
        positions = [self.start + d for d in self.depths]
        assert max(positions) < table.shape[0], "the tree is deeper than the RoPE table reaches"
        index = torch.tensor(positions, dtype=torch.int64).to(table.device)
        return table[index].view(1, -1, 1, *table.shape[1:])

    def attend(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               freqs: torch.Tensor) -> torch.Tensor:
        """RoPE, QK-norm, the cache append and the attention of one layer's (B, N, H, D)
        projections."""
        cache = self.cache
        t0, t1 = cache.ensure_window(q.size(1), k.dtype, k.device)
        pages = cache._tensor()
        if pages.dtype != k.dtype:
            raise TypeError(f"KV cache holds {pages.dtype} but the layer computes in {k.dtype}")
        k_pages, v_pages = (pages[layer_idx, i].transpose(1, 2) for i in range(2))
        q_rot = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _native.ops().rope_qknorm_append(q, k, v, freqs, q_rot, k_pages[:, t0:t1], v_pages[:, t0:t1], True)
        return attention_tree(q_rot, k_pages, v_pages, t0, self.masks)
