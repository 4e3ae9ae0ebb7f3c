"""Attention over packed sequences of different lengths, with grouped heads.

Beyond the reference, which takes one length per batch: the sequences' rows follow each
other in one tensor without padding, and a host-side layout of the batch says whose they
are.  GPT.score runs series of different lengths through the layers this way (PackedRows).
"""

import math
import operator
from typing import Sequence

import torch

from diff_gpt import _native


class PackedLayout:
    """Whose rows are whose in a packed batch, laid out once for every layer's call.

    q_lengths: the query rows of each sequence; k_lengths: its key rows (None: the same).
    Query i of a sequence sees its keys 0 .. i + (k_length - q_length): with more keys than
    queries the first keys are cached ones, with fewer the first queries see nothing.
    group: query heads per key head of the tensors the layout is for."""

    __slots__ = ("q_lengths", "k_lengths", "group", "total_q", "total_k", "tiles", "counts", "stream")

    def __init__(self, q_lengths: Sequence[int], k_lengths: Sequence[int] | None = None, group: int = 1,
                 device: torch.device | str = "cuda") -> None:
        _native.require_device_type("PackedLayout", device)
        self.q_lengths = list(map(operator.index, q_lengths))
        self.k_lengths = self.q_lengths if k_lengths is None else list(map(operator.index, k_lengths))
        if len(self.k_lengths) != len(self.q_lengths):
            raise ValueError(f"{len(self.q_lengths)} query lengths, {len(self.k_lengths)} key lengths")
        if any(n < 0 for n in self.q_lengths) or any(n < 0 for n in self.k_lengths):
            raise ValueError("a sequence's length must not be negative")
        if group < 1:
            raise ValueError(f"group must be at least 1, got {group}")
        self.group = operator.index(group)
        self.total_q, self.total_k = sum(self.q_lengths), sum(self.k_lengths)
        tiles, self.counts = _native.packed_plan(self.q_lengths, self.k_lengths, self.group)
        self.tiles = tiles.to(device)
        self.stream = torch._C._cuda_getCurrentRawStream(self.tiles.get_device())  # whose memory the table is


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, layout: PackedLayout,
                     scale: float | None = None) -> torch.Tensor:
    """Causal attention of q (Nq, H, D) over k, v (Nk, Hkv, D), within each sequence of
    ``layout``; query head h reads key head h // (H / Hkv).  scale: 1 / sqrt(D) by default,
    any other acts as its fp32 value, for fp64 tensors too.
    A query that sees no key gets zeros, and so do rows behind the last sequence."""
    y = torch.empty_like(q, memory_format=torch.contiguous_format)
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, q.size(-1)))
    _native.attention_packed_(q, k, v, y, layout, scale)
    if layout.total_q < q.size(0):
        y[layout.total_q :].zero_()
    return y


class PackedRows:
    """A packed batch of whole sequences on its way through the layers: rows (1, total, C),
    each sequence at positions 0 .. length - 1."""

    __slots__ = ("layout", "positions")

    def __init__(self, lengths: Sequence[int], device: torch.device | str) -> None:
        self.layout = PackedLayout(lengths, device=device)
        self.positions = torch.cat([torch.arange(n) for n in self.layout.q_lengths]).to(device)

    def freqs(self, table: torch.Tensor) -> torch.Tensor:
        """The rows' (1, total, 1, D/2, 2) slice of the RoPE table."""
        assert max(self.layout.q_lengths) <= table.shape[0], "a sequence is longer than the RoPE table"
        return table[self.positions].view(1, -1, 1, *table.shape[1:])

    def attend(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               freqs: torch.Tensor) -> torch.Tensor:
        """RoPE, QK-norm and the attention of one layer's (1, total, H, D) projections."""
        q_rot, k_rot = (torch.empty(q.shape, dtype=q.dtype, device=q.device) for _ in range(2))
        _native.ops().rope_qknorm_append(q, k, None, freqs, q_rot, k_rot, None, True)
        return attention_packed(q_rot[0], k_rot[0], v[0], self.layout).unsqueeze(0)
