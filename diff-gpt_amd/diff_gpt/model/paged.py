"""A KV cache in pages: rows of different lengths that share one pool, with grouped heads.

Beyond the reference, whose cache has one length for all rows.  The operators below work on
one layer's (P, S, Hkv, D) views of the pool's pages, S a power of two, and a (B, M) int32
table of page ids: position t of row b lies in page table[b, t // S].  Rows may share pages that
they only read; what is written (append_paged, the pages that evict_paged fills) is one row's.
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
    keys are NaN.  In fp32, fp64 for fp64 rows (an fp32 table's angles too), the norm's eps that
    of the arithmetic's type; everything is rounded once, as it is stored."""
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
    return Evicted(*_native.paged_evict(k_pages, v_pages, table, lengths, weights, keep, recent, to))


class PagedKVCache:
    """The K/V of rows of different lengths, in pages of ``page_size`` positions that come from
    one pool of ``pages`` for all layers; GPT.forward_paged appends to it.

    Each row has a length of its own, the positions it has cached, and the position of its
    next token, which is that length until positions are evicted.  Pages are taken as rows
    grow and given back by truncate, evict and release; a row has at most max_positions
    positions (None: all of the pool's).  weights: keep what attention gives each position, for evict.
    The bookkeeping is on the host; tables and lengths follow on the device, in the order of
    the current stream: use a cache on one stream at a time."""

    __slots__ = ("page_size", "kv", "table", "weights", "lens", "next_pos", "_state", "_pages_of", "_free", "_width",
                 "_stale", "_cut")

    def __init__(self, rows: int, num_heads: int, head_dim: int, num_layers: int, pages: int, page_size: int = 64,
                 max_positions: int | None = None, dtype: torch.dtype = torch.float32,
                 device: torch.device | str = "cuda", weights: bool = False) -> None:
        _native.require_device_type("PagedKVCache", device)
        if rows < 1 or num_heads < 1 or head_dim < 1 or num_layers < 1 or pages < 1:
            raise ValueError("PagedKVCache: rows, heads, head_dim, layers and pages must be positive")
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page_size must be a power of two, got {page_size}")
        most = pages * page_size if max_positions is None else max_positions
        self._width = -(-most // page_size)
        if not 1 <= self._width * page_size <= _native.MAX_POSITIONS:
            raise ValueError(f"PagedKVCache: {most} positions a row, 1 to 2^30")
        self.page_size = page_size
        self.kv = torch.empty((num_layers, 2, pages, num_heads, page_size, head_dim), dtype=dtype, device=device)
        self.table = torch.full((rows, self._width), -1, dtype=torch.int32, device=device)
        self._state = torch.zeros((2, rows), dtype=torch.int32, device=device)  # lens and next_pos
        self.weights: torch.Tensor | None = None
        if weights:
            self.weights = torch.zeros((num_layers, rows, num_heads, self._width * page_size), device=device)
        self.lens, self.next_pos = [0] * rows, [0] * rows
        self._pages_of: list[list[int]] = [[] for _ in range(rows)]
        self._free = list(range(pages - 1, -1, -1))
        self._stale = False  # whether the device's table is behind the host's
        # how many of a row's first positions an eviction chose, each key head its own; behind them
        # they follow one another
        self._cut = [0] * rows

    def layer_pages(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor]:
        """A layer's (pages, page_size, H, D) views of the keys and values."""
        return self.kv[layer_idx, 0].transpose(1, 2), self.kv[layer_idx, 1].transpose(1, 2)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def lengths(self) -> torch.Tensor:
        """The rows' cached positions, on the device."""
        return self._state[0]

    @property
    def positions(self) -> torch.Tensor:
        """The positions of the rows' next tokens, on the device."""
        return self._state[1]

    def ints(self, values: "list[int] | list[list[int]]") -> torch.Tensor:
        """An int32 tensor of them on the cache's device; the host does not wait for the copy."""
        return torch.tensor(values, dtype=torch.int32, pin_memory=True).to(self.table.device, non_blocking=True)

    def _sync(self) -> None:
        """The host's tables and lengths to the device."""
        if self._stale:
            self.table.copy_(self.ints([p + [-1] * (self._width - len(p)) for p in self._pages_of]))
            self._stale = False
        self._state.copy_(self.ints([self.lens, self.next_pos]))

    def reserve(self, counts: list[int]) -> None:
        """Pages for counts[b] more positions of every row b, or, where the pool or a row's
        table has no room for all of them, an error and nothing taken."""
        if len(counts) != len(self.lens) or any(n < 0 for n in counts):
            raise ValueError(f"PagedKVCache: {len(self.lens)} rows, counts {counts}")
        need = [max(0, -(-(a + n) // self.page_size) - len(p)) for a, n, p in zip(self.lens, counts, self._pages_of)]
        for b, (n, p) in enumerate(zip(need, self._pages_of)):
            if len(p) + n > self._width:
                raise RuntimeError(f"PagedKVCache: row {b} has room for {self._width * self.page_size} positions, "
                                   f"{self.lens[b] + counts[b]} needed")
        if sum(need) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(need)} more pages needed, {len(self._free)} of {self.kv.size(2)} free")
        for n, p in zip(need, self._pages_of):
            for _ in range(n):
                p.append(self._free.pop())
                self._stale = True
        if self._stale:
            self._sync()

    def advance(self, counts: list[int], on_device: torch.Tensor | None = None) -> None:
        """The rows' next counts[b] positions, which their pages hold by now, count as cached.
        on_device: the counts there, where the caller has them."""
        if len(counts) != len(self.lens):
            raise ValueError(f"PagedKVCache: {len(self.lens)} rows, counts {counts}")
        for b, n in enumerate(counts):
            if n < 0 or self.lens[b] + n > len(self._pages_of[b]) * self.page_size:
                raise ValueError(f"PagedKVCache: row {b} cannot advance by {n}")
        for b, n in enumerate(counts):
            self.lens[b] += n
            self.next_pos[b] += n
        self._state.add_(self.ints(counts) if on_device is None else on_device)

    def truncate(self, lengths: list[int]) -> None:
        """Row b goes back to its first lengths[b] cached positions, and its next token to where it
        then stands.  A row that was cut goes back no further than to the recent positions that
        the eviction kept (before them each key head has kept others), or to nothing."""
        if len(lengths) != len(self.lens) or any(not 0 <= n <= a for n, a in zip(lengths, self.lens)):
            raise ValueError(f"PagedKVCache: rows of {self.lens} positions cannot go back to {lengths}")
        if list(lengths) == self.lens:
            return
        for b, (n, a, cut) in enumerate(zip(lengths, self.lens, self._cut)):
            if 0 < n < cut and n < a:
                raise ValueError(f"PagedKVCache: row {b} was cut: it goes back to {cut} positions at least, or to none, not to {n}")
        for b, n in enumerate(lengths):
            self.next_pos[b] -= self.lens[b] - n
            self.lens[b] = n
            if n == 0:
                self.next_pos[b] = self._cut[b] = 0
            keep = -(-n // self.page_size)
            if len(self._pages_of[b]) > keep:
                self._free += reversed(self._pages_of[b][keep:])
                del self._pages_of[b][keep:]
                self._stale = True
        self._sync()
        if self.weights is not None:  # later positions start from nothing
            t = torch.arange(self.weights.size(3), dtype=torch.int32, device=self.table.device)
            self.weights.masked_fill_((t >= self.lengths[:, None])[None, :, None], 0.0)

    def release(self, rows: list[int]) -> None:
        """The rows' pages go back to the pool; each of them is empty, at position 0."""
        lengths = list(self.lens)
        for b in rows:
            lengths[b] = 0
        self.truncate(lengths)
        for b in rows:
            self.next_pos[b] = 0
        self._sync()

    def evict(self, keep: int, recent: int, rows: list[int] | None = None) -> list[list[torch.Tensor]]:
        """Cut those of the rows (None: all) that have more than ``keep`` positions to that many a key head, in every layer: the
        ``recent`` last ones and those of the largest weights (evict_paged).  Positions that
        tokens stand at go on from where they were.  The kept positions of each layer are
        returned for each group of rows that was cut at once, (rows, H, keep) int32 (a group
        is as many rows as the pool has room for beside the ones they leave)."""
        if self.weights is None:
            raise RuntimeError("PagedKVCache: evict needs a cache with weights")
        if not 1 <= keep or not 0 <= recent <= keep:
            raise ValueError(f"PagedKVCache: keep {keep} positions, {recent} of them the last ones")
        per = -(-keep // self.page_size)
        long = [b for b, n in enumerate(self.lens) if n > keep and (rows is None or b in rows)]
        out = []
        while long:
            fit = min(len(long), len(self._free) // per)
            if fit == 0:
                raise RuntimeError(f"PagedKVCache: evict needs {per} free pages, {len(self._free)} of {self.kv.size(2)} are")
            some, long = long[:fit], long[fit:]
            to = [[self._free.pop() for _ in range(per)] for _ in some]
            self._sync()
            index, to_dev = self.ints(some).long(), self.ints(to)
            table, lengths = self.table[index], self.lengths[index]
            kept = []
            for layer in range(self.kv.size(0)):
                k_pages, v_pages = self.layer_pages(layer)
                r = evict_paged(k_pages, v_pages, table, lengths, self.weights[layer, index], keep, recent, to_dev)
                row = self.weights.new_zeros((fit, *self.weights.shape[2:]))
                row[..., : r.weights.size(2)] = r.weights
                self.weights[layer, index] = row
                kept.append(r.kept)
            out.append(kept)
            for b, p in zip(some, to):
                self._free += reversed(self._pages_of[b])
                self._pages_of[b] = p
                self._cut[b] = keep - min(recent, self.lens[b] - self._cut[b])
                self.lens[b] = keep
            self._stale = True
            self._sync()
        return out


class PagedRows:
    """A chunk of new tokens of every row of a paged cache on its way through the layers: rows
    (B, N, C), row b's first counts[b] tokens real ones."""

    __slots__ = ("cache", "counts")

    def __init__(self, cache: PagedKVCache, counts: list[int]) -> None:
        self.cache = cache
        self.counts = cache.ints(counts)

    def freqs(self, table: torch.Tensor) -> torch.Tensor:
        """All of the RoPE table: the append finds each token's row of it."""
        return table

    def attend(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               freqs: torch.Tensor) -> torch.Tensor:
        """RoPE, QK-norm, the append and the attention of one layer's (B, N, H, D) projections."""
        cache = self.cache
        if cache.kv.dtype != k.dtype:
            raise TypeError(f"KV cache holds {cache.kv.dtype} but the layer computes in {k.dtype}")
        k_pages, v_pages = cache.layer_pages(layer_idx)
        q_rot = append_paged(q, k, v, freqs, k_pages, v_pages, cache.table, cache.lengths, self.counts, cache.positions)
        weights = None if cache.weights is None else cache.weights[layer_idx]
        longest = max(cache.lens) + q.size(1)
        return attention_paged(q_rot, k_pages, v_pages, cache.table, cache.lengths, self.counts, weights=weights,
                               longest=longest)
