"""KV-cache generation engine (src/diff_gpt/model/engine.py:11-169).

One batch-1 prefill of the prompt, the prompt's KV cache shared by
``num_samples`` rows (KVCache.prefill: stored once, read once per decode
step), then one single-token decode forward per step for all rows together.
Per step a token column is either sampled (``sampler`` or softmax +
multinomial with the seeded device generator) or, when
``force_schedule[step]`` is an int, forced for every row.  Each yielded
column comes with a mask column: 1 = sampled, 0 = forced.

Beyond the reference: ``generate_multi`` / ``generate_multi_batch`` decode
several prompts of one length at once -- one batched prefill, each prompt's
cache shared by its ``num_samples`` rows, one captured decode step for all
rows -- with a schedule that may differ per prompt or per row.
``score_continuations`` gives the log probabilities of candidate continuations
of a prompt, run as trees of tokens behind its cache.
``generate_paged`` decodes prompts of different lengths together over a paged
cache, with a smaller model that drafts tokens for it, and with a bound on the
positions that a row keeps.
"""

import gc
from collections import deque
from typing import Generator, Sequence

import numpy as np
import torch

from diff_gpt import _native
from diff_gpt.model.gpt import GPT, BaseGPT, plain_gpt
from diff_gpt.model.kv_cache import KVCache
from diff_gpt.model.paged import PagedKVCache
from diff_gpt.model.token_logprobs import token_logprobs
from diff_gpt.model.tree import MAX_TREE
from diff_gpt.sampler.drafts import verify_drafts
from diff_gpt.sampler.sampler import Sampler
from diff_gpt.sampler.temperature import draw_one


class RowState:
    """Per-row generation state: the tokens so far and a queue of tokens that
    must be emitted next regardless of sampling (engine.py:11-20)."""

    __slots__ = (
        "current_tokens",
        "forced_tokens",
    )

    def __init__(self, current_tokens: list[int] | None = None) -> None:
        self.current_tokens = current_tokens or list()
        self.forced_tokens = deque()


class _DecodeGraph:
    """GPT.forward over one new token per row, captured once as a HIP graph and
    replayed for every decode step.

    The cache carries a device copy of its position (KVCache.pos_dev); the
    attention layers then launch the position-reading kernels
    (dg_rope_qknorm_append_at, dg_decode_attention_at) and the model hands
    them the whole RoPE table, so nothing in the captured launches depends on
    the step.  The graph ends by advancing pos_dev; step() advances the host
    copy.  Inputs go through a static id buffer, the logits come back in a
    static buffer that the next replay overwrites."""

    __slots__ = ("cache", "ids", "graph", "logits")

    def __init__(self, model: BaseGPT, cache: KVCache, n_rows: int, device: torch.device) -> None:
        self.cache = cache
        self.ids = torch.zeros((n_rows, 1), dtype=torch.long, device=device)
        pos0 = cache.pos
        cache.pos_dev = torch.full((1,), pos0, dtype=torch.int32, device=device)
        try:
            # warm-up outside the capture (library handles, allocator); it
            # appends the K/V of a zero token at pos0, which the first replay
            # overwrites
            side = torch.cuda.Stream(device=device)
            side.wait_stream(torch.cuda.current_stream(device))
            with torch.cuda.stream(side):
                model.forward(self.ids, kv_cache=cache)
            torch.cuda.current_stream(device).wait_stream(side)
            cache.pos = pos0
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                if plain_gpt(model):  # the last launch may advance the position
                    logits, _ = model.forward(self.ids, kv_cache=cache, _advance=True)
                else:
                    logits, _ = model.forward(self.ids, kv_cache=cache)
                    cache.pos_dev.add_(1)
                self.logits = logits[:, -1, :]
            cache.pos = pos0
        except BaseException:
            cache.pos = pos0
            cache.pos_dev = None
            raise

    def step(self, ids: torch.Tensor) -> torch.Tensor:
        self.ids.copy_(ids)
        self.graph.replay()
        self.cache.pos += 1
        return self.logits

    def rewind(self) -> None:
        """Start over at the cache's (refilled) host position."""
        self.cache.pos_dev.fill_(self.cache.pos)

    def close(self) -> None:
        self.cache.pos_dev = None


# A captured decode step (and the cache it writes) is kept for the next call
# when the cache is at most this large.
_KEEP_GRAPH_BYTES = 1 << 30

# kinds of a decode step's column
_SAMPLE, _FORCE_ALL, _MIXED = 0, 1, 2


class _Schedule:
    """A force schedule resolved for ``rows`` rows over ``steps`` steps: per
    step, whether every row samples, every row is forced, or some are; the
    forced tokens as a (steps, rows) device tensor (negative: sample) when
    they differ between rows, else one token per step."""

    __slots__ = ("kinds", "shared", "per_row")

    def __init__(self, steps: int) -> None:
        self.kinds = [_SAMPLE] * steps
        self.shared: list[int | None] | None = None
        self.per_row: torch.Tensor | None = None

    @staticmethod
    def shared_list(schedule: Sequence[int | None], steps: int) -> "_Schedule":
        s = _Schedule(steps)
        s.shared = list(schedule[:steps])
        s.kinds = [_SAMPLE if t is None else _FORCE_ALL for t in s.shared]
        return s

    @staticmethod
    def table(table: np.ndarray, steps: int, device) -> "_Schedule":
        """table: (rows, >= steps) integers, negative = sample."""
        s = _Schedule(steps)
        t = np.ascontiguousarray(table[:, :steps].T, dtype=np.int64)  # (steps, rows)
        forced = t >= 0
        for i in range(steps):
            if forced[i].all():
                s.kinds[i] = _FORCE_ALL
            elif forced[i].any():
                s.kinds[i] = _MIXED
        s.per_row = torch.from_numpy(t).to(device)
        return s


class Engine:
    __slots__ = ("model", "use_graph", "_kept")

    def __init__(self, model: BaseGPT, use_graph: bool = True) -> None:
        """use_graph: replay the decode step as a captured HIP graph (same
        kernels and arithmetic as the eager forward, no per-step launch
        overhead); False runs every step eagerly.  The captured step and its
        cache (up to 1 GiB) are kept after a call and reused by the next call
        with the same prompts count, rows, prompt length and budget while the
        model's parameters are unchanged (same storage, no in-place update)."""
        self.model = model
        self.use_graph = use_graph
        self._kept = None  # (key, cache, _DecodeGraph), free for the next call

    def _graph_key(self, n_prompts: int, num_samples: int, prompt_len: int, steps: int) -> tuple:
        model = self.model
        params = tuple((p.data_ptr(), p._version) for p in model.parameters())
        buffers = tuple(b.data_ptr() for b in model.buffers())
        return (id(model), n_prompts, num_samples, prompt_len, steps, params, buffers)

    def _budget(self, prompt_len: int, max_tokens: int | None) -> int:
        # RoPE table covers 2*block_size positions (engine.py:55-64)
        ceiling = max(0, self.model.block_size * 2 - prompt_len)
        return ceiling if max_tokens is None else min(max_tokens, ceiling)

    @torch.inference_mode()
    def generate(
        self,
        tokens: list[int],
        num_samples: int = 1,
        max_tokens: int | None = None,
        sampler: Sampler | None = None,
        seed: int = 42,
        force_schedule: list[int | None] | None = None,
    ) -> Generator[tuple[list[int], list[int]], None, None]:
        """
        Streaming generation: single prefill, then clone the KV cache for each sample.

        `force_schedule`, when provided, is a per-step list aligned with the
        generation loop: `None` samples at that step, an `int` teacher-forces
        that token for every row.  Its length must be at least the number of
        generated steps.
        """
        # The per-row forcing queues of RowState are never filled inside a
        # generation call (engine.py:129-144 passes the sampled or scheduled
        # column through), so a column is the sampled/forced tokens and its
        # mask is 1 for a sampled step, 0 for a forced one.
        self._check_tokens(tokens)
        for column, mask in self._device_steps([tokens], num_samples, max_tokens, sampler, seed,
                                               force_schedule, per_prompt=False):
            yield column.tolist(), _mask_list(mask, num_samples)

    @torch.inference_mode()
    def generate_batch(
        self, tokens: list[int], num_samples: int = 1, **kwargs
    ) -> tuple[list[list[int]], list[list[int]]]:
        """
        Non-streaming batch generation that just returns the final token sequences.
        Returns (results, masks): each a list of `num_samples` lists of ints.
        """
        self._check_tokens(tokens)
        return self._collect([tokens], num_samples, kwargs, per_prompt=False)

    @torch.inference_mode()
    def generate_multi(
        self,
        prompts: list[list[int]],
        num_samples: int = 1,
        max_tokens: int | None = None,
        sampler: Sampler | None = None,
        seed: int = 42,
        force_schedule=None,
    ) -> Generator[tuple[list[int], list[int]], None, None]:
        """Streaming generation for several prompts of one length at once:
        row r = p * num_samples + i is trajectory i of prompt p.  Yields a
        (column, mask) pair of len(prompts) * num_samples ints per step.

        `force_schedule` may be None; one list shared by every row (as in
        generate); a list of per-prompt lists (the rows of a prompt share
        it); or a (rows, steps) integer array with a negative entry where the
        row samples.  A step that forces every row draws nothing from the
        generator; a step where some rows sample draws for all rows and keeps
        the forced tokens where they are scheduled."""
        self._check_prompts(prompts)
        for column, mask in self._device_steps(prompts, num_samples, max_tokens, sampler, seed,
                                               force_schedule, per_prompt=True):
            yield column.tolist(), _mask_list(mask, len(prompts) * num_samples)

    @torch.inference_mode()
    def generate_multi_batch(
        self, prompts: list[list[int]], num_samples: int = 1, **kwargs
    ) -> tuple[list[list[int]], list[list[int]]]:
        """generate_multi collected: (results, masks), len(prompts) *
        num_samples lists each, row p * num_samples + i for trajectory i of
        prompt p (the prompt followed by the generated tokens, masks 0 over
        the prompt)."""
        self._check_prompts(prompts)
        return self._collect(prompts, num_samples, kwargs, per_prompt=True)

    @torch.inference_mode()
    def score_continuations(self, tokens: list[int], continuations: list[list[int]]) -> list[list[float]]:
        """Log probability of every token of each candidate continuation of one prompt
        (row c: one float per token of continuations[c], given the prompt and the tokens
        before it).  The prompt is prefilled once; the continuations, of at most 65 tokens
        each, go behind its cache as trees of up to 64 tokens, which take them in the given
        order: beginnings that neighbours in that order share are run once.  The model must
        have GPT's forward_tree."""
        if not callable(getattr(self.model, "forward_tree", None)):
            raise TypeError(f"score_continuations needs a model with forward_tree, as GPT has: {type(self.model).__name__}")
        self._check_tokens(tokens)
        assert isinstance(continuations, list) and len(continuations) > 0, (
            "continuations must be a non-empty list of token lists"
        )
        for c in continuations:
            self._check_tokens(c)
            assert len(c) <= MAX_TREE + 1, f"a continuation has at most {MAX_TREE + 1} tokens, got {len(c)}"
        longest = max(len(c) for c in continuations)
        model = self.model
        assert all(0 <= t < model.vocab_size for c in [tokens, *continuations] for t in c), (
            "a token lies outside the vocabulary"
        )
        assert len(tokens) + longest - 1 <= model.block_size * 2, (
            f"prompt ({len(tokens)}) and continuation ({longest}) exceed 2 * block_size ({model.block_size * 2})"
        )
        device = model.device_type
        cache = KVCache(batch_size=1, num_heads=model.n_head, seq_len=len(tokens) + MAX_TREE,
                        head_dim=model.n_embd // model.n_head, num_layers=model.n_layer)
        kw = {"_last_only": True} if isinstance(model, GPT) else {}
        prompt = torch.tensor([tokens], dtype=torch.long, device=device)
        last = model.forward(prompt, kv_cache=cache, **kw)[0][0, -1:]
        scores: list[list[float]] = [[] for _ in continuations]
        for group, nodes, parents, places in _tries(continuations):
            logits = last
            if nodes:
                ids = torch.tensor([nodes], dtype=torch.long, device=device)
                logits = torch.cat([last, model.forward_tree(ids, parents, cache)[0]])
            # row 0 of the logits is the prompt's, row n + 1 token n's
            rows = torch.tensor([0 if p < 0 else p + 1 for c in group for p in places[c]], dtype=torch.long)
            wanted = torch.tensor([t for c in group for t in continuations[c]], dtype=torch.long)
            lp = token_logprobs(logits[rows.to(device)], wanted.to(device)).logprobs.tolist()
            for c in group:
                scores[c] = lp[: len(continuations[c])]
                lp = lp[len(continuations[c]) :]
        return scores

    @torch.inference_mode()
    def generate_paged(
        self,
        prompts: list[list[int]],
        max_tokens: int,
        temperature: float = 1.0,
        seed: int = 42,
        draft: BaseGPT | None = None,
        num_drafts: int = 4,
        keep: int | None = None,
        recent: int | None = None,
        page_size: int = 64,
    ) -> tuple[list[list[int]], list[list[float]]]:
        """max_tokens tokens (fewer where 2 * block_size positions end) behind each of several
        prompts of any lengths, decoded together over a PagedKVCache: returns (results,
        logprobs), each prompt followed by its tokens, and the model's log probability of each
        of these at the temperature (at 0, greedy decoding, at temperature 1).

        draft: a model of the same vocabulary, of any type, that proposes num_drafts tokens a row at a time,
        which this one runs all at once and keeps as far as verify_drafts lets them stand: the
        tokens are distributed as without it, in fewer passes.  keep: when a row comes to hold a
        page more than so many positions, it is cut to them, the ``recent`` last ones (None: half)
        and those that attention gave the largest weights; rejected drafts' weights count too."""
        self._check_ragged(prompts)
        for m in (self.model, draft):
            if m is not None and not callable(getattr(m, "forward_paged", None)):
                raise TypeError(f"generate_paged needs models with forward_paged, as GPT has: {type(m).__name__}")
        model = self.model
        assert all(0 <= t < model.vocab_size for p in prompts for t in p), "a token lies outside the vocabulary"
        assert temperature >= 0, "the temperature must not be negative"
        if draft is not None:
            assert draft.vocab_size == model.vocab_size, "the draft model must have the model's vocabulary"
            assert 1 <= num_drafts <= _native.MAX_DRAFTS, f"num_drafts must be 1 .. {_native.MAX_DRAFTS}, got {num_drafts}"
        if keep is not None:
            recent = keep // 2 if recent is None else recent
            assert keep >= 1 and 0 <= recent <= keep, f"keep {keep} positions, {recent} of them the last ones"
        device = torch.device(model.device_type)
        rng = torch.Generator(device=device)
        rng.manual_seed(seed)
        left = [self._budget(len(p), max_tokens) for p in prompts]
        if draft is not None:
            left = [min(n, max(0, draft.block_size * 2 - len(p))) for n, p in zip(left, prompts)]
        B, results, logprobs = len(prompts), [list(p) for p in prompts], [[] for _ in prompts]
        if max(left) <= 0:
            return results, logprobs
        ahead = num_drafts if draft is not None else 0
        # every row's last token is pending: run with the drafts behind it
        own = _PagedDecoder(model, prompts, left, ahead, page_size, keep, recent, device)
        side = None if draft is None else _PagedDecoder(draft, prompts, left, ahead, page_size, None, None, device)
        while max(left) > 0:
            n = [min(ahead, max(0, k - 1)) for k in left]
            N = max(n)
            drafts = drafted = None
            if N:
                drafts, drafted = side.propose(results, n, N, temperature, rng)
            logits = own.run([r[own.done[b] :] if left[b] else [] for b, r in enumerate(results)], drafts, n)
            tokens = torch.zeros((B, N), dtype=torch.long, device=device) if drafts is None else drafts
            u = e = None
            if temperature > 0:
                u = torch.rand((B, N), generator=rng, device=device)
                e = torch.empty((B, logits.size(-1)), device=device).exponential_(1, generator=rng)
            if drafted is not None and drafted.dtype != logits.dtype:  # to a type that holds both as they are
                both = torch.promote_types(drafted.dtype, logits.dtype)
                logits, drafted = logits.to(both), drafted.to(both)
            r = verify_drafts(logits, tokens, u, e, draft=drafted, counts=own.cache.ints(n), temperature=temperature)
            new, lps, stand = r.tokens.tolist(), r.logprobs.tolist(), r.accepted.tolist()
            for b in range(B):
                if left[b]:
                    results[b] += new[b][: stand[b] + 1]
                    logprobs[b] += lps[b][: stand[b] + 1]
                    left[b] -= stand[b] + 1
            for d in (own, side):
                if d is not None:
                    d.settle(results)
        return results, logprobs

    # -- shared machinery -------------------------------------------------------

    @classmethod
    def _check_ragged(cls, prompts) -> None:
        assert isinstance(prompts, list) and len(prompts) > 0, "prompts must be a non-empty list of token lists"
        for p in prompts:
            cls._check_tokens(p)

    @staticmethod
    def _check_tokens(tokens) -> None:
        assert isinstance(tokens, list), "tokens must be a list of ints"
        assert len(tokens) > 0, "tokens must be non-empty"
        assert all(isinstance(t, int) for t in tokens), "tokens must be a list of ints"

    @classmethod
    def _check_prompts(cls, prompts) -> None:
        assert isinstance(prompts, list) and len(prompts) > 0, "prompts must be a non-empty list of token lists"
        for p in prompts:
            cls._check_tokens(p)
        assert len({len(p) for p in prompts}) == 1, "prompts must all have the same length"

    def _collect(self, prompts, num_samples, kwargs, per_prompt):
        unknown = set(kwargs) - {"max_tokens", "sampler", "seed", "force_schedule"}
        if unknown:
            raise TypeError(f"generate() got unexpected keyword arguments {sorted(unknown)}")
        rows = len(prompts) * num_samples
        columns, masks = [], []
        for column, mask in self._device_steps(
            prompts, num_samples, kwargs.get("max_tokens"), kwargs.get("sampler"), kwargs.get("seed", 42),
            kwargs.get("force_schedule"), per_prompt=per_prompt,
        ):
            columns.append(column)
            masks.append(mask)
        T, steps = len(prompts[0]), len(columns)
        # the mask of a step that samples or forces every row is known on the
        # host already; when every step is such a step all rows share one mask
        on_device = [s for s, m in enumerate(masks) if isinstance(m, torch.Tensor)]
        # about 2 * rows lists of Python ints are built here: with the garbage
        # collector running, a full collection triggered meanwhile walks every
        # list already built (measured: 100+ ms on a 6400-row call)
        gc_enabled = gc.isenabled()
        gc.disable()
        try:
            # the lists that need nothing from the device are built first,
            # while it still runs the steps enqueued above
            results = [prompts[r // num_samples].copy() for r in range(rows)]
            if not on_device:
                shared = [0] * T + [int(m) for m in masks]
                out_masks = [shared.copy() for _ in range(rows)]
            else:
                mask_np = np.empty((rows, steps), dtype=np.int64)
                for s, m in enumerate(masks):
                    if not isinstance(m, torch.Tensor):
                        mask_np[:, s] = m
                mask_np[:, on_device] = torch.stack([masks[s] for s in on_device], dim=1).cpu().numpy()
                zeros = [0] * T
                out_masks = [zeros + row for row in mask_np.tolist()]
            if gc_enabled:
                # the youngest generation's collection, which these lists
                # would trigger once the collector runs again, happens now:
                # while the device may still work, and over the rows before
                # the generated tokens lengthen them
                gc.collect(0)
            # the token columns reach the host in one copy
            if columns:
                for row, gen in zip(results, torch.stack(columns, dim=1).cpu().numpy().tolist()):
                    row += gen
        finally:
            if gc_enabled:
                gc.enable()
        return results, out_masks

    def _schedule(self, force_schedule, steps: int, n_prompts: int, num_samples: int, per_prompt: bool,
                  device) -> _Schedule | None:
        if force_schedule is None:
            return None
        rows = n_prompts * num_samples
        if not per_prompt or (len(force_schedule) > 0 and not isinstance(force_schedule[0], (list, tuple))
                              and not isinstance(force_schedule, np.ndarray)
                              and not isinstance(force_schedule, torch.Tensor)):
            assert len(force_schedule) >= steps, (
                f"force_schedule must cover all generation steps "
                f"(len={len(force_schedule)} < {steps})"
            )
            return _Schedule.shared_list(force_schedule, steps)
        if isinstance(force_schedule, (np.ndarray, torch.Tensor)):
            table = np.asarray(force_schedule.cpu() if isinstance(force_schedule, torch.Tensor) else force_schedule)
            assert table.ndim == 2 and table.shape[0] == rows, (
                f"a per-row force_schedule must be (rows={rows}, steps), got {table.shape}"
            )
        else:
            assert len(force_schedule) == n_prompts, (
                f"force_schedule must hold one schedule per prompt ({len(force_schedule)} != {n_prompts})"
            )
            width = min(len(s) for s in force_schedule)
            table = np.full((n_prompts, width), -1, dtype=np.int64)
            for p, s in enumerate(force_schedule):
                table[p] = [-1 if t is None else t for t in s[:width]]
            table = np.repeat(table, num_samples, axis=0)
        assert table.shape[1] >= steps, (
            f"force_schedule must cover all generation steps (len={table.shape[1]} < {steps})"
        )
        return _Schedule.table(table, steps, device)

    def _device_steps(
        self,
        prompts: list[list[int]],
        num_samples: int,
        max_tokens: int | None,
        sampler: Sampler | None,
        seed: int,
        force_schedule,
        per_prompt: bool,
    ) -> Generator[tuple[torch.Tensor, "int | torch.Tensor"], None, None]:
        """The generation loop with the token columns kept on the device:
        yields ((rows,) int64 column, mask) per step -- mask 1 / 0 for a step
        that samples / forces every row, a (rows,) int64 device tensor
        otherwise -- and feeds each column to the next decode forward without
        a host round trip."""
        T = len(prompts[0])
        S, N = len(prompts), num_samples
        rows = S * N
        steps = self._budget(T, max_tokens)
        if steps == 0:
            return

        model = self.model
        device = model.device_type
        schedule = self._schedule(force_schedule, steps, S, N, per_prompt, device)
        rng = torch.Generator(device=device)
        rng.manual_seed(seed)
        geometry = {
            "num_heads": model.n_head,
            "head_dim": model.n_embd // model.n_head,
            "num_layers": model.n_layer,
        }
        # the prefill's caller reads the last position's logits only
        prefill_kw = {"_last_only": True} if isinstance(model, GPT) else {}
        use_graph = self.use_graph and steps > 1 and torch.device(device).type == "cuda"
        key = self._graph_key(S, N, T, steps) if use_graph else None
        kept, self._kept = self._kept, None  # taken: a concurrent call builds its own
        reuse = kept is not None and kept[0] == key
        if kept is not None and not reuse:
            kept[2].close()
        ids = torch.tensor(prompts, dtype=torch.long, device=device)

        decode = None
        if N == 1:
            # one row per prompt: the prefill writes the decode cache itself
            if reuse:
                _, cache, decode = kept
                cache.reset()
            else:
                cache = KVCache(batch_size=S, seq_len=T + steps, **geometry)
            pos_dev, cache.pos_dev = cache.pos_dev, None  # a prefill, not the captured step
            try:
                logits, _ = model.forward(ids, kv_cache=cache, **prefill_kw)
            finally:
                cache.pos_dev = pos_dev
            logits = logits[:, -1, :]
        else:
            # 1) batched prefill of the prompts
            prompt_cache = KVCache(batch_size=S, seq_len=T, **geometry)
            logits, _ = model.forward(ids, kv_cache=prompt_cache, **prefill_kw)
            logits = logits[:, -1, :]
            logits = logits.expand(N, -1) if S == 1 else logits.repeat_interleave(N, dim=0)
            # 2) every row of a prompt starts from that prompt's cache, stored
            #    once as prefix pages (read once per decode step); a step
            #    captured by an earlier call with the same key replays into its
            #    own cache
            if reuse:
                _, cache, decode = kept
                cache._prefill_groups(prompt_cache, N, reuse=True)
            else:
                cache = KVCache(batch_size=rows, seq_len=T + steps, **geometry)
                cache._prefill_groups(prompt_cache, N)
            del prompt_cache
        if decode is not None:
            decode.rewind()
        elif use_graph:
            decode = _DecodeGraph(model, cache, rows, torch.device(device))

        try:
            for step in range(steps):
                kind = _SAMPLE if schedule is None else schedule.kinds[step]
                if kind == _FORCE_ALL:
                    if schedule.per_row is not None:
                        column = schedule.per_row[step]
                    else:
                        column = torch.full((rows,), schedule.shared[step], dtype=torch.long, device=logits.device)
                    mask = 0
                else:
                    if sampler is not None:
                        picked = sampler(logits, rng=rng)
                    else:
                        picked = draw_one(torch.softmax(logits, dim=-1), rng)
                    column = picked[:, 0]
                    mask = 1
                    if kind == _MIXED:
                        forced = schedule.per_row[step]
                        scheduled = forced >= 0
                        column = torch.where(scheduled, forced, column)
                        mask = (~scheduled).long()
                yield column, mask
                if step == steps - 1:
                    break  # the last column's logits would go unused

                # 3) one decode forward for the column just emitted
                step_ids = column.unsqueeze(1)
                if decode is not None:
                    logits = decode.step(step_ids)
                else:
                    logits, _ = model.forward(step_ids, kv_cache=cache)
                    logits = logits[:, -1, :]
        finally:
            if decode is not None:
                if cache.nbytes() <= _KEEP_GRAPH_BYTES:
                    self._kept = (key, cache, decode)
                else:
                    decode.close()


class _PagedDecoder:
    """One model's side of generate_paged: its cache, and how many of each row's tokens the
    cache holds (``done``; the last token is never among them)."""

    __slots__ = ("model", "cache", "done", "keep", "recent", "device")

    # prompts go through the layers so many tokens a row at a time
    CHUNK = 256

    def __init__(self, model: BaseGPT, prompts: list[list[int]], left: list[int], ahead: int, page_size: int,
                 keep: int | None, recent: int | None, device: torch.device) -> None:
        self.model, self.keep, self.recent, self.device = model, keep, recent, device
        self.done = [0] * len(prompts)
        chunk = self.CHUNK
        most = [len(p) + n + ahead for p, n in zip(prompts, left)]
        if keep is not None:  # what a row holds before it is cut: a page and a chunk, or a round's drafts, more
            most = [min(m, keep + page_size + max(chunk, ahead + 1)) for m in most]
        pages = sum(-(-m // page_size) for m in most)
        if keep is not None:
            pages += -(-keep // page_size)  # the pages that a row is cut into
        w = next(model.parameters())
        self.cache = PagedKVCache(len(prompts), model.n_head, model.n_embd // model.n_head, model.n_layer, pages, page_size,
                                  max(most), w.dtype, device, weights=keep is not None)
        ends = [len(p) - 1 if n else 0 for p, n in zip(prompts, left)]  # rows with nothing to come stay empty
        while self.done != ends:
            parts = [p[at : min(at + chunk, end)] for p, at, end in zip(prompts, self.done, ends)]
            self._forward(parts)
            self.done = [at + len(part) for at, part in zip(self.done, parts)]
            self._cut()

    def _forward(self, parts: list[list[int]], more: torch.Tensor | None = None, counts: list[int] | None = None) -> torch.Tensor:
        """Logits of the rows' next tokens: parts[b], and behind them counts[b] of more's."""
        N = max(len(p) for p in parts)
        ids = self.cache.ints([p + [0] * (N - len(p)) for p in parts]).long()
        if more is not None:
            ids = torch.cat([ids, more], dim=1)
        n = [len(p) + (0 if counts is None else counts[b]) for b, p in enumerate(parts)]
        return self.model.forward_paged(ids, self.cache, n)

    def run(self, pending: list[list[int]], drafts: torch.Tensor | None, n: list[int]) -> torch.Tensor:
        """Logits (B, N + 1, V) behind each row's one pending token and its drafts; rows
        that have ended have none."""
        counts = [c if p else 0 for p, c in zip(pending, n)]
        return self._forward(pending, drafts, counts)

    def propose(self, results: list[list[int]], n: list[int], N: int, temperature: float,
                rng: torch.Generator) -> tuple[torch.Tensor, torch.Tensor | None]:
        """n[b] drafts of each row behind its tokens, drawn one after the other: (B, N) ids,
        and the (B, N, V) logits they were drawn from (None at temperature 0)."""
        parts = [r[at:] if c else [] for r, at, c in zip(results, self.done, n)]
        logits = self._forward(parts)
        last = self.cache.ints([max(0, len(p) - 1) for p in parts]).long()
        row = logits[torch.arange(len(parts), device=self.device), last]
        ids, rows = [], []
        for i in range(N):
            if temperature == 0:
                step = torch.argmax(row, dim=-1, keepdim=True)
            else:
                step = draw_one(torch.softmax(row.float() / temperature, dim=-1), rng)
            ids.append(step)
            rows.append(row)
            if i + 1 < N:
                row = self.model.forward_paged(step, self.cache, [int(c > i + 1) for c in n])[:, 0]
        return torch.cat(ids, dim=1), None if temperature == 0 else torch.stack(rows, dim=1)

    def settle(self, results: list[list[int]]) -> None:
        """After a round: of what the cache holds, the tokens that became results stay, all but
        the last, which is pending."""
        now = [min(p, len(r) - 1) for p, r in zip(self.cache.next_pos, results)]
        self.cache.truncate([a - (p - t) for a, p, t in zip(self.cache.lens, self.cache.next_pos, now)])
        self.done = now
        self._cut()

    def _cut(self) -> None:
        if self.keep is not None:  # each row by its own length, whatever the others'
            long = [b for b, n in enumerate(self.cache.lens) if n >= self.keep + self.cache.page_size]
            if long:
                self.cache.evict(self.keep, self.recent, long)


def _tries(continuations: list[list[int]]):
    """The continuations in groups whose tries have at most MAX_TREE inner tokens (a last
    token is scored, never run): yields a group's numbers, its trie's tokens and parents,
    and for each number the token before each of its own (-1: the prompt)."""
    at = 0
    while at < len(continuations):
        group: list[int] = []
        nodes: list[int] = []
        parents: list[int] = []
        child: dict[tuple[int, int], int] = {}
        places: dict[int, list[int]] = {}
        while at < len(continuations):
            c = continuations[at]
            new_nodes, place, above = 0, [], -1
            added: list[tuple[int, int]] = []
            for t in c:
                place.append(above)
                if len(place) == len(c):
                    break
                key = (above, t)
                if key in child:
                    above = child[key]
                else:
                    above = len(nodes) + new_nodes
                    child[key] = above
                    added.append(key)
                    new_nodes += 1
            if len(nodes) + new_nodes > MAX_TREE:
                break  # the next group's
            for key in added:
                parents.append(key[0])
                nodes.append(key[1])
            places[at] = place
            group.append(at)
            at += 1
        yield group, nodes, parents, places


def _mask_list(mask, rows: int) -> list[int]:
    return mask.tolist() if isinstance(mask, torch.Tensor) else [mask] * rows
