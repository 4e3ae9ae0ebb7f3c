"""The model over a paged cache (GPT.forward_paged, PagedKVCache) and decoding with it
(Engine.generate_paged): prompts of different lengths, drafts, evicted positions, against one
series at a time."""

import copy

import pytest
import torch

from diff_gpt.model.engine import Engine
from diff_gpt.model.gpt import GPT
from diff_gpt.model.paged import PagedKVCache
from diff_gpt.sampler.temperature import TemperatureSampler

pytestmark = pytest.mark.gpu


def _gpt(dev, dtype=torch.float32, n_embd=64, n_head=4, n_layer=2, vocab=256, block_size=138, seed=0):
    torch.manual_seed(seed)
    return GPT(vocab_size=vocab, n_embd=n_embd, block_size=block_size, n_head=n_head, n_layer=n_layer).eval().to(dev).to(dtype)


def _series(lengths, vocab=256, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def _cache(model, rows, pages=64, page_size=16, **kw):
    w = next(model.parameters())
    return PagedKVCache(rows, model.n_head, model.n_embd // model.n_head, model.n_layer, pages, page_size, dtype=w.dtype,
                        device=w.device, **kw)


def _pad(parts, dev):
    n = max(len(p) for p in parts)
    return torch.tensor([p + [7] * (n - len(p)) for p in parts], dtype=torch.long, device=dev)


# fp32, and fp64 whose other paths turn keys in fp32: within 1e-5 of the softcapped logits
TOL = 2e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("n_embd,n_head", [(64, 4), (128, 4), (512, 8), (96, 4)])
def test_forward_in_ragged_chunks(dev, dtype, n_embd, n_head):
    model = _gpt(dev, dtype, n_embd, n_head)
    seqs = _series([1, 40, 138, 276, 17])
    exact = copy.deepcopy(model).double()
    cache = _cache(model, len(seqs))
    got = [[] for _ in seqs]
    with torch.inference_mode():
        for n in (1, 30, 0, 90, 1, 200):
            parts = [s[at : at + n - b % 3 if n > 3 else at + n] for b, (s, at) in enumerate(zip(seqs, cache.lens))]
            if not any(parts):
                continue
            logits = model.forward_paged(_pad(parts, dev), cache, [len(p) for p in parts])
            for b, p in enumerate(parts):
                got[b].append(logits[b, : len(p)])
        assert cache.lens == cache.lengths.tolist() == cache.positions.tolist() == cache.next_pos
        for b, s in enumerate(seqs):
            g = torch.cat(got[b])
            assert len(g) > 0
            ids = torch.tensor([s[: len(g)]], device=dev)
            plain, ref = model(ids)[0][0], exact(ids)[0][0]
            if dtype in (torch.float32, torch.float64):
                assert bool(((g.double() - plain.double()).abs() <= TOL).all())
            else:
                # 16-bit: rounding through the layers, held to 1.5 times what the plain forward is off by
                rms = lambda x: float((x.double() - ref).square().mean().sqrt())  # noqa: E731
                assert rms(g) <= 1.5 * rms(plain)


@pytest.mark.parametrize("page_size", [4, 64])
def test_greedy_decoding_of_ragged_prompts(dev, page_size):
    model = _gpt(dev)
    prompts = _series([1, 5, 138, 64, 260, 17])
    results, logprobs = Engine(model).generate_paged(prompts, 30, temperature=0, page_size=page_size)
    for p, r, lp in zip(prompts, results, logprobs):
        want, _ = Engine(model).generate_batch(p, 1, max_tokens=30, sampler=TemperatureSampler(0))
        assert r == want[0]
        scored = model.score([r])[0].logprobs[len(p) - 1 :]
        assert torch.allclose(torch.tensor(lp), scored.cpu(), atol=1e-4)
    assert len(results[4]) == 276  # 2 * block_size positions


@pytest.mark.parametrize("num_drafts", [1, 4, 9])
def test_drafts_change_no_greedy_token(dev, num_drafts):
    model, other = _gpt(dev), _gpt(dev, n_layer=1, seed=3)
    prompts = _series([3, 90, 1, 33])
    plain = Engine(model).generate_paged(prompts, 41, temperature=0)
    for draft in (model, other):
        got = Engine(model).generate_paged(prompts, 41, temperature=0, draft=draft, num_drafts=num_drafts)
        assert got[0] == plain[0]
        for a, b in zip(got[1], plain[1]):
            assert torch.allclose(torch.tensor(a), torch.tensor(b), atol=1e-4)


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_sampling_with_and_without_drafts(dev, temperature):
    model, other = _gpt(dev), _gpt(dev, n_layer=1, seed=3)
    prompts = _series([3, 90, 1, 33])
    for draft in (None, model, other):
        engine = Engine(model)
        results, logprobs = engine.generate_paged(prompts, 25, temperature=temperature, seed=1, draft=draft)
        again = engine.generate_paged(prompts, 25, temperature=temperature, seed=1, draft=draft)
        assert (results, logprobs) == again
        for p, r, lp in zip(prompts, results, logprobs):
            assert r[: len(p)] == p and len(r) == len(p) + 25 == len(p) + len(lp)
            ids = torch.tensor([r], device=dev)
            with torch.inference_mode():
                logs = torch.log_softmax(model(ids)[0][0].double() / temperature, -1)
            want = logs[:-1].gather(-1, ids[0, 1:, None])[len(p) - 1 :, 0]
            assert torch.allclose(torch.tensor(lp, dtype=torch.float64), want.cpu(), atol=3e-4)


def test_the_models_own_drafts_stand(dev):
    """A model that drafts for itself: all drafts stand, but where rounding decides (u within 1e-5 of 1)."""
    model = _gpt(dev)
    calls = []
    inner = model.forward_paged
    model.forward_paged = lambda *a, **kw: calls.append(a[0].shape[1]) or inner(*a, **kw)
    Engine(model).generate_paged(_series([5, 9]), 40, draft=model, num_drafts=4)
    # prefills, and rounds of 4 drafts (4 passes: one of 1 or 2 tokens, 3 of one) and one of 5 tokens each
    assert calls.count(5) == 8


def test_a_budget_that_is_never_reached_changes_nothing(dev):
    model = _gpt(dev)
    prompts = _series([3, 90, 33])
    plain = Engine(model).generate_paged(prompts, 30, temperature=0)
    assert Engine(model).generate_paged(prompts, 30, temperature=0, keep=200) == plain


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("page_size,keep,recent", [(16, 40, 10), (4, 7, None), (64, 1, 1)])
def test_decoding_within_a_budget(dev, draft, page_size, keep, recent, monkeypatch):
    model = _gpt(dev)
    held = []
    advance = PagedKVCache.advance
    monkeypatch.setattr(PagedKVCache, "advance", lambda self, *a: (advance(self, *a), held.append((self.weights is not None, max(self.lens)))))
    prompts = _series([3, 250, 33, 1])
    results, logprobs = Engine(model).generate_paged(prompts, 26, keep=keep, recent=recent, page_size=page_size,
                                                     draft=_gpt(dev, n_layer=1, seed=3) if draft else None)
    assert [len(r) for r in results] == [29, 276, 59, 27] and all(len(lp) == 26 for lp in logprobs)
    assert max(n for own, n in held if own) <= keep + page_size + 256


def test_rows_are_cut_by_their_own_length(dev, monkeypatch):
    """A budget cuts a row that holds a page more, and leaves those beside it that do not."""
    model = _gpt(dev)
    cut = []
    evict = PagedKVCache.evict
    monkeypatch.setattr(PagedKVCache, "evict", lambda self, *a: (cut.append((list(self.lens), a)), evict(self, *a))[1])
    Engine(model).generate_paged(_series([60, 45, 30]), 20, temperature=0, keep=40, recent=20, page_size=16)
    assert cut and any(40 < n < 56 for lens, _ in cut for n in lens)
    for lens, a in cut:
        assert a == (40, 20, [b for b, n in enumerate(lens) if n >= 56])
    cache = _cache(model, 3, weights=True)
    model.forward_paged(_pad(_series([30, 25, 9]), dev), cache, [30, 25, 9])
    cache.evict(20, 5, [1, 2])
    assert cache.lens == [30, 20, 9] and cache.next_pos == [30, 25, 9]
    with pytest.raises(ValueError, match="counts"):
        cache.advance([1])


def test_evicted_rows_attend_to_what_is_kept(dev):
    """In a model of one layer a position's key and value depend on its token alone, so a row cut
    to some positions is a row that those tokens alone were fed to."""
    model = _gpt(dev, n_layer=1)
    prompts = _series([60, 41, 12])
    cache = _cache(model, 3, weights=True)
    model.forward_paged(_pad(prompts, dev), cache, [60, 41, 12])
    assert torch.allclose(cache.weights[0].sum((1, 2)).cpu(), torch.tensor([60.0, 41.0, 12.0]) * 4, rtol=1e-5)
    g = torch.Generator().manual_seed(0)
    cache.weights[0] = torch.rand(cache.weights.shape[-1], generator=g).to(dev)  # one choice for all heads
    free = cache.free_pages
    kept = cache.evict(20, 5)
    assert cache.lens == [20, 20, 12] and cache.next_pos == [60, 41, 12] == cache.positions.tolist()
    assert cache.free_pages == free + (4 - 2) + (3 - 2)
    other = _cache(model, 3)
    for j in range(20):
        at = [int(kept[0][0][b, 0, j]) if b < 2 else j for b in range(3)]
        n = [1, 1, int(j < 12)]
        other.next_pos = at
        other._sync()
        model.forward_paged(torch.tensor([[p[t] if c else 0] for p, t, c in zip(prompts, at, n)], device=dev), other, n)
    other.next_pos = [60, 41, 12]
    other._sync()
    ids = torch.tensor([[5, 6, 7]] * 3, device=dev)
    a, b = model.forward_paged(ids, cache), model.forward_paged(ids, other)
    assert bool(((a - b).abs() <= TOL).all())
    # what the kept positions were given moved with them, the new ones start from nothing
    assert bool((cache.weights[0, 0, :, 23:] == 0).all()) and bool((cache.weights[0, 0, :, 20:23] > 0).all())


def test_bookkeeping(dev):
    model = _gpt(dev)
    cache = _cache(model, 2, pages=4, page_size=16, weights=True)
    ids = torch.tensor([_series([40])[0]] * 2, device=dev)
    with pytest.raises(RuntimeError, match="more pages"):
        model.forward_paged(ids, cache)  # 6 pages
    assert cache.lens == [0, 0] and cache.free_pages == 4
    model.forward_paged(ids[:, :17], cache, [17, 16])
    assert cache.lens == [17, 16] and cache.free_pages == 1
    first = model.forward_paged(ids[:, 17:19], cache, [2, 0])[0]
    cache.truncate([17, 3])
    assert cache.free_pages == 1 and not cache.weights[:, 0, :, 17:].any() and not cache.weights[:, 1, :, 3:].any()
    again = model.forward_paged(ids[:, 17:19], cache, [2, 0])[0]
    assert torch.equal(first, again)
    with pytest.raises(ValueError, match="go back"):
        cache.truncate([20, 3])
    with pytest.raises(ValueError, match="counts"):
        cache.reserve([1])
    with pytest.raises(RuntimeError, match="room for"):
        cache.reserve([100, 0])
    cache.release([0])
    assert cache.lens == [0, 3] and cache.free_pages == 3
    one = model.forward_paged(ids[:, :19], cache, [19, 0])[0]
    assert torch.allclose(one[17:], first, atol=TOL)
    with pytest.raises(RuntimeError, match="free pages"):
        cache.evict(18, 2)  # 2 pages, 1 free
    assert cache.lens == [19, 3]
    with pytest.raises(RuntimeError, match="weights"):
        _cache(model, 1).evict(2, 1)
    with pytest.raises(TypeError, match="computes in"):
        model.forward_paged(ids[:, :1], PagedKVCache(2, 4, 16, 2, 4, dtype=torch.bfloat16, device=dev))
    for kw in (dict(rows=0), dict(page_size=3), dict(pages=0), dict(max_positions=2**31)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(rows=1, num_heads=1, head_dim=16, num_layers=1, pages=2, device=dev), **kw})
    with pytest.raises(RuntimeError, match="ROCm"):
        PagedKVCache(1, 1, 16, 1, 2, device="cpu")


def test_refusals(dev):
    model = _gpt(dev)
    engine = Engine(model)
    with pytest.raises(AssertionError, match="2 . block_size"):
        cache = _cache(model, 1)
        model.forward_paged(torch.zeros(1, 277, dtype=torch.long, device=dev), cache)
    with pytest.raises(AssertionError, match="rows"):
        model.forward_paged(torch.zeros(2, 1, dtype=torch.long, device=dev), _cache(model, 1))
    with pytest.raises(AssertionError, match="counts"):
        model.forward_paged(torch.zeros(1, 1, dtype=torch.long, device=dev), _cache(model, 1), [2])
    with pytest.raises(AssertionError, match="vocabulary"):
        engine.generate_paged([[256]], 3)
    with pytest.raises(AssertionError, match="non-empty"):
        engine.generate_paged([[1], []], 3)
    with pytest.raises(AssertionError, match="temperature"):
        engine.generate_paged([[1]], 3, temperature=-1)
    with pytest.raises(AssertionError, match="vocabulary"):
        engine.generate_paged([[1]], 3, draft=_gpt(dev, vocab=128))
    with pytest.raises(AssertionError, match="num_drafts"):
        engine.generate_paged([[1]], 3, draft=model, num_drafts=65)
    with pytest.raises(AssertionError, match="keep"):
        engine.generate_paged([[1]], 3, keep=2, recent=3)
    with pytest.raises(TypeError, match="forward_paged"):
        Engine(torch.nn.Identity()).generate_paged([[1]], 3)
    assert engine.generate_paged([[1, 2], [3]], 0) == ([[1, 2], [3]], [[], []])
    long = [3] * 276
    assert engine.generate_paged([long, [3] * 275], 4, temperature=0)[0][0] == long
