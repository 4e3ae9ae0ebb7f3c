"""Decoding over pages: models of different types, and rows that go back after they were cut."""

import pytest
import torch

from diff_gpt.model.engine import Engine
from diff_gpt.model.gpt import GPT
from diff_gpt.model.paged import PagedKVCache

pytestmark = pytest.mark.gpu


def _gpt(dev, dtype=torch.float32, n_layer=2, seed=0):
    torch.manual_seed(seed)
    return GPT(vocab_size=256, n_embd=64, block_size=138, n_head=4, n_layer=n_layer).eval().to(dev).to(dtype)


def _series(lengths):
    g = torch.Generator().manual_seed(0)
    return [torch.randint(0, 256, (n,), generator=g).tolist() for n in lengths]


@pytest.mark.parametrize("dtype,other", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                         (torch.bfloat16, torch.float16), (torch.float64, torch.float32)])
@pytest.mark.parametrize("temperature", [0, 1.0])
def test_a_draft_model_of_another_type(dev, dtype, other, temperature):
    model, draft = _gpt(dev, dtype), _gpt(dev, other, n_layer=1, seed=3)
    prompts = _series([3, 90, 1, 33])
    engine = Engine(model)
    results, logprobs = engine.generate_paged(prompts, 25, temperature=temperature, seed=1, draft=draft)
    for p, r, lp in zip(prompts, results, logprobs):
        assert r[: len(p)] == p and len(r) == len(p) + 25 == len(p) + len(lp)
        if dtype == torch.float32:
            scored = model.score([r])[0].logprobs[len(p) - 1 :]
            assert torch.allclose(torch.tensor(lp), scored.cpu(), atol=3e-4)
    if temperature == 0 and dtype in (torch.float32, torch.float64):
        assert results == engine.generate_paged(prompts, 25, temperature=0)[0]


def _cut(dev, model, keep=20, recent=5):
    cache = PagedKVCache(2, 4, 16, 2, 16, 16, device=dev, weights=True)
    ids = torch.tensor(_series([60, 60]), device=dev)
    model.forward_paged(ids, cache, [60, 18])
    cache.evict(keep, recent)
    return cache


def test_rows_go_back_to_the_recent_positions_of_a_cut(dev):
    """Behind a cut the newest positions are one after the other: going back to one of them, and
    to what came later, stands where it stood; among the others every key head has its own."""
    model = _gpt(dev)
    cache = _cut(dev, model)
    assert cache.lens == [20, 18] and cache.next_pos == [60, 18]
    cache.truncate([16, 10])
    assert cache.lens == [16, 10] and cache.next_pos == [56, 10]
    cache.truncate([15, 10])
    assert cache.next_pos == [55, 10]
    for n in (14, 1):
        with pytest.raises(ValueError, match="cut"):
            cache.truncate([n, 9])
        assert cache.lens == [15, 10] and cache.next_pos == [55, 10]
    cache.truncate([15, 3])
    model.forward_paged(torch.zeros(2, 6, dtype=torch.long, device=dev), cache, [6, 0])
    cache.truncate([17, 3])
    assert cache.lens == [17, 3] and cache.next_pos == [57, 3]


def test_rows_that_go_back_to_nothing_begin_anew(dev):
    model = _gpt(dev)
    cache = _cut(dev, model)
    cache.truncate([0, 18])
    assert cache.lens == [0, 18] and cache.next_pos == [0, 18] == cache.positions.tolist()
    ids = torch.tensor([_series([30])[0]] * 2, device=dev)
    got = model.forward_paged(ids, cache, [30, 0])[0]
    fresh = model.forward_paged(ids, PagedKVCache(2, 4, 16, 2, 16, 16, device=dev), [30, 0])[0]
    assert torch.equal(got, fresh)
    cache.truncate([7, 18])  # a row that begins anew was not cut
    assert cache.next_pos == [7, 18]
    cache = _cut(dev, model)
    cache.release([0])
    model.forward_paged(ids, cache, [30, 0])
    cache.truncate([7, 18])
    assert cache.next_pos == [7, 18]


def test_a_row_that_was_cut_twice(dev):
    """More recent positions than follow one another since the first cut."""
    model = _gpt(dev)
    cache = _cut(dev, model, 20, 5)
    model.forward_paged(torch.zeros(2, 6, dtype=torch.long, device=dev), cache, [6, 0])
    cache.evict(19, 15)  # of the last 15 positions 11 follow one another
    assert cache.lens == [19, 18] and cache.next_pos == [66, 18]
    with pytest.raises(ValueError, match="cut"):
        cache.truncate([7, 18])
    cache.truncate([8, 18])
    assert cache.next_pos == [55, 18]
