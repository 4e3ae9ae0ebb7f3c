"""Scoring through the model: packed series of different lengths (GPT.score,
DiffGPT.anomaly_scores_batch), trees of candidate tokens behind a cache (GPT.forward_tree,
KVCache.keep, Engine.score_continuations), against one series, or one path, at a time."""

import copy

import numpy as np
import pandas as pd
import pytest
import torch

from diff_gpt.diff_gpt import DiffGPT
from diff_gpt.model.engine import Engine
from diff_gpt.model.gpt import GPT
from diff_gpt.model.kv_cache import KVCache
from seq_cases import some_tree, tree_seen

pytestmark = pytest.mark.gpu


def _gpt(dev, dtype=torch.float32, n_embd=64, n_head=4, n_layer=2, vocab=256, block_size=138, **kw):
    torch.manual_seed(0)
    return GPT(vocab_size=vocab, n_embd=n_embd, block_size=block_size, n_head=n_head, n_layer=n_layer,
               **kw).eval().to(dev).to(dtype)


def _series(lengths, vocab, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


# Whole models agree within 1e-5 of the logits (softcapped at 15) in fp32, through other
# orders of the sums.
TOL = {torch.float32: 2e-4, torch.float64: 1e-9}


def _near(dtype, got, plain, exact):
    """fp32 and fp64: got within TOL of the same model's plain forward.  16-bit: rounding
    through the layers exceeds any such bar, so got is held to the fp64 model of the same
    weights, at 1.5 times the root mean square the plain forward is off by."""
    got, plain, exact = got.double(), plain.double(), exact.double()
    if dtype in TOL:
        return bool(((got - plain).abs() <= TOL[dtype]).all())
    rms = lambda x: float((x - exact).square().mean().sqrt())  # noqa: E731
    return rms(got) <= 1.5 * rms(plain)


def _exact(model):
    return copy.deepcopy(model).double()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("n_embd,n_head", [(64, 4), (128, 4), (512, 8), (96, 4)])
def test_score_matches_one_series_at_a_time(dev, dtype, n_embd, n_head):
    model = _gpt(dev, dtype, n_embd, n_head)
    exact = _exact(model)
    seqs = _series([1, 2, 138, 17, 276, 64, 33, 128], 256)
    lps, ents, tops = [], [], []
    with torch.inference_mode():
        got = model.score(seqs, top=3)
        assert len(got) == len(seqs)
        for s, r in zip(seqs, got):
            assert r.logprobs.shape == (len(s) - 1,) and r.top_ids.shape == (len(s) - 1, 3)
            ids = torch.tensor([s], device=dev)
            rows = []
            for m in (model, exact):
                logs = torch.log_softmax(m(ids)[0][0, :-1].double(), dim=-1)
                rows.append((logs.gather(-1, ids[0, 1:, None])[:, 0], -(logs.exp() * logs).sum(-1),
                             logs.gather(-1, r.top_ids), logs))
            lps.append((r.logprobs, rows[0][0], rows[1][0]))
            ents.append((r.entropy, rows[0][1], rows[1][1]))
            tops.append((r.top_logprobs, rows[0][2], rows[1][2]))
            if dtype in TOL and len(s) > 1:
                # no other id is likelier than the named ones by more than both are off
                best = rows[0][3].sort(-1, descending=True)[0][:, :3]
                assert bool((best - rows[0][2] <= 2 * TOL[dtype]).all())
    for parts in (lps, ents, tops):
        assert _near(dtype, *(torch.cat([p[i] for p in parts]) for i in range(3)))


def test_score_in_batches_of_tokens(dev):
    model = _gpt(dev)
    seqs = _series([100, 30, 60, 5, 276, 1, 44], 256, seed=1)
    whole = model.score(seqs)
    for limit in (1, 64, 131, 300):
        for a, b in zip(whole, model.score(seqs, max_tokens=limit)):
            assert a.logprobs.shape == b.logprobs.shape
            assert bool(((a.logprobs - b.logprobs).abs() <= TOL[torch.float32]).all())
    assert model.score([]) == []


def test_score_on_another_stream(dev):
    model = _gpt(dev)
    seqs = _series([50, 90, 20], 256, seed=2)
    want = model.score(seqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = model.score(seqs)
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a.logprobs, b.logprobs)


def test_score_refusals(dev):
    model = _gpt(dev, vocab=64)
    for bad in ([[]], [[0] * 277], [[64]], [[-1]]):
        with pytest.raises(AssertionError):
            model.score(bad)
    with pytest.raises(AssertionError):
        model.score([[1, 2]], top=65)
    with pytest.raises(AssertionError):
        model.score([[1, 2]], max_tokens=0)


def _path(parents, n):
    path = []
    while n >= 0:
        path.append(n)
        n = parents[n]
    return path[::-1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("n_embd,n_head,prompt,N", [(64, 4, 40, 12), (512, 8, 100, 31), (128, 4, 1, 64), (64, 4, 17, 1)])
def test_forward_tree_matches_its_paths(dev, dtype, n_embd, n_head, prompt, N):
    model = _gpt(dev, dtype, n_embd, n_head)
    B = 3
    parents = some_tree(N, seed=N)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 256, (B, prompt), generator=g).to(dev)
    nodes = torch.randint(0, 256, (B, N), generator=g).to(dev)
    with torch.inference_mode():
        cache = KVCache(B, n_head, prompt + N, n_embd // n_head, 2)
        model(ids, kv_cache=cache)
        logits = model.forward_tree(nodes, parents, cache)
        assert cache.pos == prompt and logits.shape == (B, N, 256)
        exact = _exact(model)
        parts = []
        for n in sorted({0, N - 1, N // 2, N // 3}):
            whole = torch.cat([ids, nodes[:, _path(parents, n)]], dim=1)
            parts.append((logits[:, n], model(whole)[0][:, -1], exact(whole)[0][:, -1]))
        assert _near(dtype, *(torch.stack([p[i] for p in parts]) for i in range(3)))


@pytest.mark.parametrize("per_row", [False, True])
def test_keep_goes_on_with_a_path(dev, per_row):
    model = _gpt(dev)
    B, prompt, N = 2, 30, 10
    parents = [-1, 0, 0, 1, 2, 4, -1, 6, 7, 5]
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 256, (B, prompt), generator=g).to(dev)
    nodes = torch.randint(0, 256, (B, N), generator=g).to(dev)
    paths = [[0, 2, 4], [6, 7, 8]] if per_row else [[0, 2, 4]] * B
    with torch.inference_mode():
        cache = KVCache(B, 4, prompt + N + 4, 16, 2)
        model(ids, kv_cache=cache)
        model.forward_tree(nodes, parents, cache)
        cache.keep(paths if per_row else paths[0])
        assert cache.pos == prompt + 3
        nxt = torch.randint(0, 256, (B, 1), generator=g).to(dev)
        got = model(nxt, kv_cache=cache)[0][:, -1]
        kept = torch.stack([nodes[b, p] for b, p in enumerate(paths)])
        want = model(torch.cat([ids, kept, nxt], dim=1))[0][:, -1]
        assert bool(((got - want).abs() <= TOL[torch.float32]).all())
        with pytest.raises(AssertionError, match="no tree"):
            cache.keep([0])


def test_a_tree_leaves_the_cache_as_it_was(dev):
    """Without keep, the next append takes the tree's place; a cache that must grow does."""
    model = _gpt(dev)
    ids = torch.tensor([_series([20], 256)[0]], device=dev)
    with torch.inference_mode():
        cache, plain = KVCache(1, 4, 21, 16, 2), KVCache(1, 4, 64, 16, 2)
        for c in (cache, plain):
            model(ids, kv_cache=c)
        model.forward_tree(torch.arange(9, device=dev)[None], [-1, 0, 1, 0, 3, -1, 5, 6, 7], cache)
        a = model(ids[:, :1], kv_cache=cache)[0]
        b = model(ids[:, :1], kv_cache=plain)[0]
        # the decode step splits its keys by the cache's capacity: other sums, not other keys
        assert bool(((a - b).abs() <= TOL[torch.float32]).all())
        with pytest.raises(AssertionError, match="no tree"):
            cache.keep([0])


def test_tree_and_keep_over_a_shared_prefix(dev):
    """Rows that share their prompt's cache (KVCache.prefill)."""
    model = _gpt(dev)
    ids = torch.tensor([_series([40], 256, seed=5)[0]], device=dev)
    rows = 5
    g = torch.Generator().manual_seed(6)
    nodes = torch.randint(0, 256, (rows, 6), generator=g).to(dev)
    parents = [-1, 0, 1, 0, 3, 4]
    with torch.inference_mode():
        prompt, cache = KVCache(1, 4, 40, 16, 2), KVCache(rows, 4, 60, 16, 2)
        model(ids, kv_cache=prompt)
        cache.prefill(prompt)
        logits = model.forward_tree(nodes, parents, cache)
        path = [0, 3, 4, 5]
        whole = torch.cat([ids.expand(rows, -1), nodes[:, path]], dim=1)
        want = model(whole)[0]
        assert bool(((logits[:, path] - want[:, -4:]).abs() <= TOL[torch.float32]).all())
        cache.keep(path)
        nxt = torch.randint(0, 256, (rows, 1), generator=g).to(dev)
        got = model(nxt, kv_cache=cache)[0][:, -1]
        want = model(torch.cat([whole, nxt], dim=1))[0][:, -1]
        assert bool(((got - want).abs() <= TOL[torch.float32]).all())


def test_a_tree_behind_an_empty_cache(dev):
    """No cached position: the roots see themselves alone, as a first token does."""
    model = _gpt(dev)
    nodes = torch.tensor([[5, 9, 7, 200]], device=dev)
    with torch.inference_mode():
        cache = KVCache(1, 4, 16, 16, 2)
        logits = model.forward_tree(nodes, [-1, 0, -1, 2], cache)
        for path in ([0, 1], [2, 3]):
            want = model(nodes[:, path])[0]
            assert bool(((logits[:, path] - want).abs() <= TOL[torch.float32]).all())
        cache.keep([2, 3])
        got = model(nodes[:, :1], kv_cache=cache)[0][:, -1]
        want = model(nodes[:, [2, 3, 0]])[0][:, -1]
        assert bool(((got - want).abs() <= TOL[torch.float32]).all())


def test_tree_refusals(dev):
    model = _gpt(dev)
    ids = torch.tensor([_series([20], 256)[0]], device=dev)
    nodes = torch.zeros(1, 3, dtype=torch.long, device=dev)
    with torch.inference_mode():
        cache = KVCache(1, 4, 60, 16, 2)
        model(ids, kv_cache=cache)
        with pytest.raises(ValueError, match="parent"):
            model.forward_tree(nodes, [-1, 2, 0], cache)
        with pytest.raises(AssertionError, match="parents"):
            model.forward_tree(nodes, [-1, 0], cache)
        with pytest.raises(AssertionError, match="rows"):
            model.forward_tree(nodes.expand(2, -1), [-1, 0, 1], cache)
        with pytest.raises(AssertionError, match="no tree"):
            cache.keep([0])
        model.forward_tree(nodes, [-1, 0, 0], cache)
        for bad in ([1], [0, 1, 2], [3], [[0], [0]], [[0], [0, 1]]):
            with pytest.raises(AssertionError):
                cache.keep(bad)
        cache.keep([0, 2])
        long = KVCache(1, 4, 276, 16, 2)
        model(torch.zeros(1, 275, dtype=torch.long, device=dev), kv_cache=long)
        with pytest.raises(AssertionError, match="deeper"):
            model.forward_tree(nodes[:, :2], [-1, 0], long)
        model.forward_tree(nodes, [-1, -1, -1], long)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_score_continuations(dev, dtype):
    model = _gpt(dev, dtype)
    prompt = _series([50], 256, seed=7)[0]
    some = _series([5, 1, 9, 65, 30, 2], 256, seed=8)
    some += [some[2][:4] + [7], some[2], some[3][:40] + [1, 2, 3], some[0][:1]]
    got = Engine(model).score_continuations(prompt, some)
    exact = _exact(model)
    parts = []
    with torch.inference_mode():
        for c, lp in zip(some, got):
            assert len(lp) == len(c)
            ids = torch.tensor([prompt + c], device=dev)
            rows = [torch.tensor(lp, dtype=torch.float64, device=dev)]
            for m in (model, exact):
                logs = torch.log_softmax(m(ids)[0][0].double(), dim=-1)
                rows.append(logs[len(prompt) - 1 : -1].gather(-1, ids[0, len(prompt) :, None])[:, 0])
            parts.append(rows)
    assert _near(dtype, *(torch.cat([p[i] for p in parts]) for i in range(3)))


def test_score_continuations_refusals(dev):
    engine = Engine(_gpt(dev))
    for prompt, some in (([], [[1]]), ([1], []), ([1], [[]]), ([1], [[0] * 66]), ([1], [[256]]), ([1] * 270, [[1] * 8])):
        with pytest.raises(AssertionError):
            engine.score_continuations(prompt, some)


def test_tries_cover_every_token_in_groups():
    from diff_gpt.model.engine import _tries

    some = _series([65, 65, 3, 1, 20, 40, 64], 3, seed=9) + [[0], [0, 0], [0, 0, 0]]
    seen = set()
    for group, nodes, parents, places in _tries(some):
        assert len(nodes) == len(parents) <= 64 and all(p < n for n, p in enumerate(parents))
        for c in group:
            assert len(places[c]) == len(some[c])
            for i, p in enumerate(places[c]):
                assert [nodes[n] for n in _path(parents, p)] == some[c][:i]
            seen.add(c)
    assert seen == set(range(len(some)))


def test_anomaly_scores_batch(dev):
    model = _gpt(dev)
    rng = np.random.default_rng(0)
    dgpt = DiffGPT(model=model, order_of_derivative=1, domain_of_definition=np.array([1.0]), use_decimal=False)
    dfs = [pd.DataFrame({"x": np.cumsum(rng.normal(size=n))}) for n in (40, 2, 100, 139, 1)]
    got = dgpt.anomaly_scores_batch(dfs)
    assert len(got) == len(dfs)
    for df, s in zip(dfs, got):
        assert s.shape == df.shape and list(s.columns) == list(df.columns)
        if len(df) > 1:
            want = dgpt.anomaly_scores(df).to_numpy()
            assert np.array_equal(np.isnan(s.to_numpy()), np.isnan(want))
            assert np.nanmax(np.abs(s.to_numpy() - want), initial=0.0) <= TOL[torch.float32]
        else:
            assert np.isnan(s.to_numpy()).all()
    with pytest.raises(AssertionError):
        dgpt.anomaly_scores_batch([])
    with pytest.raises(AssertionError):
        dgpt.anomaly_scores_batch([pd.DataFrame({"x": rng.normal(size=200)})])


def test_trees_seen_by_masks_are_paths():
    """The tests' own two readings of a tree agree."""
    parents = some_tree(40, seed=1)
    seen = tree_seen(parents)
    for n in range(40):
        assert seen[n].nonzero()[:, 0].tolist() == sorted(_path(parents, n))
