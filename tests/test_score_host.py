"""Refusals and bookkeeping of the scoring paths through the model, without a GPU."""

import numpy as np
import pandas as pd
import pytest
import torch

from diff_gpt.diff_gpt import DiffGPT
from diff_gpt.model.engine import Engine
from diff_gpt.model.gpt import GPT, BaseGPT
from diff_gpt.model.kv_cache import KVCache
from diff_gpt.model.packed import PackedLayout
from diff_gpt.model.tree import tree_depths, tree_masks


class _Other(BaseGPT):
    """A model that has neither GPT's score nor its forward_tree."""

    def __init__(self):
        super().__init__(block_size=16, vocab_size=64, n_embd=8, n_head=2, n_layer=1)
        self.forwards = 0

    def forward(self, idx, targets=None, kv_cache=None):
        self.forwards += 1
        return torch.zeros(*idx.shape, self.vocab_size), None

    def generate(self, idx, max_new_tokens, sampler, seed=None):
        raise NotImplementedError

    @property
    def device_type(self):
        return "cpu"


@pytest.mark.parametrize("continuations", [[[1]], [[1, 2], [1, 3]]])
def test_continuations_of_a_model_without_trees(continuations):
    model = _Other()
    with pytest.raises(TypeError, match="forward_tree"):
        Engine(model).score_continuations([1, 2, 3], continuations)
    assert model.forwards == 0


def test_frames_of_a_model_without_score():
    dgpt = DiffGPT(model=_Other(), order_of_derivative=1, domain_of_definition=np.array([1.0]), use_decimal=False)
    with pytest.raises(TypeError, match="score"):
        dgpt.anomaly_scores_batch([pd.DataFrame({"x": np.arange(8.0)})])


class _Refuses(_Other):
    def score(self, sequences):
        assert not self.training
        raise MemoryError("no room for the logits")


@pytest.mark.parametrize("training", [True, False])
def test_a_failed_batch_leaves_the_models_mode(training):
    model = _Refuses().train(training)
    dgpt = DiffGPT(model=model, order_of_derivative=1, domain_of_definition=np.array([1.0]), use_decimal=False)
    with pytest.raises(MemoryError):
        dgpt.anomaly_scores_batch([pd.DataFrame({"x": np.arange(8.0)})])
    assert model.training is training


def test_keep_where_the_tree_does_not_lie():
    """A cache whose position was set back (or on) after the tree ran: its next places hold
    something else."""
    cache = KVCache(batch_size=1, num_heads=1, seq_len=16, head_dim=4, num_layers=1)
    cache.pos = cache.tree_start = 5
    cache.tree = [-1, 0, 1]
    for pos in (3, 6):
        cache.pos = pos
        with pytest.raises(AssertionError, match="behind position 5"):
            cache.keep([0, 1])
    cache.pos = 5
    cache.keep([0, 1])
    assert cache.pos == 7 and cache.tree is None


def test_numbers_that_are_not_whole_are_refused():
    """Never cut to whole ones: a token of 1.7 is not token 1."""
    model = GPT(vocab_size=64, n_embd=8, block_size=8, n_head=2, n_layer=1)
    with pytest.raises(TypeError):
        model.score([[1, 1.7]])
    with pytest.raises(TypeError):
        PackedLayout([3, 2.5])
    with pytest.raises(TypeError):
        PackedLayout([3], [3.5])
    with pytest.raises(TypeError):
        PackedLayout([3], group=1.5)
    for parents in ([-1, 0.5], [-0.5]):
        with pytest.raises(TypeError):
            tree_masks(parents, device="cpu")
        with pytest.raises(TypeError):
            tree_depths(parents)
    assert tree_depths(np.array([-1, 0, 0])) == tree_depths(torch.tensor([-1, 0, 0])) == [0, 1, 1]
