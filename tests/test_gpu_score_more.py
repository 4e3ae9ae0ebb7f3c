"""More of scoring through the model: its memory, 16-bit models, and trees behind caches
that are larger than their rows."""

import copy

import numpy as np
import pandas as pd
import pytest
import torch

from diff_gpt.diff_gpt import DiffGPT
from diff_gpt.model.gpt import GPT

pytestmark = pytest.mark.gpu


def _gpt(dev, dtype=torch.float32, vocab=256, n_embd=64, n_head=4, n_layer=2, block_size=138):
    torch.manual_seed(0)
    return GPT(vocab_size=vocab, n_embd=n_embd, block_size=block_size, n_head=n_head, n_layer=n_layer).eval().to(dev).to(dtype)


def test_a_large_vocabularys_batches_are_smaller(dev):
    """51200 tokens over 32768 words: 6.7 GB of fp32 logits at once, of which a batch holds 2 GiB."""
    model = _gpt(dev, vocab=32768)
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, 32768, (200,), generator=g).tolist() for _ in range(256)]
    model.score(seqs[:2])
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    got = model.score(seqs)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - held <= 2.3 * 2**30
    # one sequence alone, its sums in other workgroups: fp32 whole-model agreement
    for i in (0, 90, 255):
        alone = model.score([seqs[i]])[0]
        assert bool(((got[i].logprobs - alone.logprobs).abs() <= 2e-4).all())
