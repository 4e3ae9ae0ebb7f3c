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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_anomaly_scores_batch_in_every_type(dev, dtype):
    """Against the fp64 model of the same weights, beside the model's plain forward over one
    frame at a time: a batch's scores are at most as far off in the root mean square (1.5
    times, as for the plain forwards elsewhere), fp32 within 2e-4 of the exact ones."""
    model = _gpt(dev, dtype)
    exact = copy.deepcopy(model).double()
    rng = np.random.default_rng(1)
    dfs = [pd.DataFrame({"x": np.cumsum(rng.normal(size=n)), "y": rng.normal(size=n)}) for n in (30, 5, 60, 69, 2)]
    kw = dict(order_of_derivative=1, domain_of_definition=np.array([1.0, 1.0]), use_decimal=False)
    got = DiffGPT(model=model, **kw).anomaly_scores_batch(dfs)
    off, off_single = [], []
    for df, s in zip(dfs, got):
        want = DiffGPT(model=exact, **kw).anomaly_scores(df).to_numpy()
        s = s.to_numpy()
        assert np.array_equal(np.isnan(s), np.isnan(want))
        want = want[~np.isnan(want)]
        off.append(s[~np.isnan(s)] - want)
        tokens = DiffGPT(model=model, **kw)._encode_frame(df)[2].reshape(1, -1).astype(np.int64)
        tokens = torch.from_numpy(tokens).to(dev)
        with torch.inference_mode():
            logs = torch.log_softmax(model(tokens)[0][0, :-1].double(), dim=-1)
        off_single.append(-logs.gather(-1, tokens[0, 1:, None])[:, 0].cpu().numpy() - want)
    off, off_single = np.concatenate(off), np.concatenate(off_single)
    if dtype == torch.float32:
        assert np.abs(off).max() <= 2e-4
    else:
        assert np.sqrt((off**2).mean()) <= 1.5 * np.sqrt((off_single**2).mean())
