"""Decoding over pages with a model and a draft model of different types."""

import pytest
import torch

from diff_gpt.model.engine import Engine
from diff_gpt.model.gpt import GPT

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
