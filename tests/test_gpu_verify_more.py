"""Verification of drafts over rows whose sums are hard to come by."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1 << 20, (1 << 20) + 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_rows_keep_their_faint_tokens(dev, V, dtype):
    """A thread has 4096 logits of a row that is not split.  Behind a few loud ones, each four or
    eight of the others are less than half a step of fp32 of what was summed before."""
    from diff_gpt.sampler.drafts import verify_drafts

    B, VE = 171, 16 // torch.empty((), dtype=dtype).element_size()
    low = -6.3125 if dtype == torch.float32 else -6.375
    row = torch.full((V,), low, dtype=torch.float64)
    row[: 256 * VE] = 0.0
    row[256 * VE : 512 * VE] = 11.0
    total = math.log(math.fsum([256 * VE, 256 * VE * math.exp(11.0), (V - 512 * VE) * math.exp(low)]))
    target = row.to(dtype).to(dev).expand(B, 2, V)
    ids = torch.tensor([256 * VE + 1, V - 1, 5], device=dev)[torch.arange(B, device=dev) % 3][:, None].contiguous()
    r = verify_drafts(target, ids, torch.zeros(B, 1, device=dev), torch.ones(1, V, device=dev).expand(B, V))
    assert r.accepted.tolist() == [1] * B
    want = row[ids[:, 0].cpu()] - total
    # the exponent's rounding at 16 log2 units, exp2's and sums of up to 32 in fp32; the result's own
    assert bool(((r.logprobs[:, 0].double().cpu() - want).abs() <= (16 * math.log(2) + 2 + 32) * 2.0**-24 + 2.0**-24 * want.abs()).all())
