"""Many alternatives of a row of logits: rows whose candidates overflow the buffer they are
ranked in (dg_logprobs.hip)."""

import pytest
import torch

from diff_gpt.model.token_logprobs import token_logprobs

pytestmark = pytest.mark.gpu
TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _check(x, ids, top):
    """Ids by value and, where equal, by ascending id; log probabilities within what three
    fp32 operations on numbers of their size and the sum's 4e-6 leave."""
    r = token_logprobs(x, ids, top)
    z = x.double()
    order = torch.sort(z, dim=-1, descending=True, stable=True)[1][:, :top]
    assert torch.equal(r.top_ids, order)
    logs = z - z.amax(-1, keepdim=True)
    logs = logs - logs.exp().sum(-1, keepdim=True).log()
    want = logs.gather(-1, order)
    assert bool(((r.top_logprobs.double() - want).abs() <= 4e-6 + 2.0**-22 * want.abs()).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [257, 320, 448, 511, 512, 1024, 2000, 4096, 4099, 9000, 40000, 70001, 300000])
@pytest.mark.parametrize("top", [48, 64])
def test_rows_of_random_logits(dev, dtype, V, top):
    """With one wave a row (V <= 4096) half of them have more candidates than the buffer's 256."""
    g = torch.Generator(device=dev).manual_seed(V + top)
    M = 64 if V <= 4096 else 4
    x = (torch.randn(M, V, generator=g, device=dev) * 3).to(TDT[dtype])
    _check(x, torch.randint(0, V, (M,), generator=g, device=dev), top)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [300, 1000, 4096, 8000, 50000, 200000])
@pytest.mark.parametrize("shape", ["stairs_up", "stairs_down", "one_lane", "ties_above", "two_steps"])
def test_rows_that_raise_the_bound_slowly(dev, dtype, V, shape):
    """Staircases of ties in either order, rows whose large logits lie in few threads' parts,
    and ties among those that a raised bound leaves."""
    i = torch.arange(V, device=dev)
    if shape == "stairs_up":
        x = (i // 70).float() % 128
    elif shape == "stairs_down":
        x = (V // 70 - i // 70).float() % 128
    elif shape == "one_lane":
        x = torch.where(i % 512 < 8, (i % 97).float(), -1.0 - (i % 3).float())
    elif shape == "ties_above":
        x = torch.where(i % 5 == 0, 3.0, (i % 2).float())
    else:
        x = (i > V // 3).float() + (i > V - 40).float()
    x = x.to(TDT[dtype])[None].repeat(3, 1)
    x[1] = x[1].flip(0)
    for top in (33, 64):
        _check(x, torch.tensor([0, V // 2, V - 1], device=dev), top)


@pytest.mark.parametrize("V", [320, 1024, 4096])
def test_sixty_four_alternatives_cost_no_pass_each(dev, V):
    """64 passes over every row took 14 to 56 times as long as 32 alternatives."""
    x = torch.randn(4096, V, device=dev) * 3
    ids = torch.zeros(4096, dtype=torch.int64, device=dev)

    def fastest(top):
        best = float("inf")
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                token_logprobs(x, ids, top)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert fastest(64) <= 6 * fastest(32)
