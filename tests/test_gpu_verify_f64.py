"""Verification of drafts from float64 logits, decided in float64 throughout."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(dev, B, N, V, seed, scale=4.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    target = torch.randn(B, N + 1, V, generator=g, device=dev, dtype=torch.float64) * scale
    draft = target[:, :N] + 0.05 * torch.randn(B, N, V, generator=g, device=dev, dtype=torch.float64)
    tokens = (torch.softmax(draft, -1) / torch.empty_like(draft).exponential_(generator=g)).argmax(-1)
    uniforms = torch.rand(B, N, generator=g, device=dev)
    noise = torch.empty(B, V, device=dev).exponential_(generator=g)
    return target, draft, tokens, uniforms, noise


def _logs(x):
    """Log softmax in 64 bits on the host, whose sums are pairwise."""
    x = x.cpu()
    top = x.amax(-1, keepdim=True)
    return x - top - torch.exp(x - top).sum(-1, keepdim=True).log()


def _lps_close(got, want):
    # rounded once to fp32, beside float64's own sums
    return bool(((got.double().cpu() - want).abs() <= 2.0**-24 * want.abs() + 1e-11).all())


@pytest.mark.parametrize("N,V", [(0, 1), (1, 7), (3, 500), (2, 5001), (4, 50001), (1, 131072)])
@pytest.mark.parametrize("certain,T", [(False, 1.0), (True, 0.7), (False, 2.5)])
def test_against_64_bits(dev, N, V, certain, T):
    from diff_gpt.sampler.drafts import verify_drafts

    B = 5
    target, draft, tokens, uniforms, noise = _inputs(dev, B, N, V, V)
    r = verify_drafts(target, tokens, uniforms, noise, draft=None if certain else draft, temperature=T)
    p, q = _logs(target / T), _logs(draft / T)
    for b in range(B):
        x, u, e = tokens[b].tolist(), uniforms[b].double().cpu(), noise[b].double().cpu()
        i = 0
        while i < N and float(u[i]) * (1.0 if certain else float(q[b, i, x[i]].exp())) < float(p[b, i, x[i]].exp()):
            i += 1
        rest = p[b, i].exp()
        if i < N:
            if certain:
                rest[x[i]] = 0
            else:
                rest = (rest - q[b, i].exp()).clamp(min=0)
        t = int((rest / e).argmax())
        assert int(r.accepted[b]) == i
        assert r.tokens[b].tolist() == x[:i] + [t] + [-1] * (N - i)
        assert _lps_close(r.logprobs[b, : i + 1], torch.stack([p[b, j, k] for j, k in enumerate(x[:i] + [t])]))


@pytest.mark.parametrize("V", [300, 40000])
def test_first_maxima_that_fp32_takes_for_equal(dev, V):
    """At temperature 0 the largest logit is the token, by however little, and the first of equal ones."""
    from diff_gpt.sampler.drafts import verify_drafts

    g = torch.Generator(device=dev).manual_seed(0)
    target = 10.0 + 1e-12 * torch.randint(0, 1000, (4, 3, V), generator=g, device=dev).double()
    at = torch.randint(0, V, (4, 3), generator=g, device=dev)
    target.scatter_(-1, at[..., None], 10.0 + 2e-9)
    target[3] = 10.0
    at[3] = 0
    r = verify_drafts(target, at[:, :2].contiguous(), temperature=0)
    assert r.accepted.tolist() == [2] * 4 and torch.equal(r.tokens, at)
    assert _lps_close(r.logprobs, _logs(target).gather(-1, at.cpu()[..., None])[..., 0])


@pytest.mark.parametrize("V", [300, 40000])
def test_borders_that_fp32_does_not_tell_apart(dev, V):
    """u against p of a certain draft: a half step of fp32 of p below it stands, above it does not."""
    from diff_gpt.sampler.drafts import verify_drafts

    B = 64
    target, _, _, _, noise = _inputs(dev, B, 1, V, 3, scale=1.0)
    tokens = target[:, :1].argmax(-1)
    p = _logs(target[:, 0]).exp().gather(-1, tokens.cpu())
    u = p.float()
    r = verify_drafts(target, tokens, u.to(dev), noise)
    assert r.accepted.tolist() == (u.double() < p)[:, 0].int().tolist()


@pytest.mark.parametrize("V", [300, 40000])
def test_logits_that_fp32_does_not_hold(dev, V):
    """Logits past fp32's largest, and apart by less than its smallest."""
    from diff_gpt.sampler.drafts import verify_drafts

    B = 3
    target, _, _, _, noise = _inputs(dev, B, 1, V, 5)
    tokens = target[:, :1].argmax(-1)
    zeros = torch.zeros(B, 1, device=dev)
    far = target.clone()
    far[0] -= 1e15
    far[1] = -1e300
    far[1, :, 7] = 1e300
    tokens[1] = 7
    far[2] = 0.0
    far[2, :, 5] = 1e-60
    tokens[2] = 5
    r = verify_drafts(far, tokens, zeros, noise)
    assert r.accepted.tolist() == [1, 1, 1] and int(r.tokens[1, 1]) == 7
    assert _lps_close(r.logprobs[:, 0], _logs(far[:, 0]).gather(-1, tokens.cpu())[:, 0])
    r = verify_drafts(far, tokens, temperature=0)
    assert r.accepted.tolist() == [1, 1, 1] and r.tokens[1:, 0].tolist() == [7, 5]


def test_nan_and_infinities(dev):
    from diff_gpt.sampler.drafts import verify_drafts

    for V in (100, 40000):
        target, draft, tokens, uniforms, noise = _inputs(dev, 5, 2, V, 2)
        target[:, :, V // 2 :] = float("-inf")
        tokens = tokens % (V // 3)
        target[0, 0, 3], target[1, 0, 3], target[2, 0], draft[3, 0, 1] = float("nan"), float("inf"), float("-inf"), float("nan")
        for T in (1.0, 0.8, 0):
            r = verify_drafts(target, tokens, uniforms, noise, draft=draft, temperature=T)
            assert r.accepted[: 4 if T else 3].tolist() == [0] * (4 if T else 3)
            assert bool(((r.tokens >= -1) & (r.tokens < V)).all()) and bool((r.tokens[:, 0] >= 0).all())


def test_captured_calls_replay(dev):
    from diff_gpt.sampler.drafts import verify_drafts

    for V in (300, 30000):
        state = _inputs(dev, 3, 3, V, 8)
        target, draft, tokens, uniforms, noise = state
        verify_drafts(target, tokens, uniforms, noise, draft=draft)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = verify_drafts(target, tokens, uniforms, noise, draft=draft)
        for i in range(3):
            for x, y in zip(state, _inputs(dev, 3, 3, V, 20 + i)):
                x.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            eager = verify_drafts(target, tokens, uniforms, noise, draft=draft)
            assert all(torch.equal(a, b) for a, b in zip(r, eager))
