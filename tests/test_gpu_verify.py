"""Verification of drafted tokens against the same decisions in 64 bits."""

import pytest
import torch

from seq_cases import HALF, TDT

pytestmark = pytest.mark.gpu


def _inputs(dev, dtype, B, N, V, seed, near=0.05, scale=0.3, T=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    raw = torch.randn(B, N + 1, V, generator=g, device=dev) * scale
    target = (15 * torch.tanh(raw)).to(TDT[dtype])
    draft = (15 * torch.tanh(raw[:, :N] + near * torch.randn(B, N, V, generator=g, device=dev))).to(TDT[dtype])
    race = torch.empty(B, N, V, device=dev).exponential_(generator=g)
    tokens = (torch.softmax(draft.float() / T, -1) / race).argmax(-1)
    uniforms = torch.rand(B, N, generator=g, device=dev)
    noise = torch.empty(B, V, device=dev).exponential_(generator=g)
    return target, draft, tokens, uniforms, noise


def _exact(target, tokens, uniforms, noise, draft, counts, T):
    B, N = tokens.shape
    acc, out, lps = [], torch.full((B, N + 1), -1), torch.zeros(B, N + 1, dtype=torch.float64)
    for b in range(B):
        p = torch.softmax(target[b].double().cpu() / T, -1)
        q = None if draft is None else torch.softmax(draft[b].double().cpu() / T, -1)
        u, e, x = uniforms[b].double().cpu(), noise[b].double().cpu(), tokens[b].tolist()
        i = 0
        while i < counts[b]:
            inside = 0 <= x[i] < p.size(1)
            qx = 1.0 if q is None else float(q[i, x[i]]) if inside else 1.0
            if not (inside and float(u[i]) * qx < float(p[i, x[i]])):
                break
            out[b, i], lps[b, i] = x[i], p[i, x[i]].log()
            i += 1
        r = p[i].clone()
        if i < counts[b]:
            if q is not None:
                r = (p[i] - q[i]).clamp(min=0)
            elif 0 <= x[i] < p.size(1):
                r[x[i]] = 0
            if not bool((r > 0).any()):
                r = p[i]
        t = int((r / e).argmax())
        out[b, i], lps[b, i] = t, p[i, t].log()
        acc.append(i)
    return torch.tensor(acc), out, lps


def _check(r, want, dtype_tol=2e-6):
    acc, out, lps = want
    assert r.accepted.tolist() == acc.tolist()
    assert r.tokens.tolist() == out.tolist()
    # log p = z - log(sum): z exact to half a step of up to 30 nats, the sum to a few of 1
    assert bool(((r.logprobs.double().cpu() - lps).abs() <= dtype_tol + 2.0**-24 * lps.abs()).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("B,N,V", [(1, 0, 1), (3, 0, 77), (1, 1, 2), (5, 4, 64), (33, 4, 256), (7, 64, 40), (4, 5, 4099),
                                   (2, 3, 50001), (1, 8, 131072), (70, 2, 9001), (3, 64, 2000)])
@pytest.mark.parametrize("certain,T", [(False, 1.0), (True, 0.8), (False, 1.7)])
def test_against_64_bits(dev, dtype, B, N, V, certain, T):
    from diff_gpt.sampler.drafts import verify_drafts

    target, draft, tokens, uniforms, noise = _inputs(dev, dtype, B, N, V, B + N + V, T=T)
    if certain:
        draft = None
        tokens = torch.where(torch.arange(N, device=dev) % 2 == 0, target[:, :N].argmax(-1), tokens)
    counts = [(3 * b) % (N + 1) if b else N for b in range(B)]
    n = torch.tensor(counts, dtype=torch.int32, device=dev)
    r = verify_drafts(target, tokens, uniforms, noise, draft=draft, counts=n, temperature=T)
    _check(r, _exact(target, tokens, uniforms, noise, draft, counts, T))


def test_rows_that_start_anywhere(dev):
    from diff_gpt.sampler.drafts import verify_drafts

    for off in (1, 2, 3, 5, 7):
        B, N, V = 3, 4, 3001
        target, draft, tokens, uniforms, noise = _inputs(dev, "bf16", B, N, V, off)
        wide = torch.full((B, N + 1, V + 11), float("nan"), device=dev, dtype=torch.bfloat16)
        at = wide[..., off : off + V]
        at.copy_(target)
        loud = torch.full((B, V + 3), 1e-30, device=dev)[:, 1 : V + 1]
        loud.copy_(noise)
        r = verify_drafts(at, tokens, uniforms, loud, draft=draft.transpose(0, 1).contiguous().transpose(0, 1))
        _check(r, _exact(target, tokens, uniforms, noise, draft, [N] * B, 1.0))


@pytest.mark.parametrize("V", [100, 40000])
def test_borders(dev, V):
    """Drafts that must and must not stand, and what is left of equal distributions."""
    from diff_gpt.sampler.drafts import verify_drafts

    target, draft, tokens, uniforms, noise = _inputs(dev, "f32", 4, 3, V, 1)
    same = target[:, :3].contiguous()
    r = verify_drafts(target, tokens, torch.full_like(uniforms, 1 - 2.0**-24), noise, draft=same)
    assert r.accepted.tolist() == [3] * 4  # u q < p for p = q
    # a draft outside the vocabulary, and one whose probability is 0, do not stand
    bad = tokens.clone()
    bad[0, 1], bad[1, 0] = -1, V
    bad[2, 2] = 5
    hidden = target.clone()
    hidden[2, 2, 5] = float("-inf")
    r = verify_drafts(hidden, bad, torch.zeros_like(uniforms), noise, draft=same)
    assert r.accepted.tolist() == [1, 0, 2, 3]
    assert bool(((r.tokens >= -1) & (r.tokens < V)).all())
    # rejected by a draft distribution that equals the target's: the target's own draw
    want = (torch.softmax(target[0, 1].double(), -1) / noise[0].double()).argmax()
    assert int(r.tokens[0, 1]) == int(want)


@pytest.mark.parametrize("V", [100, 40000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_hidden_tokens_and_broken_rows(dev, V, dtype):
    """-inf logits are never drawn; rows of NaN, +inf or -inf alone end in a token of the vocabulary."""
    from diff_gpt.sampler.drafts import verify_drafts

    target, draft, tokens, uniforms, noise = _inputs(dev, dtype, 6, 2, V, 2)
    target[:, :, V // 2 :] = float("-inf")
    draft[:, :, V // 3 :] = float("-inf")
    tokens = tokens % (V // 3)
    for T in (1.0, 0.8):
        r = verify_drafts(target, tokens, uniforms, noise, draft=draft, temperature=T)
        _check(r, _exact(target, tokens, uniforms, noise, draft, [2] * 6, T))
    target[0, 0, 3], target[1, 0, 3], target[2, 0] = float("nan"), float("inf"), float("-inf")
    draft[3, 0, 1] = float("nan")
    r = verify_drafts(target, tokens, uniforms, noise, draft=draft)
    assert r.accepted[:4].tolist() == [0, 0, 0, 0]
    assert bool(((r.tokens >= -1) & (r.tokens < V)).all()) and bool((r.tokens[:4, 0] >= 0).all())
    want = _exact(target[4:], tokens[4:], uniforms[4:], noise[4:], draft[4:], [2] * 2, 1.0)
    assert r.accepted[4:].tolist() == want[0].tolist() and r.tokens[4:].tolist() == want[1].tolist()


@pytest.mark.parametrize("V", [100, 40000])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f64"])
@pytest.mark.parametrize("at", [0, 37, -1])
def test_nan_among_hidden_tokens(dev, V, dtype, at):
    """A NaN breaks its row wherever it stands, among tokens that are all hidden too, and no draft
    of a broken row stands, at temperature 0 neither."""
    from diff_gpt.sampler.drafts import verify_drafts

    target, _, _, uniforms, noise = _inputs(dev, dtype, 2, 1, V, 4)
    target[:, :, : V // 2] = float("-inf")
    tokens = target[:, :1].argmax(-1)
    lone = torch.arange(V, device=dev) != tokens[0, 0]
    target[0, 0, lone] = float("-inf")  # the draft's token alone is left
    for T in (1.0, 0):
        fine = verify_drafts(target, tokens, torch.zeros_like(uniforms), noise, temperature=T)
        assert fine.accepted.tolist() == [1, 1]
        broken = target.clone()
        broken[0, 0, at] = broken[1, 0, at] = float("nan")
        r = verify_drafts(broken, tokens, torch.zeros_like(uniforms), noise, temperature=T)
        assert r.accepted.tolist() == [0, 0]
        assert bool(((r.tokens[:, 0] >= 0) & (r.tokens[:, 0] < V)).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f64"])
@pytest.mark.parametrize("B,N,V", [(3, 4, 200), (5, 3, 33000), (2, 0, 64)])
def test_temperature_zero(dev, dtype, B, N, V):
    from diff_gpt.sampler.drafts import verify_drafts

    target, _, _, _, _ = _inputs(dev, dtype, B, N, V, 3)
    target[:, :, V // 2] = target.amax(-1)  # a tie, of which the earlier id counts
    first = (target == target.amax(-1, keepdim=True)).int().argmax(-1)
    tokens = first[:, :N].clone()
    if N:
        tokens[0, N - 1] = (tokens[0, N - 1] + 1) % V
    counts = torch.tensor([N if b < 2 else max(0, N - 1) for b in range(B)], dtype=torch.int32, device=dev)
    r = verify_drafts(target, tokens, counts=counts, temperature=0)
    for b in range(B):
        a = int(counts[b]) if b or not N else N - 1
        assert int(r.accepted[b]) == a
        assert r.tokens[b].tolist() == first[b, : a + 1].tolist() + [-1] * (N - a)
        lp = torch.log_softmax(target[b].double(), -1).gather(-1, first[b][:, None])[: a + 1, 0]
        assert bool(((r.logprobs[b, : a + 1].double() - lp).abs() <= 2e-6).all())


def test_what_comes_out_is_the_targets_distribution(dev):
    """The first token after a draft is distributed as the target's own draw: 5 deviations of
    200000 draws."""
    from diff_gpt.sampler.drafts import verify_drafts

    B, V = 200000, 8
    g = torch.Generator(device=dev).manual_seed(5)
    p, q = torch.randn(V, generator=g, device=dev), torch.randn(V, generator=g, device=dev)
    tokens = torch.multinomial(torch.softmax(q, -1), B, replacement=True, generator=g)[:, None]
    u = torch.rand(B, 1, generator=g, device=dev)
    e = torch.empty(B, V, device=dev).exponential_(generator=g)
    r = verify_drafts(p.expand(B, 2, V), tokens, u, e, draft=q.expand(B, 1, V))
    share = torch.bincount(r.tokens[:, 0], minlength=V).double() / B
    want = torch.softmax(p.double(), -1)
    assert bool(((share - want).abs() <= 5 * (want * (1 - want) / B).sqrt()).all())


@pytest.mark.parametrize("V", [300, 20000])
def test_captured_calls_replay(dev, V):
    from diff_gpt.sampler.drafts import verify_drafts

    target, draft, tokens, uniforms, noise = _inputs(dev, "bf16", 4, 3, V, 8)
    verify_drafts(target, tokens, uniforms, noise, draft=draft)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = verify_drafts(target, tokens, uniforms, noise, draft=draft)
    for i in range(4):
        for x, y in zip((target, draft, tokens, uniforms, noise), _inputs(dev, "bf16", 4, 3, V, 20 + i)):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        _check(r, _exact(target, tokens, uniforms, noise, draft, [3] * 4, 1.0))
        eager = verify_drafts(target, tokens, uniforms, noise, draft=draft)
        assert all(torch.equal(a, b) for a, b in zip(r, eager))


def test_refusals_of_the_python_entry_point(dev):
    from diff_gpt.sampler.drafts import verify_drafts

    target, draft, tokens, uniforms, noise = _inputs(dev, "f32", 3, 2, 40, 0)
    ok = dict(target=target, tokens=tokens, uniforms=uniforms, noise=noise, draft=draft)
    verify_drafts(**ok)
    for kw in [dict(target=target[0]), dict(target=target[:, :0]), dict(target=target[:, :2]), dict(target=target[..., ::2]),
               dict(tokens=tokens.int()), dict(tokens=tokens[:, :1]), dict(tokens=tokens.t().contiguous().t()), dict(uniforms=None),
               dict(uniforms=uniforms.double()), dict(noise=None), dict(noise=noise[:, :30]), dict(noise=noise.half()),
               dict(noise=noise.cpu()), dict(draft=draft[:, :1]), dict(draft=draft.cpu()), dict(counts=torch.tensor([1, 1, 1])),
               dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e-40),
               dict(target=torch.zeros(1, 66, 4, device=dev), tokens=torch.zeros(1, 65, dtype=torch.long, device=dev), draft=None)]:
        with pytest.raises((ValueError, RuntimeError)):
            verify_drafts(**{**ok, **kw})
    with pytest.raises(TypeError):
        verify_drafts(**{**ok, "draft": draft.half()})
