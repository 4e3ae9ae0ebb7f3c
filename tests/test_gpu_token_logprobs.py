"""Log probabilities of given tokens, entropy and alternatives (dg_logprobs.hip) against
float64."""

import math

import pytest
import torch

from diff_gpt import _native
from diff_gpt.model.token_logprobs import token_logprobs

pytestmark = pytest.mark.gpu
TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "f64": torch.float64}
INF, NAN = float("inf"), float("nan")


def _ranked(x, k):
    """The k first ids in (value descending, id ascending, NaN last) order."""
    y = x.double()
    nan = y.isnan()
    order = torch.sort(torch.where(nan, -INF, y), dim=-1, descending=True, stable=True)[1]
    # NaN rank behind -inf: a second stable sort on "is NaN" keeps the order among the rest
    behind = torch.sort(nan.gather(-1, order).int(), dim=-1, stable=True)[1]
    return order.gather(-1, behind)[:, :k]


def _check(x, ids, r, dtype, top):
    """fp32: log s and x - max are each off by half a step of values up to |lp| + the
    entropy's own (2^-22 of both in all), and the sum of the exponentials by some 4e-6 (its
    terms by 2^-22 each, the chains of the partial sums by less)."""
    z = x.double()
    logs = z - z.amax(-1, keepdim=True)
    logs = logs - logs.exp().sum(-1, keepdim=True).log()
    p = logs.exp()
    lp = logs.gather(-1, ids.clamp(0, x.size(-1) - 1)[:, None])[:, 0]
    h = -torch.where(p == 0, 0.0, p * logs).sum(-1)
    spread = (p * (z.amax(-1, keepdim=True) - z).nan_to_num(0, 0, 0)).sum(-1)
    eps, base = (2.0**-22, 4e-6) if dtype != "f64" else (2.0**-50, 1e-13)
    fine = lambda got, want, tol: bool((((got.double() - want).abs() <= tol) | (got.double() == want)  # noqa: E731
                                        | (got.isnan() & want.isnan())).all())
    assert fine(r.logprobs, lp, base + eps * lp.abs())
    assert fine(r.entropy, h, 2 * base * (1 + spread))
    assert torch.equal(r.top_ids, _ranked(x, top))
    want = logs.gather(-1, r.top_ids)
    assert fine(r.top_logprobs, want, base + eps * want.abs())
    assert r.logprobs.dtype == (torch.float64 if dtype == "f64" else torch.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("M,V", [(1, 1), (3, 2), (5, 63), (7, 64), (4, 65), (33, 256), (9, 257), (130, 1024), (3, 1025),
                                 (6, 4099), (2, 50001), (1, 131072), (3, 65600), (2, 140003), (1, 262149), (1, 524291), (1, 600000)])
@pytest.mark.parametrize("top", [0, 1, 5, 64])
def test_matches_float64(dev, dtype, M, V, top):
    top = min(top, V)
    g = torch.Generator(device=dev).manual_seed(M + V)
    x = (torch.randn(M, V, generator=g, device=dev) * 3).to(TDT[dtype])
    ids = torch.randint(0, V, (M,), generator=g, device=dev)
    _check(x, ids, token_logprobs(x, ids, top), dtype, top)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [64, 256, 1000, 20000, 100003, 300000])
@pytest.mark.parametrize("order", ["ascending", "descending", "equal", "two", "few_finite"])
def test_orders_and_ties(dev, dtype, V, order):
    """Rows sorted either way, of one value, of two, and with all but five logits -inf:
    equal ones come by ascending id."""
    g = torch.Generator(device=dev).manual_seed(V)
    x = torch.randn(3, V, generator=g, device=dev)
    if order == "ascending":
        x = x.sort(-1)[0]
    elif order == "descending":
        x = x.sort(-1, descending=True)[0]
    elif order == "equal":
        x = torch.full_like(x, 0.5)
    elif order == "two":
        x = (x > 1.0).float()
    else:
        keep = torch.zeros_like(x, dtype=torch.bool)
        keep[:, torch.randperm(V, device=dev, generator=g)[:5]] = True
        x = x.masked_fill(~keep, -INF)
    x = x.to(TDT[dtype])
    ids = torch.randint(0, V, (3,), generator=g, device=dev)
    _check(x, ids, token_logprobs(x, ids, 33), dtype, 33)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [256, 5000, 70000, 150001])
def test_rows_that_are_no_distribution(dev, dtype, V):
    """NaN, +inf and -inf alone give NaN; their neighbours are untouched."""
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(7, V, generator=g, device=dev).to(TDT[dtype])
    x[1, V // 2] = NAN
    x[2, 3] = INF
    x[3] = -INF
    x[4, : V // 2] = -INF
    x[5] = NAN
    ids = torch.randint(V // 2, V, (7,), generator=g, device=dev)
    r = token_logprobs(x, ids, 8)
    _check(x, ids, r, dtype, 8)
    bad = torch.tensor([False, True, True, True, False, True, False], device=dev)
    for t in (r.logprobs, r.entropy):
        assert torch.equal(t.isnan(), bad)
    assert torch.equal(r.top_logprobs.isnan().all(-1), bad)


def test_extreme_values(dev):
    """Logits at the type's lowest and highest values, and equal ones of any size."""
    low = torch.finfo(torch.float32).min
    x = torch.tensor([[low, 0.0, 1.0], [low, low, low], [3e38, 1.0, -3e38], [88.0, -88.0, 0.0]], device=dev)
    ids = torch.tensor([0, 1, 0, 2], device=dev)
    r = token_logprobs(x, ids, 3)
    logs = torch.log_softmax(x.double(), dim=-1)
    want = logs.gather(-1, ids[:, None])[:, 0]
    assert bool(((r.logprobs.double() - want).abs() <= 4e-6 + 2.0**-22 * want.abs()).all())
    h = -torch.where(logs.exp() > 0, logs.exp() * logs, 0.0).sum(-1)
    assert bool(((r.entropy.double() - h).abs() <= 1e-5).all())
    assert r.top_ids.tolist() == [[2, 1, 0], [0, 1, 2], [0, 1, 2], [0, 2, 1]]


@pytest.mark.parametrize("V", [3000, 40000, 140000])
def test_extreme_values_in_long_rows(dev, V):
    """Maxima that grow from the type's lowest value to its highest over a row: earlier sums
    vanish, differences overflow."""
    x = (torch.linspace(-1, 1, V, dtype=torch.float64) * 3.4e38).float().to(dev)  # in fp32 the step overflows
    rows = torch.stack([x, x.flip(0), torch.full_like(x, torch.finfo(torch.float32).min), x * 1e-37])
    ids = torch.tensor([V - 1, 0, 7, V - 1], device=dev)
    r = token_logprobs(rows, ids, 3)
    assert r.logprobs[:2].tolist() == [0.0, 0.0] and r.entropy[:2].tolist() == [0.0, 0.0]
    assert r.top_ids.tolist() == [[V - 1, V - 2, V - 3], [0, 1, 2], [0, 1, 2], [V - 1, V - 2, V - 3]]
    assert abs(float(r.logprobs[2]) + math.log(V)) <= 1e-5 and abs(float(r.entropy[2]) - math.log(V)) <= 1e-4
    _check(rows[3:], ids[3:], token_logprobs(rows[3:], ids[3:], 3), "f32", 3)


def test_ids_outside_the_vocabulary(dev):
    x = torch.randn(4, 100, device=dev)
    r = token_logprobs(x, torch.tensor([-1, 100, -100, 2**40], device=dev), 2)
    assert bool(r.logprobs.isnan().all()) and not bool(r.entropy.isnan().any())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_leading_dims(dev, dtype):
    """Rows an odd number of elements apart, and (B, T, V) logits."""
    g = torch.Generator(device=dev).manual_seed(9)
    wide = torch.randn(6, 5, 301, generator=g, device=dev).to(TDT[dtype])
    x = wide[:, :, 1:258]
    ids = torch.randint(0, 257, (6, 5), generator=g, device=dev)
    r = token_logprobs(x, ids, 4)
    assert r.logprobs.shape == (6, 5) and r.top_ids.shape == (6, 5, 4)
    s = token_logprobs(x.contiguous(), ids, 4)
    for a, b in zip(r, s):
        assert torch.equal(a, b)
    none = token_logprobs(x[:0], ids[:0], 4)
    assert none.logprobs.shape == (0, 5) and none.top_ids.shape == (0, 5, 4)


def test_agrees_with_log_softmax(dev):
    """What DiffGPT.anomaly_scores takes from a whole log_softmax."""
    x = torch.randn(50, 256, device=dev) * 5
    ids = torch.randint(0, 256, (50,), device=dev)
    want = torch.log_softmax(x, dim=-1).gather(-1, ids[:, None])[:, 0]
    assert float((token_logprobs(x, ids).logprobs - want).abs().max()) <= 1e-5


def test_replayed(dev):
    x = torch.randn(20, 700, device=dev)
    ids = torch.randint(0, 700, (20,), device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_logprobs(x, ids, 6)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = token_logprobs(x, ids, 6)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(r, token_logprobs(x, ids, 6)):
            assert torch.equal(a, b)


def test_refusals(dev):
    x, ids = torch.randn(4, 100, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="top"):
        token_logprobs(x, ids, 65)
    with pytest.raises(ValueError, match="top"):
        token_logprobs(x[:, :3], ids, 4)
    with pytest.raises(ValueError, match="top"):
        token_logprobs(x, ids, -1)
    with pytest.raises(ValueError, match="ids"):
        token_logprobs(x, ids[:3])
    with pytest.raises(ValueError, match="ids"):
        token_logprobs(x, ids.int())
    with pytest.raises(TypeError):
        token_logprobs(x.int(), ids)
    with pytest.raises(RuntimeError, match="inference-only"):
        token_logprobs(x.requires_grad_(), ids)
    with pytest.raises(ValueError, match="contiguous"):
        _native.token_logprobs_(torch.randn(100, 4, device=dev).t(), ids, torch.empty(4, device=dev), None)
