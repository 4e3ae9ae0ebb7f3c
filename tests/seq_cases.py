"""Inputs and 64-bit answers of the packed and tree attention tests."""

import torch

TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "f64": torch.float64}
# half a step of a rounding, relative to the value
HALF = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11, "f64": 2.0**-53}


def attend64(q, k, v, seen):
    """y (n, H, D) of queries q (n, H, D) over k, v (t, Hkv, D), and the same with |v|:
    what the rounding of a probability is relative to.  seen (n, t)."""
    q, k, v = q.double(), k.double(), v.double()
    H, Hkv, D = q.size(1), k.size(1), q.size(2)
    y, a = torch.zeros_like(q), torch.zeros_like(q)
    some = seen.any(-1)
    if not k.size(0):
        return y, a
    for h in range(H):
        kh, vh = k[:, h // (H // Hkv)].contiguous(), v[:, h // (H // Hkv)].contiguous()
        s = (q[:, h] @ kh.t().contiguous()) * D**-0.5
        # spelled out: torch's fp64 softmax over rows of 3000 is 1e-8 off on the device
        p = torch.exp(s.masked_fill(~seen, float("-inf")) - s.masked_fill(~seen, float("-inf")).amax(-1, keepdim=True))
        p = torch.where(some[:, None], p / p.sum(-1, keepdim=True), 0.0)
        y[:, h], a[:, h] = p @ vh, p @ vh.abs()
    return y, a


def close(y, ref, a, dtype, keys, vmax):
    """The result's rounding, that of the probabilities as 16-bit products take them (half a
    step of each, so of the sum of p |v|; fp16 ones below its normal range, 2^-14, are off by
    up to 2^-25 each beside a largest one of at least 1), and fp32's arithmetic, held to
    1e-5 of the row's largest sum of p |v| as elsewhere for fp32 attention (fp64: 1e-12)."""
    tol = HALF[dtype] * ref.abs()
    row = a.amax(-1, keepdim=True)
    if dtype == "f64":
        tol = tol + 1e-12 * row
    else:
        tol = tol + 1e-5 * row
    if dtype in ("bf16", "f16"):
        tol = tol + HALF[dtype] * a
    if dtype == "f16":
        tol = tol + keys * 2.0**-25 * vmax
        tol = tol + 2.0**-25  # a subnormal result
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((y.double() - ref).abs().max()), bad.nonzero()[:4].tolist())


def tree_seen(parents):
    """(N, N) truth values: token n sees token m."""
    N = len(parents)
    seen = torch.zeros(N, N, dtype=torch.bool)
    for n in range(N):
        m = n
        while m >= 0:
            seen[n, m] = True
            m = parents[m]
    return seen


def some_tree(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [int(torch.randint(max(-1, i - 5), i, (1,), generator=g)) if i else -1 for i in range(n)]
