"""How exact packed and tree attention are: outputs within their own rounding of the 64-bit
ones, whatever the other rows of a tile hold."""

import math

import pytest
import torch

from diff_gpt import _native
from diff_gpt.model.packed import PackedLayout, attention_packed
from diff_gpt.model.tree import attention_tree, tree_masks
from seq_cases import HALF, TDT, attend64, some_tree, tree_seen

pytestmark = pytest.mark.gpu
INF = float("inf")
# A probability's two terms, of 8 (bf16) and 11 (fp16) bits each: the first is cut off
# (2^-7, 2^-10 of it are left), the second off by half a step of that (2^-8) or a whole
# one (2^-10).
TERMS = {"bf16": 2.0**-15, "f16": 2.0**-20}


def _causal(n, t, dev):
    return torch.arange(t, device=dev)[None] <= torch.arange(n, device=dev)[:, None] + (t - n)


def _rounded_once(y, ref, a, dtype, keys, vmax):
    """The output's one rounding beside fp32 arithmetic's 1e-5 of the row's largest sum of
    p |v|, and what two terms leave of the probabilities.  fp16's second term has steps of
    2^-24 beside a largest probability of at least 1."""
    tol = HALF[dtype] * ref.abs() + (1e-5 + TERMS[dtype]) * a.amax(-1, keepdim=True)
    if dtype == "f16":
        tol = tol + keys * 2.0**-24 * vmax + 2.0**-25
    off = (y.double() - ref).abs()
    assert bool((off <= tol).all()), (int((off > tol).sum()), float((off - tol).max()))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [16, 32, 64, 80, 128, 256])
@pytest.mark.parametrize("copies", [1, 4, 24])
def test_packed_is_rounded_once(dev, dtype, D, copies):
    """In each of the three workgroup shapes."""
    q_lens = [130, 5, 64, 200, 1, 128, 33, 300] * copies
    k_lens = [130, 40, 64, 333, 1, 100, 33, 300] * copies
    H = 4
    g = torch.Generator(device=dev).manual_seed(D)
    q, k, v = (torch.randn(n, H, D, generator=g, device=dev).to(TDT[dtype]) for n in (sum(q_lens), sum(k_lens), sum(k_lens)))
    y = attention_packed(q, k, v, PackedLayout(q_lens, k_lens))
    assert _native.last_kernel() == f"seq_mfma_packed_{32 if copies == 1 else 64 if copies == 4 else 128}"
    a = b = 0
    for n, t in list(zip(q_lens, k_lens))[-8:]:
        a, b = a + n, b + t
    a, b = q.size(0) - a, k.size(0) - b
    for n, t in list(zip(q_lens, k_lens))[-8:]:
        ref, mag = attend64(q[a : a + n], k[b : b + t], v[b : b + t], _causal(n, t, dev))
        _rounded_once(y[a : a + n], ref, mag, dtype, t, float(v.abs().max()))
        a, b = a + n, b + t


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("N,G,Tcap", [(1, 4, 900), (31, 1, 200), (24, 4, 7000), (64, 2, 20000)])
def test_trees_are_rounded_once(dev, dtype, D, N, G, Tcap):
    B = 3
    g = torch.Generator(device=dev).manual_seed(N)
    q = torch.randn(B, N, 2 * G, D, generator=g, device=dev).to(TDT[dtype])
    k, v = (torch.randn(B, Tcap, 2, D, generator=g, device=dev).to(TDT[dtype]) for _ in range(2))
    lens = [0, Tcap // 3, Tcap - N]
    parents = some_tree(N, seed=N)
    y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), tree_masks(parents))
    for b, n in enumerate(lens):
        seen = torch.cat([torch.ones(N, n, dtype=torch.bool), tree_seen(parents)], dim=1).to(dev)
        ref, mag = attend64(q[b], k[b, : n + N], v[b, : n + N], seen)
        _rounded_once(y[b], ref, mag, dtype, n + N, float(v.abs().max()))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_infinite_values_of_even_weights(dev, dtype, D):
    """Weights of exactly 1, nothing beyond their leading bits, on infinite values that every
    row of a later tile sees."""
    n = 300
    q, k = (torch.zeros(n, 2, D, dtype=TDT[dtype], device=dev) for _ in range(2))
    v = torch.ones(n, 2, D, dtype=TDT[dtype], device=dev)
    v[5] = INF
    y = attention_packed(q, k, v, PackedLayout([n]))
    assert bool((y[:5] == 1).all()) and bool((y[5:] == INF).all())
    v[5] = -INF
    y = attention_tree(q[None, :9], k[None], v[None], 280)
    assert bool((y == -INF).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("copies,at", [(1, 40), (1, 200), (12, 70), (12, 200), (100, 70), (100, 200)])
def test_a_large_key_leaves_the_rows_that_do_not_see_it(dev, dtype, D, copies, at):
    """A finite key whose scores raise the maximum of the rows that see it by hundreds: the
    other rows of the tile keep their bits."""
    n, H = 256, 2
    g = torch.Generator(device=dev).manual_seed(D + at)
    q, k, v = (torch.randn(copies * n, H, D, generator=g, device=dev).to(TDT[dtype]) for _ in range(3))
    lay = PackedLayout([n] * copies)
    clean = attention_packed(q, k, v, lay)
    k[at::n] = 400 * q[at + 1 :: n].sign()
    y = attention_packed(q, k, v, lay)
    hidden = torch.arange(copies * n, device=dev) % n < at
    assert torch.equal(y[hidden], clean[hidden])
    assert not torch.equal(y[~hidden], clean[~hidden])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,Hkv,G,Tcap", [(20, 2, 1, 200), (64, 4, 2, 1300), (48, 2, 8, 9000)])
def test_a_large_key_of_another_branch(dev, dtype, N, Hkv, G, Tcap):
    """The same of a token that only its own branch of the tree sees."""
    B, D = 40, 64
    g = torch.Generator(device=dev).manual_seed(N)
    q = torch.randn(B, N, Hkv * G, D, generator=g, device=dev).to(TDT[dtype])
    k, v = (torch.randn(B, Tcap, Hkv, D, generator=g, device=dev).to(TDT[dtype]) for _ in range(2))
    lens = torch.tensor([(97 * b) % (Tcap - N) + 1 for b in range(B)], dtype=torch.int32, device=dev)
    masks = tree_masks([-1] + [0, 1] * ((N - 1) // 2) + [0] * ((N - 1) % 2))
    clean = attention_tree(q, k, v, lens, masks)
    for b, n in enumerate(lens.tolist()):
        k[b, n + 1] = 400 * q[b, 1, ::G].sign()  # token 1: seen by itself and those that hang on it
    y = attention_tree(q, k, v, lens, masks)
    hidden = ((masks >> 1) & 1) == 0
    assert torch.equal(y[:, hidden], clean[:, hidden])
    assert not torch.equal(y[:, ~hidden], clean[:, ~hidden])


@pytest.mark.parametrize("D", [16, 64, 128, 40, 65, 256])
@pytest.mark.parametrize("far", [25.05, 24.4, 17.3])
@pytest.mark.parametrize("tree", [True, False])
def test_faint_keys_count_in_a_long_rows_sum(dev, D, far, tree):
    """One key 2^far times as likely as each of 100000 others, in fp32: the others' weights,
    each below the last bit of the row's sum or a little above it, make up 100000 2^-far
    of the one's.  The one's value is held to fp32 attention's 1e-5; the others' is a sum of
    100000 equal terms in fp32, each of whose additions may be off by half a step of the sum
    the same way: 100000 2^-24 of it."""
    n = 100000
    q = torch.zeros(1, 4, 1, D, device=dev)
    q[..., 0] = 1.0
    k = torch.zeros(1, n + 4, 1, D, device=dev)
    k[:, :, :, 0] = -far * math.log(2) * D**0.5
    k[:, 77] = 0.0
    v = torch.zeros(1, n + 4, 1, D, device=dev)
    v[:, 77, :, 0] = 1.0
    v[..., 1] = 1.0
    v[:, 77, :, 1] = 0.0
    if tree:
        y = attention_tree(q, k, v, n, tree_masks([-1] * 4))[0, :, 0]
    else:
        y = attention_packed(q[0], k[0], v[0], PackedLayout([4], [n + 4]))[:, 0]
    for i in range(4):
        others = (n - 1 + (1 if tree else i + 1)) * math.exp(float(k[0, 0, 0, 0].double()) * D**-0.5)
        want = torch.tensor([1 / (1 + others), others / (1 + others)], dtype=torch.float64, device=dev)
        off = (y[i, :2].double() - want).abs().tolist()
        assert off[0] <= 1e-5 and off[1] <= 1e-5 + n * 2.0**-24 * float(want[1]), (y[i, :2].tolist(), want.tolist())
        assert not bool(y[i, 2:].any())


@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("far", [25.05, 24.4, 17.3])
@pytest.mark.parametrize("tree", [True, False])
def test_faint_keys_of_a_long_row_keep_their_weight(dev, D, far, tree):
    """One key 2^far times as likely as each of 100000 others, in fp16: the others' weight
    is 100000 2^-far of its, all of one value.  A weight is off by at most one step of
    fp16's second term, 2^-24 beside a largest one of 2^7: 100000 2^-31 in all, 5e-5; the
    others' value is a sum of 100000 terms in fp32, as above."""
    n = 100000
    q = torch.zeros(1, 4, 1, D, dtype=torch.float16, device=dev)
    q[..., 0] = 16.0
    k = torch.zeros(1, n + 4, 1, D, dtype=torch.float16, device=dev)
    # scores -k far log(2): k's own fp16 rounding moves far alike in the answer
    k[:, :, :, 0] = -far * math.log(2) * D**0.5 / 16.0
    k[:, 77] = 0.0
    v = torch.zeros(1, n + 4, 1, D, dtype=torch.float16, device=dev)
    v[:, 77, :, 0] = 1.0
    v[..., 1] = 1.0
    v[:, 77, :, 1] = 0.0
    if tree:
        y = attention_tree(q, k, v, n, tree_masks([-1] * 4))[0, :, 0]
    else:
        y = attention_packed(q[0], k[0], v[0], PackedLayout([4], [n + 4]))[:, 0]
    s = float(k[0, 0, 0, 0].double()) * 16.0 * D**-0.5
    for i in range(4):
        others = (n - 1 + (1 if tree else i + 1)) * math.exp(s)
        want = torch.tensor([1 / (1 + others), others / (1 + others)], dtype=torch.float64, device=dev)
        tol = 2.0**-11 * want + 5e-5
        tol[1] += n * 2.0**-24 * want[1]
        assert bool(((y[i, :2].double() - want).abs() <= tol).all()), (y[i, :2].tolist(), want.tolist())
        assert not bool(y[i, 2:].any())
