"""Packed attention and token trees over a cache (dg_attn_seq.hip, dg_attn_seq_mfma.hip)
against float64 at the lengths, masks and layouts where they can go wrong."""

import pytest
import torch

from diff_gpt import _native
from diff_gpt.model.packed import PackedLayout, attention_packed
from diff_gpt.model.tree import attention_tree, tree_masks
from seq_cases import TDT, attend64, close, some_tree, tree_seen

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _causal(n, t, dev):
    return torch.arange(t, device=dev)[None] <= torch.arange(n, device=dev)[:, None] + (t - n)


def _packed_case(dev, q_lens, k_lens, H, Hkv, D, dt, seed=0, slack=0, scale=1.0):
    """q, k, v as column slices of wider rows (an odd number of columns apart when slack)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    new = lambda n, h: (torch.randn(n, h * D + slack, generator=g, device=dev) * scale).to(dt)  # noqa: E731
    n, t = sum(q_lens), sum(k_lens)
    return (new(n, H)[:, : H * D].view(n, H, D), new(t, Hkv)[:, : Hkv * D].view(t, Hkv, D),
            new(t, Hkv)[:, : Hkv * D].view(t, Hkv, D))


def _check_packed(q, k, v, y, q_lens, k_lens, dtype):
    a = b = 0
    for n, t in zip(q_lens, k_lens):
        if n:
            ref, mag = attend64(q[a : a + n], k[b : b + t], v[b : b + t], _causal(n, t, q.device))
            close(y[a : a + n], ref, mag, dtype, t, float(v.abs().max()) if v.numel() else 0.0)
        a, b = a + n, b + t


LENGTHS = [
    ([1], [1]),
    ([1, 1, 1], [1, 64, 1000]),  # single tokens behind caches of their own length
    ([0, 5, 0], [0, 5, 7]),
    ([31, 32, 33, 64, 65], [31, 32, 33, 64, 65]),
    ([127, 128, 129, 130, 2], [127, 128, 129, 130, 2]),
    ([10, 200, 3], [300, 200, 150]),  # chunks behind cached keys
    ([5, 40], [3, 0]),  # queries that see nothing
    ([700], [701]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 16), (2, 1, 32), (6, 2, 64), (8, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("q_lens,k_lens", LENGTHS)
def test_packed_matches_float64(dev, dtype, H, Hkv, D, q_lens, k_lens):
    q, k, v = _packed_case(dev, q_lens, k_lens, H, Hkv, D, TDT[dtype], seed=D + H)
    y = attention_packed(q, k, v, PackedLayout(q_lens, k_lens, group=H // Hkv))
    _check_packed(q, k, v, y, q_lens, k_lens, dtype)


# lengths that leave a tile's waves unequal work, 14 tiles in all without groups
MIXED = ([130, 5, 64, 200, 1, 128, 33, 300], [130, 40, 64, 333, 1, 100, 33, 300])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 8, 24, 40, 80, 120, 200, 256])
@pytest.mark.parametrize("Hkv,G,copies,rows", [(1, 1, 1, 32), (8, 1, 2, 64), (4, 3, 2, 64), (8, 1, 7, 128), (6, 2, 7, 128)])
def test_packed_in_every_workgroup_shape(dev, dtype, D, Hkv, G, copies, rows):
    """One, two and four 32-row waves a tile, by how many tiles there are."""
    q_lens, k_lens = MIXED[0] * copies, MIXED[1] * copies
    q, k, v = _packed_case(dev, q_lens, k_lens, Hkv * G, Hkv, D, TDT[dtype], seed=copies)
    y = attention_packed(q, k, v, PackedLayout(q_lens, k_lens, group=G))
    assert _native.last_kernel() == ("seq_tile_kernel" if dtype == "f32" and D > 128 else f"seq_mfma_packed_{rows}")
    _check_packed(q, k, v, y, q_lens, k_lens, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 8, 24, 40, 80, 120, 200, 256])
@pytest.mark.parametrize("Hkv,copies,rows", [(1, 1, 32), (8, 2, 64), (8, 7, 128)])
def test_packed_hidden_values_in_every_workgroup_shape(dev, dtype, D, Hkv, copies, rows):
    """NaN keys and infinite and NaN values that some rows of a tile see and others do not:
    bits of the rows that do not are those without them."""
    q_lens, k_lens = MIXED[0] * copies, MIXED[1] * copies
    q, k, v = (x.clone() for x in _packed_case(dev, q_lens, k_lens, Hkv, Hkv, D, TDT[dtype], seed=8))
    lay = PackedLayout(q_lens, k_lens)
    clean = attention_packed(q, k, v, lay)
    kk, vv = k.clone(), v.clone()
    hidden = torch.ones(q.size(0), dtype=torch.bool, device=dev)
    what = torch.zeros(q.size(0), device=dev)
    a = b = 0
    for i, (n, t) in enumerate(zip(q_lens, k_lens)):
        at = (37 * (i + 1)) % t  # the key that is not finite
        first = max(0, at - (t - n))
        vv[b + at] = (INF, -INF, NAN)[i % 3]
        what[a + first : a + n] = (INF, -INF, NAN)[i % 3]
        if i % 4 == 3:
            kk[b + at] = NAN
            what[a + first : a + n] = NAN
        hidden[a + first : a + n] = False
        a, b = a + n, b + t
    y = attention_packed(q, kk, vv, lay)
    assert _native.last_kernel() == ("seq_tile_kernel" if dtype == "f32" and D > 128 else f"seq_mfma_packed_{rows}")
    assert torch.equal(y[hidden], clean[hidden])
    want = what[~hidden][:, None, None].expand_as(y[~hidden])
    got = y[~hidden].float()
    assert bool(((got == want) | (got.isnan() & want.isnan())).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 1), (3, 1, 7), (2, 1, 24), (4, 2, 80), (2, 2, 96), (2, 1, 256), (1, 1, 1000)])
def test_packed_takes_every_head_dim(dev, dtype, H, Hkv, D):
    q_lens, k_lens = [1, 37, 70], [50, 37, 71]
    q, k, v = _packed_case(dev, q_lens, k_lens, H, Hkv, D, TDT[dtype], seed=D)
    y = attention_packed(q, k, v, PackedLayout(q_lens, k_lens, group=H // Hkv))
    _check_packed(q, k, v, y, q_lens, k_lens, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [16, 64, 128])
def test_packed_takes_unaligned_rows(dev, dtype, D):
    """Rows an odd number of elements apart: no 16-byte loads."""
    q_lens = [40, 133]
    q, k, v = _packed_case(dev, q_lens, q_lens, 4, 2, D, TDT[dtype], slack=3)
    y = attention_packed(q, k, v, PackedLayout(q_lens, group=2))
    _check_packed(q, k, v, y, q_lens, q_lens, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 8, 24, 40, 80, 120, 200, 256])
def test_packed_hidden_values_stay_hidden(dev, dtype, D):
    """NaN and infinities in the keys and values of later positions, and in rows behind
    the last sequence, reach no query that does not see them; those that do see an infinite
    value get it."""
    q_lens, k_lens = [50, 70, 5], [50, 90, 40]
    q, k, v = (x.clone() for x in _packed_case(dev, q_lens, k_lens, 2, 2, D, TDT[dtype], seed=3))
    extra = torch.full((9, 2, D), NAN, dtype=k.dtype, device=dev)
    k, v = torch.cat([k, extra]), torch.cat([v, extra])
    clean = attention_packed(q, k, v, PackedLayout(q_lens, k_lens))
    kk, vv = k.clone(), v.clone()
    bad = 50 + 20 + 33  # key 53 of the second sequence: queries 33 .. 69 see it
    kk[bad] = NAN
    vv[bad] = INF
    y = attention_packed(q, kk, vv, PackedLayout(q_lens, k_lens))
    hidden = torch.ones(125, dtype=torch.bool, device=dev)
    hidden[50 + 33 : 120] = False
    assert torch.equal(y[hidden], clean[hidden])
    assert bool(y[~hidden].isnan().all())
    vv[bad] = -INF
    y = attention_packed(q, k, vv, PackedLayout(q_lens, k_lens))
    assert torch.equal(y[hidden], clean[hidden])
    assert bool((y[~hidden] == -INF).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_packed_large_scores_rescale(dev, dtype):
    """Scores that grow to about 200 along the keys: the running maximum is raised block
    after block.  One key takes nearly the whole weight of each row, and the scores' fp32
    rounding, some 16 ulps of 200 (2^-24 * 16 * 200 = 2e-4), moves a probability by as much."""
    D, n = 64, 300
    q, k, v = _packed_case(dev, [n], [n], 2, 2, D, torch.float32, seed=5)
    k = k * torch.linspace(0.1, 10.0, n, device=dev)[:, None, None]
    q, k, v = (x.mul(3.0 if x is q else 1.0).to(TDT[dtype]) for x in (q, k, v))
    y = attention_packed(q, k, v, PackedLayout([n]))
    ref, mag = attend64(q, k, v, _causal(n, n, dev))
    half = {"f32": 0.0, "bf16": 2.0**-8, "f16": 2.0**-11}[dtype]
    tol = 2 * half * mag + 2e-4 * mag.amax(-1, keepdim=True) + (2e-4 if dtype == "f16" else 0)
    assert bool(((y.double() - ref).abs() <= tol).all())


def test_packed_rows_behind_the_last_sequence(dev):
    q, k, v = _packed_case(dev, [100], [100], 2, 2, 64, torch.bfloat16)
    y = torch.full_like(q, 7.0)
    lay = PackedLayout([30, 41])
    _native.attention_packed_(q, k, v, y, lay, 0.125)
    assert bool((y[71:] == 7.0).all())
    z = attention_packed(q, k, v, lay, 0.125)
    assert bool((z[71:] == 0).all()) and torch.equal(z[:71], y[:71])


def test_packed_all_minus_inf_scores(dev):
    """Every visible score -inf: 0 / 0, as a softmax gives; no visible key: zeros."""
    for D in (16, 64, 24):
        q = torch.ones(4, 1, D, device=dev)
        k = torch.full((2, 1, D), -INF, device=dev)
        v = torch.ones(2, 1, D, device=dev)
        y = attention_packed(q, k, v, PackedLayout([4], [2]))
        assert bool((y[:2] == 0).all()) and bool(y[2:].isnan().all())


def test_packed_agrees_with_the_framework_attention(dev):
    """One length, every head its own key head: the operator beside ops.attention."""
    B, T, H, D = 3, 150, 4, 64
    g = torch.Generator(device=dev).manual_seed(1)
    q, k, v = (torch.randn(B, T, H, D, generator=g, device=dev) for _ in range(3))
    y = attention_packed(q.view(-1, H, D), k.view(-1, H, D), v.view(-1, H, D), PackedLayout([T] * B))
    ref = _native.ops().attention(q, k, v, D**-0.5)
    assert float((y.view_as(ref) - ref).abs().max()) <= 2e-5 * float(ref.abs().max())


def test_packed_layout_outlives_another_streams_call(dev):
    """A layout dropped while a call on a stream of its own still waits: its memory is not
    handed on before that call has read it."""
    q, k, v = _packed_case(dev, [700, 300], [700, 300], 2, 2, 64, torch.bfloat16)
    want = attention_packed(q, k, v, PackedLayout([700, 300]))
    torch.cuda.synchronize()
    lay = PackedLayout([700, 300])
    shape, at = lay.tiles.shape, lay.tiles.data_ptr()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(40_000_000)
        y = attention_packed(q, k, v, lay)
    del lay
    other = [torch.zeros(shape, dtype=torch.int32, device=dev) for _ in range(4)]
    assert at not in [t.data_ptr() for t in other]
    side.synchronize()
    assert torch.equal(y, want)


def test_packed_refusals(dev):
    q, k, v = _packed_case(dev, [8], [8], 4, 2, 64, torch.bfloat16)
    lay = PackedLayout([8], group=2)
    with pytest.raises(ValueError, match="groups of 1"):
        attention_packed(q, k, v, PackedLayout([8]))
    with pytest.raises(ValueError, match="covers"):
        attention_packed(q, k, v, PackedLayout([9], group=2))
    with pytest.raises(ValueError, match="covers"):
        attention_packed(q, k, v, PackedLayout([8], [9], group=2))
    with pytest.raises(TypeError):
        attention_packed(q, k.float(), v, lay)
    with pytest.raises(TypeError):
        attention_packed(q.int(), k.int(), v.int(), lay)
    with pytest.raises(ValueError, match="scale"):
        attention_packed(q, k, v, lay, scale=0.0)
    with pytest.raises(ValueError, match="contiguous"):
        attention_packed(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, lay)
    with pytest.raises(ValueError):
        attention_packed(q[None], k[None], v[None], lay)
    with pytest.raises(RuntimeError, match="inference-only"):
        attention_packed(q.float().requires_grad_(), k.float(), v.float(), lay)


def _tree_case(dev, B, N, H, Hkv, Tcap, D, dt, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn(B, N, H, D, generator=g, device=dev).to(dt)
    pages = torch.randn(2, B, Hkv, Tcap, D, generator=g, device=dev).to(dt)
    return q, pages[0].transpose(1, 2), pages[1].transpose(1, 2)


def _check_tree(q, k, v, y, lens, parents, dtype):
    N = q.size(1)
    for b, n in enumerate(lens):
        among = tree_seen(parents if not isinstance(parents[0], list) else parents[b])
        seen = torch.cat([torch.ones(N, n, dtype=torch.bool), among], dim=1).to(q.device)
        ref, mag = attend64(q[b], k[b, : n + N], v[b, : n + N], seen)
        close(y[b], ref, mag, dtype, n + N, float(v[b].float().nan_to_num(0, 0, 0).abs().max()))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 16), (2, 1, 32), (6, 2, 64), (8, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("N,lens,Tcap", [(1, [0, 1, 31, 32, 33], 64), (1, [100, 900, 2000], 2001), (5, [0, 3, 27, 59], 64),
                                         (31, [0, 64, 130], 200), (33, [1, 1000], 1100), (64, [0, 37, 700], 764),
                                         (17, [5000], 6000)])
def test_tree_matches_float64(dev, dtype, H, Hkv, D, N, lens, Tcap):
    q, k, v = _tree_case(dev, len(lens), N, H, Hkv, Tcap, D, TDT[dtype], seed=N + D)
    parents = some_tree(N, seed=N)
    y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), tree_masks(parents))
    assert _native.last_kernel() in ("seq_mfma_tree_32", "seq_mfma_tree_64", "seq_join_kernel")
    _check_tree(q, k, v, y, lens, parents, dtype)


@pytest.mark.parametrize("dtype,D,B,N,Hkv,G,Tcap,rows", [
    ("f32", 16, 2, 60, 1, 3, 70, 32), ("bf16", 32, 3, 40, 2, 2, 300, 32), ("f32", 64, 2, 50, 1, 3, 90, 32),
    ("f32", 128, 2, 50, 2, 3, 100, 64), ("f32", 128, 60, 64, 4, 1, 100, 64), ("bf16", 64, 3, 41, 2, 4, 1000, 32),
    ("f16", 128, 3, 64, 2, 1, 900, 32), ("bf16", 64, 65, 33, 4, 1, 1300, 64), ("f16", 64, 40, 64, 4, 3, 700, 32), ("f16", 64, 40, 64, 4, 3, 1000, 64),
    ("bf16", 128, 64, 50, 4, 3, 700, 64), ("f16", 128, 128, 45, 1, 2, 2500, 128), ("bf16", 64, 250, 37, 1, 3, 1300, 128),
    ("bf16", 56, 65, 33, 4, 1, 1300, 64), ("f16", 96, 128, 45, 1, 2, 2500, 128), ("f32", 100, 60, 64, 4, 1, 100, 64),
    ("f32", 4, 3, 50, 2, 1, 100, 32), ("bf16", 256, 2, 9, 1, 1, 100, 32), ("f16", 136, 64, 50, 4, 3, 700, 64),
    ("bf16", 256, 128, 45, 1, 2, 2500, 128)])
def test_tree_in_every_workgroup_shape(dev, dtype, D, B, N, Hkv, G, Tcap, rows):
    """32, 64 and 128 rows a workgroup, where one takes all of a row's keys."""
    lens = [(131 * (b + 1)) % (Tcap - N + 1) for b in range(B)]
    q, k, v = _tree_case(dev, B, N, Hkv * G, Hkv, Tcap, D, TDT[dtype], seed=B)
    parents = some_tree(N, seed=B)
    y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), tree_masks(parents))
    assert _native.last_kernel() in (f"seq_mfma_tree_{rows}", "seq_join_kernel")
    _check_tree(q, k, v, y, lens, parents, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 8, 24, 40, 80, 120, 200, 256])
@pytest.mark.parametrize("N,G", [(3, 1), (13, 4), (40, 3)])
@pytest.mark.parametrize("B,Tcap", [(1, 60000), (2, 9000)])
def test_tree_splits_meet(dev, dtype, D, N, G, B, Tcap):
    """Rows split over many and over few workgroups, of very different lengths."""
    lens = [Tcap - N, 700][:B]
    q, k, v = _tree_case(dev, B, N, 2 * G, 2, Tcap, D, TDT[dtype], seed=G)
    parents = some_tree(N, seed=2)
    y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), tree_masks(parents))
    assert _native.last_kernel() == "seq_join_kernel"
    _check_tree(q, k, v, y, lens, parents, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 1), (3, 1, 7), (2, 1, 24), (4, 2, 80), (2, 1, 256), (1, 1, 1000)])
def test_tree_takes_every_head_dim(dev, dtype, H, Hkv, D):
    lens, N = [0, 40, 600], 9
    q, k, v = _tree_case(dev, 3, N, H, Hkv, 700, D, TDT[dtype], seed=D)
    parents = some_tree(N)
    y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), tree_masks(parents))
    _check_tree(q, k, v, y, lens, parents, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tree_masks_of_each_row_and_chains(dev, dtype):
    lens, N = [3, 200, 64], 20
    q, k, v = _tree_case(dev, 3, N, 4, 2, 300, 64, TDT[dtype], seed=2)
    trees = [some_tree(N, seed=s) for s in range(3)]
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    y = attention_tree(q, k, v, ln, torch.stack([tree_masks(t) for t in trees]))
    _check_tree(q, k, v, y, lens, trees, dtype)
    y = attention_tree(q, k, v, ln)
    _check_tree(q, k, v, y, lens, list(range(-1, N - 1)), dtype)
    # a cache whose tokens' rows lie head by head (b, t, h, d) and one host length
    kc, vc = k.contiguous(), v.contiguous()
    y = attention_tree(q, kc, vc, 100)
    _check_tree(q, k, v, y, [100] * 3, list(range(-1, N - 1)), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("D", [16, 64, 128, 40, 65, 200, 300])
@pytest.mark.parametrize("Tcap", [128, 3000])
def test_tree_hidden_positions_stay_hidden(dev, dtype, D, Tcap):
    """NaN and infinities behind a row's tokens and in tokens that others do not see;
    empty masks and lengths beyond the cache."""
    B, N, H = 4, 8, 2
    lens = [0, 30, 57, Tcap - N]
    q, k, v = (x.clone() for x in _tree_case(dev, B, N, H, H, Tcap, D, TDT[dtype], seed=4))
    parents = [-1, 0, 0, 1, 1, 2, -1, 6]
    masks = tree_masks(parents)
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    clean = attention_tree(q, k, v, ln, masks)
    _check_tree(q, k, v, clean, lens, parents, dtype)
    for b, n in enumerate(lens):
        k[b, n + N :] = NAN
        v[b, n + N :] = INF
        k[b, n + 2], v[b, n + 2] = NAN, NAN  # token 2: seen by itself and token 5
        v[b, n + 6] = INF  # token 6: seen by itself and token 7
    y = attention_tree(q, k, v, ln, masks)
    same = [0, 1, 3, 4]
    assert torch.equal(y[:, same], clean[:, same])
    assert bool(y[:, [2, 5]].isnan().all()) and bool((y[:, [6, 7]] == INF).all())
    # lengths outside the cache are taken as its ends
    wild = torch.tensor([-5, 30, 57, 2**31 - 1], dtype=torch.int32, device=dev)
    assert torch.equal(attention_tree(q, k, v, wild, masks)[:, same], clean[:, same])
    # tokens that see nothing
    empty = masks.clone()
    empty[4] = 0
    y = attention_tree(q, k, v, ln, empty)
    assert bool((y[0, 4] == 0).all()) and torch.equal(y[:, [0, 1, 3]], clean[:, [0, 1, 3]])
    # bits beyond the tokens mean nothing
    y = attention_tree(q, k, v, ln, masks | (-1 << N))
    assert torch.equal(y[:, same], clean[:, same])


@pytest.mark.parametrize("D", [64, 24])
def test_tree_replayed_with_other_lengths(dev, D):
    """A captured call reads the lengths as they are at each replay, with eager work on the
    same shapes between the replays."""
    B, N, Tcap = 3, 4, 2000
    q, k, v = _tree_case(dev, B, N, 4, 2, Tcap, D, torch.bfloat16, seed=6)
    ln = torch.tensor([10, 20, 30], dtype=torch.int32, device=dev)
    masks = tree_masks([-1, 0, 0, 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_tree(q, k, v, ln, masks)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = attention_tree(q, k, v, ln, masks)
    for lens in ([0, 1500, 7], [1990, 1, 600], [10, 20, 30]):
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, attention_tree(q, k, v, ln, masks))
        _check_tree(q, k, v, got, lens, [-1, 0, 0, 2], "bf16")


def test_packed_replayed(dev):
    q, k, v = _packed_case(dev, [70, 200], [70, 200], 4, 4, 64, torch.bfloat16)
    lay = PackedLayout([70, 200])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_packed(q, k, v, lay)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = attention_packed(q, k, v, lay)
    for s in range(3):
        q.copy_(torch.randn(q.shape, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, attention_packed(q, k, v, lay))


def test_tree_past_32_bit_offsets(dev):
    """A cache page of more than 2^31 elements: the last row's keys lie beyond it."""
    B, Tcap, D = 2, 150000, 128
    big = torch.zeros(B, Tcap, 60, D, dtype=torch.bfloat16, device=dev)  # 2.3e9 elements, 1.15e9 a row
    k = big[:, :, 7:8]
    v = big[:, :, 33:34]
    g = torch.Generator(device=dev).manual_seed(0)
    k.copy_(torch.randn(k.shape, generator=g, device=dev))
    v.copy_(torch.randn(v.shape, generator=g, device=dev))
    q = torch.randn(B, 2, 4, D, generator=g, device=dev).bfloat16()
    lens = [149000, 149998]
    y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev))
    _check_tree(q, k, v, y, lens, [-1, 0], "bf16")
    y = attention_packed(q.view(4, 4, D), k.reshape(-1, 1, D), v.reshape(-1, 1, D),
                         PackedLayout([2, 2], [150000, 150000], group=4))
    _check_packed(q.view(4, 4, D), k.reshape(-1, 1, D), v.reshape(-1, 1, D), y, [2, 2], [150000, 150000], "bf16")
    # the packed rows themselves 60 heads apart
    flat = big.view(B * Tcap, 60, D)
    y2 = attention_packed(q.view(4, 4, D), flat[:, 7:8], flat[:, 33:34],
                          PackedLayout([2, 2], [150000, 150000], group=4))
    assert torch.equal(y, y2)


@pytest.mark.parametrize("D,kernel", [(64, "mfma"), (80, "tile"), (128, "tile")])
@pytest.mark.parametrize("N,G,Tcap", [(1, 1, 100), (2, 4, 100), (1, 3, 1500)])
def test_fp32_steps_of_many_rows(dev, D, kernel, N, G, Tcap):
    lens = [(37 * b) % (Tcap - N + 1) for b in range(33)]
    q, k, v = _tree_case(dev, 33, N, 2 * G, 2, Tcap, D, torch.float32, seed=D)
    parents = some_tree(N, seed=1)
    y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), tree_masks(parents))
    assert _native.last_kernel() == "seq_join_kernel" or kernel in _native.last_kernel()
    _check_tree(q, k, v, y, lens, parents, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("D", [1, 7, 63, 65, 130, 255, 257, 511, 1023, 1024])
@pytest.mark.parametrize("N,G", [(1, 1), (2, 4), (3, 3), (40, 1)])
def test_tree_of_any_shape(dev, dtype, D, N, G):
    """8, 16 and 32 rows a workgroup of the kernel for any head_dim, with splits and without."""
    for Tcap, lens in ((90, [0, 31, 50]), (1500, [1460, 700, 3])):
        q, k, v = _tree_case(dev, 3, N, 2 * G, 2, Tcap, D, TDT[dtype], seed=D)
        parents = some_tree(N, seed=N)
        y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), tree_masks(parents))
        assert _native.last_kernel() in ("seq_tile_kernel", "seq_join_kernel")
        _check_tree(q, k, v, y, lens, parents, dtype)


@pytest.mark.parametrize("dtype,D", [("f32", 16), ("bf16", 64), ("f16", 128), ("bf16", 65), ("f64", 16)])
@pytest.mark.parametrize("G", [33, 130])
def test_wide_groups(dev, dtype, D, G):
    """A query's heads lie in several tiles, and a tile holds parts of two queries' heads."""
    q_lens, k_lens = [1, 5, 3], [70, 5, 300]
    q, k, v = _packed_case(dev, q_lens, k_lens, G, 1, D, TDT[dtype], seed=G)
    _check_packed(q, k, v, attention_packed(q, k, v, PackedLayout(q_lens, k_lens, group=G)), q_lens, k_lens, dtype)
    q, k, v = _tree_case(dev, 2, 3, G, 1, 400, D, TDT[dtype], seed=G)
    parents = [-1, 0, 0]
    y = attention_tree(q, k, v, torch.tensor([0, 397], dtype=torch.int32, device=dev), tree_masks(parents))
    _check_tree(q, k, v, y, [0, 397], parents, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f64"])
@pytest.mark.parametrize("D", [5, 65, 129, 300, 1023])
@pytest.mark.parametrize("q_lens,k_lens", [([1, 3, 0, 2], [70, 3, 9, 1]), ([40, 100, 7], [40, 133, 3])])
def test_packed_of_any_shape(dev, dtype, D, q_lens, k_lens):
    """And with values that are not finite, hidden from some rows of a tile: those keep their bits."""
    q, k, v = (x.clone() for x in _packed_case(dev, q_lens, k_lens, 4, 2, D, TDT[dtype], seed=D))
    lay = PackedLayout(q_lens, k_lens, group=2)
    clean = attention_packed(q, k, v, lay)
    assert _native.last_kernel() == "seq_tile_kernel"
    _check_packed(q, k, v, clean, q_lens, k_lens, dtype)
    hidden = torch.ones(q.size(0), dtype=torch.bool, device=dev)
    a = b = 0
    for n, t in zip(q_lens, k_lens):
        k[b + t - 1], v[b + t - 1] = NAN, INF  # the last key, that the last query alone sees
        if n > 0:
            hidden[a + n - 1] = False
        a, b = a + n, b + t
    y = attention_packed(q, k, v, lay)
    assert torch.equal(y[hidden], clean[hidden])
    assert bool(y[~hidden].isnan().all())


def test_calls_on_two_streams_at_once(dev):
    """Split trees and packed batches on two streams, each call with a workspace of its own
    and both with one layout: the bits of calls one after the other."""
    lens = torch.tensor([3000, 17, 2100], dtype=torch.int32, device=dev)
    trees = [_tree_case(dev, 3, 12, 8, 2, 3100, 64, torch.bfloat16, seed=s) for s in range(2)]
    masks = [tree_masks(some_tree(12, seed=s)) for s in range(2)]
    lay = PackedLayout([500, 30, 200], group=3)
    packed = [_packed_case(dev, [500, 30, 200], [500, 30, 200], 6, 2, 64, torch.bfloat16, seed=s) for s in range(2)]

    def run(s):
        return attention_tree(*trees[s], lens, masks[s]), attention_packed(*packed[s], lay)

    want = [run(s) for s in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s].append(run(s))
    torch.cuda.synchronize()
    for s in range(2):
        for a, b in got[s]:
            assert torch.equal(a, want[s][0]) and torch.equal(b, want[s][1])


def test_tree_refusals(dev):
    q, k, v = _tree_case(dev, 2, 3, 4, 2, 40, 64, torch.bfloat16)
    ln = torch.tensor([1, 2], dtype=torch.int32, device=dev)
    ok = attention_tree(q, k, v, ln)
    assert ok.shape == q.shape
    with pytest.raises(ValueError, match="lengths"):
        attention_tree(q, k, v, ln.long())
    with pytest.raises(ValueError, match="lengths"):
        attention_tree(q, k, v, ln[:1])
    with pytest.raises(ValueError, match="lengths"):
        attention_tree(q, k, v, ln.cpu())
    with pytest.raises(ValueError, match="cached positions"):
        attention_tree(q, k, v, 38)
    with pytest.raises(ValueError, match="masks"):
        attention_tree(q, k, v, ln, torch.zeros(4, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError, match="masks"):
        attention_tree(q, k, v, ln, torch.zeros(3, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="heads"):
        attention_tree(q[:, :, :3], k, v, ln)
    with pytest.raises(ValueError):
        attention_tree(q, k[:1], v[:1], ln)
    with pytest.raises(ValueError, match="does not hold"):
        attention_tree(q, k[:, :2], v[:, :2], 0)
    with pytest.raises(TypeError):
        attention_tree(q, k.float(), v.float(), ln)
    with pytest.raises(RuntimeError, match="inference-only"):
        attention_tree(q.requires_grad_(), k, v, ln)
