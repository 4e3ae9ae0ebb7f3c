"""The operators over a cache in pages against 64 bits: attention of chunks and single
tokens with and without the positions' weights, the append, and eviction."""

import math

import pytest
import torch

from paged_cases import Pool, attend_rows
from seq_cases import HALF, TDT, close

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _queries(dev, dtype, B, N, H, D, seed):
    g = torch.Generator().manual_seed(seed + 77)
    return torch.randn(B, N, H, D, generator=g).to(TDT[dtype]).to(dev)


def _check(dev, dtype, lens, counts, N, H, Hkv, D, S, seed=0, weights=True, head_major=True, longest=None, pass_counts=True):
    from diff_gpt.model.paged import attention_paged

    pool = Pool(dev, dtype, lens, counts, Hkv, D, S, seed, head_major=head_major)
    q = _queries(dev, dtype, len(lens), N, H, D, seed)
    for b, n in enumerate(counts):
        q[b, n:] = NAN  # tokens that are not there
    ref, a, ref_w, most = attend_rows(torch.nan_to_num(q), pool)
    w = None
    if weights:
        g = torch.Generator().manual_seed(seed)
        before = torch.rand(len(lens), Hkv, pool.table.size(1) * S + 3, generator=g).to(dev)
        w = before.clone()
    y = attention_paged(q, pool.k, pool.v, pool.table, pool.lengths, counts=pool.new if pass_counts else None, weights=w,
                        longest=longest)
    vmax = max([1.0] + [float(v.double().abs().max()) for v in pool.v_rows if v.numel()])
    for b, n in enumerate(counts):
        assert not y[b, n:].any(), "tokens that are not there have zeros"
        if n:
            close(y[b, :n], ref[b, :n], a[b, :n], dtype, lens[b] + n, vmax)
    if weights:
        # a score of D products and its row's sum are off by (D + 8) half steps of sum |q||k| each;
        # exp2, the sums over tokens and the addition by a few half steps of the result
        rel = 2 * (D + 8) * 2.0**-24 * most + 40 * 2.0**-24 if dtype != "f64" else 2.0**-24
        for b, (at, n) in enumerate(zip(lens, counts)):
            t = at + n if n else 0  # a row without tokens gives nothing
            got, old = w[b, :, :t].double(), before[b, :, :t].double()
            tol = rel * ref_w[b][:, :t] + 2.0**-23 * (old + ref_w[b][:, :t])
            assert bool(((got - old - ref_w[b][:, :t]).abs() <= tol).all())
            assert torch.equal(w[b, :, t:], before[b, :, t:]), "nothing is written behind a row's positions"
    return y, w


RAGGED = [0, 1, 15, 16, 17, 63, 64, 200, 513]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 16), (4, 2, 32), (8, 2, 64), (6, 2, 80), (8, 8, 128), (5, 1, 65), (2, 1, 256),
                                     (3, 3, 24), (2, 2, 300)])
@pytest.mark.parametrize("S", [1, 16, 128])
def test_single_tokens(dev, dtype, H, Hkv, D, S):
    _check(dev, dtype, RAGGED, [1] * len(RAGGED), 1, H, Hkv, D, S, pass_counts=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 16), (4, 1, 32), (8, 2, 64), (6, 2, 80), (16, 4, 128), (4, 2, 65), (2, 1, 256)])
@pytest.mark.parametrize("N,S", [(2, 4), (31, 16), (70, 64), (150, 8)])
def test_chunks(dev, dtype, H, Hkv, D, N, S):
    counts = [N, 0, 1, N - 1, (N + 1) // 2, N, N, N // 3, N]
    _check(dev, dtype, RAGGED, counts, N, H, Hkv, D, S)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_many_rows_take_the_wide_workgroups(dev, dtype, D):
    """Enough tiles for 64 and 128 rows a workgroup."""
    B = 40
    lens = [(37 * b) % 300 for b in range(B)]
    counts = [130 - (b % 3) for b in range(B)]
    _check(dev, dtype, lens, counts, 130, 16, 4, D, 16, weights=D == 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("N,D,S", [(1, 64, 256), (8, 64, 16), (40, 128, 64), (1, 65, 32), (3, 128, 1024), (1, 16, 8)])
def test_long_rows_are_split(dev, dtype, N, D, S):
    from diff_gpt import _native

    lens = [9000, 1, 4097, 1024, 0]
    counts = [N, N, 0, N, N]
    _check(dev, dtype, lens, counts, N, 4, 2, D, S)
    _check(dev, dtype, lens, counts, N, 4, 2, D, S, weights=False)
    assert "join" in _native.last_kernel()
    # a hint far off changes how rows are split and nothing else
    _check(dev, dtype, lens, counts, N, 4, 2, D, S, longest=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B", [63, 64, 65])
@pytest.mark.parametrize("N,H,Hkv,D", [(1, 16, 8, 128), (3, 8, 8, 64)])
def test_rows_in_turns(dev, dtype, B, N, H, Hkv, D):
    """More workgroups than run at once, whose longest rows come first: rows alike, rows of nothing
    and rows without tokens among them."""
    lens = [(331 * b) % 1300 if b % 5 else 700 for b in range(B)]
    lens[0] = 1500
    counts = [0 if b % 11 == 7 else max(1, N - b % 3) for b in range(B)]
    _check(dev, dtype, lens, counts, N, H, Hkv, D, 64)


def test_positions_outside_the_hint_and_the_table(dev):
    """Lengths are cut to what the table covers, counts to what is left of it."""
    from diff_gpt.model.paged import attention_paged

    pool = Pool(dev, "f32", [48, 48], [0, 0], 2, 16, 16)
    table = pool.table[:, :3].contiguous()
    q = _queries(dev, "f32", 2, 4, 2, 16, 0)
    lens = torch.tensor([46, 1000], dtype=torch.int32, device=dev)
    y = attention_paged(q, pool.k, pool.v, table, lens, counts=torch.tensor([4, -3], dtype=torch.int32, device=dev))
    pool.lens, pool.counts = [46, 48], [2, 0]
    ref, a, _, _ = attend_rows(q, pool)
    close(y[:1, :2], ref[:1, :2], a[:1, :2], "f32", 48, 5.0)
    assert not y[0, 2:].any() and not y[1].any()


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("f32", 64), ("bf16", 65), ("f64", 16)])
def test_pages_that_the_pool_lacks_read_as_zeros(dev, dtype, D):
    from diff_gpt.model.paged import attention_paged

    pool = Pool(dev, dtype, [64], [1], 1, D, 16)
    q = _queries(dev, dtype, 1, 1, 2, D, 3)
    table = pool.table.clone()
    table[0, 1], table[0, 2] = -5, pool.k.size(0)
    y = attention_paged(q, pool.k, pool.v, table, pool.lengths)
    pool.k_rows[0][16:48] = 0
    pool.v_rows[0][16:48] = 0
    ref, a, _, _ = attend_rows(q, pool)
    close(y, ref, a, dtype, 65, 5.0)


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("f16", 128), ("f32", 32), ("bf16", 40), ("f32", 33)])
def test_values_that_are_not_finite_reach_only_who_sees_them(dev, dtype, D):
    from diff_gpt.model.paged import attention_paged

    lens, N = [70, 3], 5
    pool = Pool(dev, dtype, lens, [N, N], 2, D, 16)
    q = _queries(dev, dtype, 2, N, 4, D, 5)
    ref, a, _, _ = attend_rows(q, pool)
    bad = lens[0] + 3  # a key that tokens 3 and 4 of row 0 see
    page = pool.pages_of[0][bad // 16]
    pool.k[page, bad % 16, :] = NAN
    pool.v[page, bad % 16, :] = float("inf")
    w = torch.zeros(2, 2, pool.table.size(1) * 16, device=dev)
    y = attention_paged(q, pool.k, pool.v, pool.table, pool.lengths, weights=w)
    close(y[0, :3], ref[0, :3], a[0, :3], dtype, 80, 5.0)
    close(y[1], ref[1], a[1], dtype, 80, 5.0)
    assert bool(torch.isnan(y[0, 3:]).all())
    assert bool(torch.isfinite(w[1]).all())


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("f32", 16), ("f16", 66)])
def test_layouts_and_strides(dev, dtype, D):
    """Pages with their heads side by side, queries as columns of a projection, and pages whose
    rows start anywhere."""
    from diff_gpt.model.paged import attention_paged

    _check(dev, dtype, [5, 100, 40], [3, 2, 3], 3, 4, 2, D, 16, head_major=False)
    pool = Pool(dev, dtype, [5, 100, 40], [3, 3, 3], 2, D, 16, seed=4)
    wide = torch.randn(3, 3, 4 * D + 9, device=dev).to(TDT[dtype])
    q = wide[..., 3 : 3 + 4 * D].view(3, 3, 4, D) if D == 66 else wide[..., : 4 * D].view(3, 3, 4, D)
    y = attention_paged(q, pool.k, pool.v, pool.table, pool.lengths)
    ref, a, _, _ = attend_rows(q, pool)
    close(y, ref, a, dtype, 110, 6.0)
    odd = torch.full((*pool.k.shape[:3], D + 1), NAN, dtype=pool.k.dtype, device=dev)[..., 1:]
    odd.copy_(pool.k)
    y = attention_paged(q, odd, pool.v, pool.table, pool.lengths)
    close(y, ref, a, dtype, 110, 6.0)


def test_scales(dev):
    from diff_gpt.model.paged import attention_paged

    pool = Pool(dev, "f32", [50], [1], 2, 64, 16)
    q = _queries(dev, "f32", 1, 1, 4, 64, 1)
    y = attention_paged(q, pool.k, pool.v, pool.table, pool.lengths, scale=0.25)
    ref, a, _, _ = attend_rows(q * (0.25 * 8), pool)
    close(y, ref, a, "f32", 51, 5.0)


def test_pools_behind_four_gigabytes(dev):
    """Page offsets past 32 bits, in bytes and in elements."""
    from diff_gpt.model.paged import append_paged, attention_paged, evict_paged

    S, Hkv, D = 256, 4, 128
    P = (1 << 32) // (S * Hkv * D) + 3  # elements past 2^32
    k, v = (torch.empty(P, Hkv, S, D, dtype=torch.bfloat16, device=dev).transpose(1, 2) for _ in range(2))
    table = torch.tensor([[P - 1, 1], [P - 2, -1]], dtype=torch.int32, device=dev)
    lens = torch.tensor([255, 3], dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(0)
    for page in (P - 1, P - 2, 1):
        for x in (k, v):
            x[page].normal_(generator=g)
    q, kn, vn = (torch.randn(2, 2, h, D, generator=g, device=dev).bfloat16() for h in (8, 4, 4))
    freqs = torch.ones(300, D // 2, 2, device=dev)
    append_paged(q, kn, vn, freqs, k, v, table, lens)
    assert torch.equal(v[P - 1, 255], vn[0, 0]) and torch.equal(v[1, 0], vn[0, 1]) and torch.equal(v[P - 2, 3:5], vn[1])
    small_k, small_v = (torch.stack([x[1], x[P - 2], x[P - 1]]) for x in (k, v))
    small = torch.tensor([[2, 0], [1, -1]], dtype=torch.int32, device=dev)
    w, ws = torch.zeros(2, 4, 512, device=dev), torch.zeros(2, 4, 512, device=dev)
    y = attention_paged(q, k, v, table, lens, weights=w)
    assert torch.equal(y, attention_paged(q, small_k, small_v, small, lens, weights=ws)) and torch.equal(w, ws)
    to = torch.tensor([[2], [P - 3]], dtype=torch.int32, device=dev)
    r = evict_paged(k, v, table, lens + 2, w, 40, 8, to)
    at = r.kept[0, 1].long()
    src = torch.where(at < 256, at, at - 256)
    rows = torch.where((at < 256)[:, None], k[P - 1, src, 1], k[1, src, 1])
    assert torch.equal(k[2, :40, 1], rows) and torch.equal(k[P - 3, :5], k[P - 2, :5])


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


def _turn(x, cs, norm):
    x, cs = x.double(), cs.double()
    a, b, c, s = x[..., 0::2], x[..., 1::2], cs[..., 0], cs[..., 1]
    y = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    size = y.abs().amax(-1, keepdim=True)
    if norm:
        f = torch.rsqrt(y.square().mean(-1, keepdim=True) + 2.0**-23)
        y, size = y * f, size * f
    return y, size


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 16), (8, 2, 128), (3, 1, 80), (5, 5, 2), (2, 1, 66), (1, 1, 1024), (2, 2, 520),
                                     (6, 2, 32), (2, 1, 130)])
@pytest.mark.parametrize("N,S", [(1, 16), (7, 1), (40, 64)])
@pytest.mark.parametrize("odd", [False, True])
def test_append(dev, dtype, H, Hkv, D, N, S, odd):
    from diff_gpt.model.paged import append_paged

    lens = [0, 3, 64, 17]
    counts = [N, 0, N, (N + 1) // 2]
    pool = Pool(dev, dtype, lens, counts, Hkv, D, S, seed=3)
    before = pool.k.clone(), pool.v.clone()
    g = torch.Generator().manual_seed(9)
    extra = 3 if odd else 0
    rows = torch.randn(4, N, (H + 2 * Hkv) * D + extra, generator=g).to(TDT[dtype]).to(dev)[..., extra:]
    q = rows[..., : H * D].unflatten(-1, (H, D))
    k = rows[..., H * D : (H + Hkv) * D].unflatten(-1, (Hkv, D))
    v = rows[..., (H + Hkv) * D :].unflatten(-1, (Hkv, D))
    freqs = torch.randn(200, D // 2, 2, generator=g)
    freqs = freqs.to(dev) if odd else freqs.to(TDT[dtype]).to(dev)  # an fp32 table, or one of the data's type
    positions = torch.tensor([5, 0, 100, 1], dtype=torch.int32, device=dev) if odd else None
    out = append_paged(q, k, v, freqs, pool.k, pool.v, pool.table, pool.lengths, counts=pool.new, positions=positions,
                       qknorm=not (odd and N == 7))
    norm = not (odd and N == 7)
    # the rotation and the norm in fp32: eight half steps of a head's largest element, and D of its mean square's
    half, step = HALF[dtype], (2.0**-53 if dtype == "f64" else 2.0**-24) * (8 + D)
    seen = torch.zeros(pool.k.shape[:2], dtype=torch.bool, device=dev)
    for b, n in enumerate(counts):
        assert not out[b, n:].any()
        at = lens[b] if positions is None else int(positions[b])
        cs = freqs[at : at + n][:, None]
        for x, got in ((q[b, :n], out[b, :n]), (k[b, :n], None)):
            pages = torch.tensor([pool.pages_of[b][(lens[b] + i) // S] for i in range(n)], dtype=torch.long, device=dev)
            slot = (lens[b] + torch.arange(n, device=dev)) % S
            if got is None:
                got = pool.k[pages, slot]
                assert torch.equal(pool.v[pages, slot], v[b, :n])
                seen[pages, slot] = True
            ref, size = _turn(x, cs, norm)
            tol = half * ref.abs() + step * size + (2.0**-25 if dtype == "f16" else 0.0)
            assert bool(((got.double() - ref).abs() <= tol).all())
    for now, old in zip((pool.k, pool.v), before):  # every other place is as it was, NaN included
        assert torch.equal(torch.nan_to_num(now[~seen], nan=7.0), torch.nan_to_num(old[~seen], nan=7.0))


@pytest.mark.parametrize("N", [1, 900])
def test_append_of_single_heads_whose_stride_is_any(dev, N):
    """One head is not stepped over: a stride no 32 bits hold says nothing."""
    from diff_gpt.model.paged import append_paged

    freqs = torch.randn(N, 8, 2, device=dev)
    lengths, table = torch.zeros(5, dtype=torch.int32, device=dev), torch.arange(5 * 57, dtype=torch.int32, device=dev).view(5, 57)

    def far(t):
        s = t.stride()
        return t.as_strided(t.shape, (s[0], s[1], 2**40, 1))

    x = [torch.randn(5, N, 1, 16, device=dev) for _ in range(3)]
    near = [torch.zeros(5 * 57, 16, 1, 16, device=dev) for _ in range(2)]
    pages = [torch.zeros_like(t) for t in near]
    a = append_paged(*x, freqs, *near, table, lengths)
    b = append_paged(*map(far, x), freqs, *map(far, pages), table, lengths)
    assert torch.equal(a, b) and torch.equal(near[0], pages[0]) and torch.equal(near[1], pages[1]) and bool(near[0].any())


def test_append_of_rows_whose_squares_overflow_or_vanish(dev):
    """As the norm in fp32 has it: infinite squares leave zeros, zeros stay zeros, NaN stays NaN."""
    from diff_gpt.model.paged import append_paged

    pool = Pool(dev, "f32", [0], [5], 1, 16, 8)
    q = torch.ones(1, 5, 1, 16, device=dev) * torch.tensor([1e20, 0.0, 1e-20, float("nan"), 3.0], device=dev)[:, None, None]
    freqs = torch.tensor([1.0, 0.0], device=dev).expand(5, 8, 2)
    out = append_paged(q, q, q, freqs, pool.k, pool.v, pool.table, pool.lengths)[0, :, 0]
    assert not out[0].any() and not out[1].any() and bool(torch.isnan(out[3]).all())
    # 1e-20 squared is lost beside eps = 2^-23
    assert torch.allclose(out[2], q[0, 2, 0] * 2.0**11.5, rtol=1e-6)
    assert torch.allclose(out[4], torch.ones(16, device=dev), rtol=1e-6)
    assert torch.equal(torch.nan_to_num(pool.v[pool.pages_of[0][0], :5, 0]), torch.nan_to_num(q[0, :, 0]))


def test_append_positions_outside_the_table_and_pages_outside_the_pool(dev):
    from diff_gpt.model.paged import append_paged

    pool = Pool(dev, "f32", [10, 10, 14], [4, 4, 4], 1, 16, 8)
    table = pool.table.clone()
    table[1, 1] = -1
    before = pool.k.clone()
    q, k, v = (torch.randn(3, 4, 1, 16, device=dev) for _ in range(3))
    freqs = torch.ones(12, 8, 2, device=dev)
    at = torch.tensor([-2, 0, 10], dtype=torch.int32, device=dev)
    out = append_paged(q, k, v, freqs, pool.k, pool.v, table[:, :2], pool.lengths, positions=at)
    nan = torch.isnan(out).all(-1).all(-1)
    assert nan.tolist() == [[True, True, False, False], [False] * 4, [False, False, False, False]]
    assert not out[2, 2:].any()  # the two tokens that two pages of 8 have no room for behind 14
    p = pool.pages_of[1]
    assert torch.equal(torch.nan_to_num(pool.k[p[1]]), torch.nan_to_num(before[p[1]]))
    # positions past the table's end
    out = append_paged(q, k, v, freqs, pool.k, pool.v, table, pool.lengths)
    assert torch.isnan(out).all(-1).all(-1)[0].tolist() == [False, False, True, True]


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------


def _kept(w, n, keep, recent):
    if n <= keep:
        return list(range(n))
    old = w[: n - recent].tolist()
    key = [(0, 0.0) if x != x else (1, -x) for x in old]
    return sorted(sorted(range(len(old)), key=lambda i: (key[i], i))[: keep - recent]) + list(range(n - recent, n))


@pytest.mark.parametrize("kind", ["spread", "zeros", "few", "signs", "nan", "close"])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (40, 0), (40, 40), (40, 7), (1000, 300), (3000, 100)])
@pytest.mark.parametrize("dtype,D,S", [("bf16", 64, 16), ("f32", 7, 8), ("f16", 3, 64), ("f64", 16, 1)])
def test_evict(dev, dtype, D, S, keep, recent, kind):
    from diff_gpt.model.paged import evict_paged

    Hkv, lens = 3, [0, 1, 39, 40, 41, 65, 1500, 2500]
    room = -(-keep // S)
    pool = Pool(dev, dtype, lens, [0] * len(lens), Hkv, D, S, seed=keep, spare=room * len(lens) + 1)
    to_host = [[pool.free[b * room + i] for i in range(room)] for b in range(len(lens))]
    to = torch.tensor(to_host, dtype=torch.int32, device=dev)
    cap = pool.table.size(1) * S
    g = torch.Generator().manual_seed(recent)
    w = torch.randn(len(lens), Hkv, cap + 5, generator=g)
    w = {"spread": w.exp(), "zeros": w.relu(), "few": (w * 2).round().abs(), "signs": torch.where(w.abs() < 0.5, w * 0.0, w),
         "nan": torch.where(w > 1.5, NAN, torch.where(w < -1.5, float("inf"), w)),
         "close": 1.0 + torch.randint(0, 3, w.shape, generator=g) * 2.0**-23}[kind].to(dev)
    before = pool.k.clone()
    r = evict_paged(pool.k, pool.v, pool.table, pool.lengths, w, keep, recent, to)
    assert r.lengths.tolist() == [min(n, keep) for n in lens]
    assert r.weights.shape == (len(lens), Hkv, room * S)
    touched = torch.zeros(pool.k.shape[:3], dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        for h in range(Hkv):
            want = _kept(w[b, h], n, keep, recent)
            assert r.kept[b, h].tolist() == want + [-1] * (keep - len(want))
            src = torch.tensor(want, dtype=torch.long, device=dev)
            same = torch.nan_to_num(r.weights[b, h, : len(want)], nan=-9.0), torch.nan_to_num(w[b, h, src], nan=-9.0)
            assert torch.equal(*same) and not r.weights[b, h, len(want) :].any()
            dst = torch.arange(len(want), device=dev)
            pages = to[b].long()[dst // S]
            assert torch.equal(pool.k[pages, dst % S, h], pool.k_rows[b][src, h])
            assert torch.equal(pool.v[pages, dst % S, h], pool.v_rows[b][src, h])
            touched[pages, dst % S, h] = True
    assert torch.equal(torch.nan_to_num(pool.k[~touched], nan=7.0), torch.nan_to_num(before[~touched], nan=7.0))


def test_evict_long_rows_and_strided_weights(dev):
    from diff_gpt.model.paged import evict_paged

    S, n, keep, recent = 512, 150001, 60000, 1000
    pool = Pool(dev, "bf16", [n, 700], [0, 0], 1, 8, S, spare=2 * 118)
    to = torch.tensor([pool.free[:118], pool.free[118:236]], dtype=torch.int32, device=dev)
    w = torch.rand(2, 4, pool.table.size(1) * S, device=dev)[:, 1:2]
    w[..., ::3] = 0.25
    r = evict_paged(pool.k, pool.v, pool.table, pool.lengths, w, keep, recent, to)
    old = w[0, 0, : n - recent]
    order = torch.sort(old, descending=True, stable=True).indices[: keep - recent].sort().values
    assert torch.equal(r.kept[0, 0].long(), torch.cat([order, torch.arange(n - recent, n, device=dev)]))
    at = torch.arange(keep, device=dev)
    assert torch.equal(pool.v[to[0].long()[at // S], at % S, 0], pool.v_rows[0][r.kept[0, 0].long(), 0])


# ---------------------------------------------------------------------------
# streams, graphs, a run of them together
# ---------------------------------------------------------------------------


def test_captured_calls_replay(dev):
    """Append, attention with weights and eviction in one graph, replayed for other lengths and inputs."""
    from diff_gpt.model.paged import append_paged, attention_paged, evict_paged

    S, Hkv, H, D, N = 16, 2, 4, 64, 3
    pool = Pool(dev, "bf16", [3000, 40], [N, N], Hkv, D, S, spare=2 * 8 + 2)
    table = pool.table.clamp(min=0, max=pool.k.size(0) - 1)
    to = torch.tensor([pool.free[:8], pool.free[8:16]], dtype=torch.int32, device=dev)
    freqs = torch.randn(4000, D // 2, 2, device=dev)
    q, k, v = (torch.randn(2, N, h, D, device=dev).bfloat16() for h in (H, Hkv, Hkv))
    w = torch.zeros(2, Hkv, table.size(1) * S, device=dev)
    new = torch.full((2,), N, dtype=torch.int32, device=dev)

    def step():
        q_rot = append_paged(q, k, v, freqs, pool.k, pool.v, table, pool.lengths, counts=new)
        y = attention_paged(q_rot, pool.k, pool.v, table, pool.lengths, counts=new, weights=w)
        return y, evict_paged(pool.k, pool.v, table, pool.lengths + new, w, 100, 10, to)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, r = step()
    for i in range(4):
        q.normal_(), k.normal_(), v.normal_(), w.zero_()
        pool.lengths.copy_(torch.tensor([2900 + 30 * i, 40 - 9 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone(), r.lengths.clone(), r.weights.clone(), r.kept.clone(), w.clone()
        w.zero_()
        ey, er = step()
        for a, b in zip(got, (ey, er.lengths, er.weights, er.kept, w)):
            assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


def test_two_streams_at_once(dev):
    from diff_gpt.model.paged import attention_paged

    a, b = (Pool(dev, "bf16", [6000, 500, 20], [2] * 3, 2, 64, 32, seed=s) for s in (1, 2))
    q = _queries(dev, "bf16", 3, 2, 8, 64, 0)
    alone = [attention_paged(q, p.k, p.v, p.table, p.lengths) for p in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, p in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(attention_paged(q, p.k, p.v, p.table, p.lengths))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in outs[i])


def test_chunks_give_what_one_prompt_gives(dev):
    """A prompt appended and attended in chunks of any size has one prompt's outputs and weights."""
    from diff_gpt.model.paged import append_paged, attention_paged

    S, H, Hkv, D, T = 16, 4, 2, 32, 97
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, T, h, D, generator=g).to(dev) for h in (H, Hkv, Hkv))
    freqs = torch.randn(T, D // 2, 2, generator=g).to(dev)
    table = torch.randperm(8, generator=g).int().to(dev)[None]
    outs = []
    for cuts in ([97], [1, 31, 64, 1], [1] * 97):
        pages = torch.full((2, 8, S, Hkv, D), NAN, device=dev)
        w = torch.zeros(1, Hkv, 8 * S, device=dev)
        y, at = [], 0
        for n in cuts:
            lens = torch.tensor([at], dtype=torch.int32, device=dev)
            part = slice(at, at + n)
            q_rot = append_paged(q[:, part], k[:, part], v[:, part], freqs, pages[0], pages[1], table, lens)
            y.append(attention_paged(q_rot, pages[0], pages[1], table, lens, weights=w))
            at += n
        outs.append((torch.cat(y, 1), w, pages[:, table[0].long()].flatten(1, 2)[:, :T]))
    for y, w, pages in outs[1:]:
        assert torch.equal(pages, outs[0][2])
        assert torch.allclose(y, outs[0][0], rtol=0, atol=1e-5)
        assert torch.allclose(w, outs[0][1], rtol=1e-5, atol=1e-5)
    assert math.isclose(float(outs[0][1].sum()), T * H, rel_tol=1e-5)


@pytest.mark.parametrize("dtype,D,N", [("bf16", 64, 1), ("bf16", 64, 20), ("f32", 256, 2), ("f32", 128, 12), ("bf16", 65, 3)])
def test_weights_past_the_hint(dev, dtype, D, N):
    """Every form of the weights goes over all of a row's positions, whatever the hint says."""
    _check(dev, dtype, [2500, 10, 700], [N, N, N], N, 2, 2, D, 16, longest=20)


def test_rows_of_weights_must_not_overlap(dev):
    from diff_gpt.model.paged import attention_paged

    pool = Pool(dev, "f32", [5, 9], [1, 1], 2, 16, 16)
    q = _queries(dev, "f32", 2, 1, 2, 16, 0)
    cap = pool.table.size(1) * 16
    flat = torch.zeros(8 * cap, device=dev)
    for strides in ((cap, cap, 1), (cap - 1, 4 * cap, 1), (0, cap, 1), (2 * cap, 0, 1), (3 * cap, 2 * cap, 1)):
        with pytest.raises(ValueError, match="overlap"):
            attention_paged(q, pool.k, pool.v, pool.table, pool.lengths, weights=flat.as_strided((2, 2, cap), strides))
    for strides in ((2 * cap, cap, 1), (cap, 2 * cap, 1)):
        w = flat.zero_().as_strided((2, 2, cap), strides)
        attention_paged(q, pool.k, pool.v, pool.table, pool.lengths, weights=w)
        assert torch.allclose(w.sum(-1), torch.ones(2, 2, device=dev), atol=1e-6)


def test_refusals_of_the_python_entry_points(dev):
    from diff_gpt.model.paged import append_paged, attention_paged, evict_paged

    pool = Pool(dev, "f32", [5, 9], [1, 1], 2, 16, 16)
    q, k, v, t, n = _queries(dev, "f32", 2, 1, 4, 16, 0), pool.k, pool.v, pool.table, pool.lengths
    new = torch.zeros(2, 1, 2, 16, device=dev)
    freqs = torch.ones(20, 8, 2, device=dev)
    w = torch.zeros(2, 2, t.size(1) * 16, device=dev)
    to = torch.tensor([[pool.free[0]], [pool.free[1]]], dtype=torch.int32, device=dev)
    attend = lambda **kw: attention_paged(**{**dict(q=q, k_pages=k, v_pages=v, table=t, lengths=n), **kw})  # noqa: E731
    append = lambda **kw: append_paged(**{**dict(q=q, k=new, v=new, freqs=freqs, k_pages=k, v_pages=v, table=t, lengths=n), **kw})  # noqa: E731
    evict = lambda **kw: evict_paged(**{**dict(k_pages=k, v_pages=v, table=t, lengths=n, weights=w, keep=4, recent=2, to=to), **kw})  # noqa: E731
    attend(), append(), evict()
    bad_pages = torch.zeros(3, 12, 2, 16, device=dev)
    for call, kw in [(attend, dict(q=q[0])), (attend, dict(q=q[:, :, :3])), (attend, dict(q=q[..., :8])), (attend, dict(v_pages=v[:1])),
                     (attend, dict(k_pages=bad_pages, v_pages=bad_pages)), (attend, dict(table=t.long())), (attend, dict(table=t[:1])),
                     (attend, dict(table=t[:, :0])), (attend, dict(table=t.t().contiguous().t())), (attend, dict(lengths=n.long())),
                     (attend, dict(lengths=n[:1])), (attend, dict(lengths=n.cpu())), (attend, dict(counts=n.cpu())),
                     (attend, dict(weights=w[..., :3])), (attend, dict(weights=w.double())), (attend, dict(weights=w[:1])),
                     (attend, dict(scale=0.0)), (attend, dict(scale=float("inf"))), (attend, dict(q=q.expand(2, 1, 4, 16)[..., ::2])),
                     (append, dict(q=q[..., :8])), (append, dict(k=new[:, :, :1])), (append, dict(v=new[:1])),
                     (append, dict(freqs=freqs[:, :4])), (append, dict(freqs=freqs[:0])), (append, dict(freqs=freqs.cpu())),
                     (append, dict(positions=n.long())), (append, dict(table=t.cpu())),
                     (append, dict(q=torch.zeros(2, 1, 4, 16, 2, device=dev)[..., 0])),
                     (evict, dict(keep=0, recent=0)), (evict, dict(recent=5)), (evict, dict(keep=17)), (evict, dict(to=to.long())),
                     (evict, dict(to=to[:1])), (evict, dict(weights=w[:, :1])), (evict, dict(to=to.cpu()))]:
        with pytest.raises(ValueError):
            call(**kw)
    for call, kw in [(attend, dict(q=q.bfloat16())), (attend, dict(v_pages=v.half())), (append, dict(freqs=freqs.half())),
                     (append, dict(v=new.double())), (attend, dict(q=q.int(), k_pages=k.int(), v_pages=v.int())), (evict, dict(keep=2.5))]:
        with pytest.raises(TypeError):
            call(**kw)
    with pytest.raises(RuntimeError, match="inference"):
        attend(q=q.clone().requires_grad_())
