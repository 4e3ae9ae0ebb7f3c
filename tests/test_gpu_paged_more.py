"""Attention over a cache in pages where its splits, its page layouts and its callers' strides
are out of the ordinary."""

import pytest
import torch

from paged_cases import Pool, attend_rows
from seq_cases import TDT, close

pytestmark = pytest.mark.gpu


def _queries(dev, dtype, B, N, H, D, seed):
    g = torch.Generator().manual_seed(seed + 77)
    return torch.randn(B, N, H, D, generator=g).to(TDT[dtype]).to(dev)


@pytest.mark.parametrize("dtype,D", [("bf16", 16), ("bf16", 32), ("f16", 32), ("f32", 16), ("bf16", 64)])
@pytest.mark.parametrize("S", [4, 64, 256])
@pytest.mark.parametrize("at,sign", [(2700, 1), (2636, 1), (2745, -1), (2687, 1), (5, -1)])
def test_infinite_values_beside_a_splits_end(dev, dtype, D, S, at, sign):
    """2748 positions in eight splits of 384, whose stages of 256 reach past a split's end: what
    lies there, the next split's values or others of the last page, is not this one's.  An
    infinite value of a visible key is the output, not NaN, also where the waves that go past
    the end of theirs have no key of any weight in their own split."""
    from diff_gpt import _native
    from diff_gpt.model.paged import attention_paged

    pool = Pool(dev, dtype, [2747, 2740], [1, 1], 2, D, S)
    q = _queries(dev, dtype, 2, 1, 8, D, 5)
    q[0] = 1.0
    for t in range(2432, 2560):  # scores 230 and more (log2 units) below the others
        pool.k[pool.pages_of[0][t // S], t % S] = -40.0
        pool.k_rows[0][t] = -40.0
    ref, a, _, _ = attend_rows(q, pool)
    pool.v[pool.pages_of[0][at // S], at % S, 0, : D // 2] = sign * float("inf")
    y = attention_paged(q, pool.k, pool.v, pool.table, pool.lengths, longest=2048)
    assert "join" in _native.last_kernel()
    assert bool((y[0, :, :4, : D // 2] == sign * float("inf")).all())
    close(y[0, :, :4, D // 2 :], ref[0, :, :4, D // 2 :], a[0, :, :4, D // 2 :], dtype, 2748, 6.0)
    close(y[0, :, 4:], ref[0, :, 4:], a[0, :, 4:], dtype, 2748, 6.0)
    close(y[1], ref[1], a[1], dtype, 2748, 6.0)


def test_lengths_cut_where_they_are(dev):
    """dg_paged_evict's new lengths in the place of the old ones: every key head is cut alike."""
    from diff_gpt import _native
    from diff_gpt.model.paged import evict_paged

    S, Hkv, D, keep, recent = 16, 7, 16, 40, 9
    lens = [0, 39, 40, 41, 300, 1500] * 8
    room = -(-keep // S)
    pool = Pool(dev, "f32", lens, [0] * len(lens), Hkv, D, S, spare=room * len(lens))
    to = torch.tensor(pool.free, dtype=torch.int32, device=dev)[: room * len(lens)].view(len(lens), room)
    w = torch.rand(len(lens), Hkv, pool.table.size(1) * S, device=dev)
    want = evict_paged(pool.k, pool.v, pool.table, pool.lengths, w, keep, recent, to)
    moved = pool.k[to.long()].clone()
    pool.k[to.long()] = 0.0
    at = pool.lengths.clone()
    rows, _ = _native._paged_rows("evict_paged", pool.k, pool.v, pool.k.shape, pool.table, at, None, len(lens), 0)
    weights, kept = torch.empty_like(want.weights), torch.empty_like(want.kept)
    args = _native._PAGED_EVICT(len(lens), Hkv, D, 0, *rows, w.data_ptr(), w.stride(0), w.stride(1), keep, recent, to.data_ptr(),
                                room, room, at.data_ptr(), weights.data_ptr(), kept.data_ptr())
    _native._launch("evict_paged", 0, _native.lib().dg_paged_evict, args)
    assert at.tolist() == [min(n, keep) for n in lens] == want.lengths.tolist()
    assert torch.equal(kept, want.kept) and torch.equal(weights, want.weights)
    for b, n in enumerate(lens):
        n = min(n, keep)
        assert torch.equal(pool.k[to[b].long()].flatten(0, 1)[:n], moved[b].flatten(0, 1)[:n])


def _attend(dev, dtype, B, N, H, Hkv, D, S, weights, v_wider=0):
    """Ragged rows, without weights, so that the last kernel is the attention's, and with them."""
    from diff_gpt import _native
    from diff_gpt.model.paged import attention_paged

    lens = [(37 * b) % 150 for b in range(B)]
    counts = [0 if b % 13 == 5 else N - b % 3 for b in range(B)]
    pool = Pool(dev, dtype, lens, counts, Hkv, D, S, seed=D + S)
    q = _queries(dev, dtype, B, N, H, D, 1)
    for b, n in enumerate(counts):
        q[b, n:] = float("nan")
    if v_wider:
        wide = torch.full((*pool.v.shape[:3], D + v_wider), float("nan"), dtype=pool.v.dtype, device=dev)
        wide[..., :D] = pool.v
        pool.v = wide[..., :D]
    ref, a, ref_w, most = attend_rows(torch.nan_to_num(q), pool)
    w = torch.zeros(B, Hkv, pool.table.size(1) * S, device=dev) if weights else None
    y = attention_paged(q, pool.k, pool.v, pool.table, pool.lengths, counts=pool.new, weights=w)
    if not weights:
        kernel = _native.last_kernel()
    for b, n in enumerate(counts):
        assert not y[b, n:].any()
        if n:
            close(y[b, :n], ref[b, :n], a[b, :n], dtype, lens[b] + n, 6.0)
    if not weights:
        return kernel
    # a score's D products, the row's sum and the sums over tokens, in half steps of fp32
    rel = 2 * (D + 8) * 2.0**-24 * most + 40 * 2.0**-24
    for b, n in enumerate(counts):
        t = lens[b] + n if n else 0
        assert bool(((w[b, :, :t].double() - ref_w[b][:, :t]).abs() <= rel * ref_w[b][:, :t] + 2.0**-23 * ref_w[b][:, :t]).all())
        assert not w[b, :, t:].any()


@pytest.mark.parametrize("dtype,D,S", [("bf16", 16, 8), ("f16", 16, 16), ("bf16", 32, 8), ("f16", 24, 4), ("bf16", 64, 4),
                                       ("f16", 128, 4), ("bf16", 80, 1), ("f32", 16, 8), ("f32", 32, 4), ("f32", 64, 2),
                                       ("f32", 128, 4)])
@pytest.mark.parametrize("B,rows", [(40, 64), (60, 128)])
def test_wide_workgroups_over_pages_smaller_than_a_copy(dev, dtype, D, S, B, rows):
    """An address for every lane, in workgroups of 64 and 128 rows."""
    if D > 64 and rows == 64:
        B = 24
    assert _attend(dev, dtype, B, 130, 16, 4, D, S, False) == f"seq_mfma_paged_any_{rows}"
    _attend(dev, dtype, B, 130, 16, 4, D, S, True)


@pytest.mark.parametrize("dtype,D", [("bf16", 16), ("bf16", 64), ("f16", 128), ("f32", 32), ("f32", 64)])
@pytest.mark.parametrize("B,N,rows", [(3, 2, 32), (24, 130, 64), (60, 130, 128)])
def test_keys_and_values_of_different_strides(dev, dtype, D, B, N, rows):
    """Values as columns of a wider buffer, in whole 16-byte pieces."""
    if D <= 64 and rows == 64:
        B = 40
    kernel = _attend(dev, dtype, B, N, 16, 4, D, 64, False, v_wider=16)
    assert kernel == f"seq_mfma_paged_any_{rows}"
    _attend(dev, dtype, B, N, 16, 4, D, 64, True, v_wider=16)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,N,most", [(1, 1, 20000), (30, 1, 2500), (6, 40, 1500)])
def test_calls_repeat_themselves(dev, dtype, B, N, most):
    """The same call has the same bits, outputs and weights, as often as it is made."""
    from diff_gpt.model.paged import attention_paged

    pool = Pool(dev, dtype, [most - (most // 40) * b for b in range(B)], [N] * B, 2, 64, 16)
    q = _queries(dev, dtype, B, N, 8, 64, 3)
    first = None
    for _ in range(5):
        w = torch.zeros(B, 2, pool.table.size(1) * 16, device=dev)
        y = attention_paged(q, pool.k, pool.v, pool.table, pool.lengths, weights=w)
        alone = attention_paged(q, pool.k, pool.v, pool.table, pool.lengths)
        first = (y, w, alone) if first is None else first
        assert torch.equal(y, first[0]) and torch.equal(w, first[1]) and torch.equal(alone, first[2])
