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
