"""float64 rows over a cache in pages: the append's rotation with a table of either type."""

import pytest
import torch

from paged_cases import Pool

pytestmark = pytest.mark.gpu


def _rows(dev, H, Hkv, D, N, odd, scale=1.0):
    """q, k, v of four rows as columns of one projection; odd: rows that start anywhere."""
    g = torch.Generator().manual_seed(D + N)
    extra = 3 if odd else 0
    rows = (torch.randn(4, N, (H + 2 * Hkv) * D + extra, generator=g, dtype=torch.float64) * scale).to(dev)[..., extra:]
    return (rows[..., : H * D].unflatten(-1, (H, D)), rows[..., H * D : (H + Hkv) * D].unflatten(-1, (Hkv, D)),
            rows[..., (H + Hkv) * D :].unflatten(-1, (Hkv, D)))


def _check(dev, table, D, N, odd, scale=1.0):
    from diff_gpt.model.paged import append_paged

    H, Hkv, S, lens = 4, 2, 16, [0, 3, 64, 17]
    counts = [N, 0, N, (N + 1) // 2]
    pool = Pool(dev, "f64", lens, counts, Hkv, D, S, seed=3)
    q, k, v = _rows(dev, H, Hkv, D, N, odd, scale)
    g = torch.Generator().manual_seed(1)
    freqs = torch.randn(64 + N, D // 2, 2, generator=g).to(torch.float64 if table == "f64" else torch.float32).to(dev)
    out = append_paged(q, k, v, freqs, pool.k, pool.v, pool.table, pool.lengths, counts=pool.new, qknorm=False)
    for b, n in enumerate(counts):
        assert not out[b, n:].any()
        slot = torch.arange(lens[b], lens[b] + n, device=dev)
        pages = torch.tensor(pool.pages_of[b], dtype=torch.long, device=dev)[slot // S]
        assert torch.equal(pool.v[pages, slot % S], v[b, :n])
        cs = freqs[slot][:, None].double()
        for x, got in ((q[b, :n], out[b, :n]), (k[b, :n], pool.k[pages, slot % S])):
            re, im, c, s = x[..., 0::2], x[..., 1::2], cs[..., 0], cs[..., 1]
            ref = torch.stack([re * c - im * s, re * s + im * c], dim=-1).flatten(-2)
            # two products and their sum, here and there: three half steps of the pair's products each
            size = torch.stack([(re * c).abs() + (im * s).abs(), (re * s).abs() + (im * c).abs()], dim=-1).flatten(-2)
            tol = 6 * 2.0**-53 * size
            assert bool(((got - ref).abs() <= tol).all())


@pytest.mark.parametrize("table", ["f64", "f32"])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("D", [2, 4, 12, 64, 66, 130, 300, 1024])
@pytest.mark.parametrize("N", [1, 40, 1500])
def test_the_rotation_with_a_table_of_either_type(dev, table, odd, D, N):
    """Rows aligned to 16 bytes and not, few tokens and many."""
    if N * D > 100000:
        N = 100000 // D
    _check(dev, table, D, N, odd)
