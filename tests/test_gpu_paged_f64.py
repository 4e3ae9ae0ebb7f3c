"""float64 rows over a cache in pages: the append's rotation with a table of either type and its
norm with the type's own eps, and a float64 model over a PagedKVCache."""

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


def _check(dev, table, D, N, odd, qknorm, scale=1.0):
    from diff_gpt.model.paged import append_paged

    H, Hkv, S, lens = 4, 2, 16, [0, 3, 64, 17]
    counts = [N, 0, N, (N + 1) // 2]
    pool = Pool(dev, "f64", lens, counts, Hkv, D, S, seed=3)
    q, k, v = _rows(dev, H, Hkv, D, N, odd, scale)
    g = torch.Generator().manual_seed(1)
    freqs = torch.randn(64 + N, D // 2, 2, generator=g).to(torch.float64 if table == "f64" else torch.float32).to(dev)
    out = append_paged(q, k, v, freqs, pool.k, pool.v, pool.table, pool.lengths, counts=pool.new, qknorm=qknorm)
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
            if qknorm:
                f = torch.rsqrt(ref.square().mean(-1, keepdim=True) + 2.0**-52)
                ref = ref * f
                # D squares summed, the root and the quotient on both sides
                tol = tol * f + 2 * (D + 8) * 2.0**-53 * (size * f).amax(-1, keepdim=True)
            assert bool(((got - ref).abs() <= tol).all())


@pytest.mark.parametrize("table", ["f64", "f32"])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("D", [2, 4, 12, 64, 66, 130, 300, 1024])
@pytest.mark.parametrize("N", [1, 40, 1500])
def test_the_rotation_with_a_table_of_either_type(dev, table, odd, D, N):
    """Rows aligned to 16 bytes and not, few tokens and many."""
    if N * D > 100000:
        N = 100000 // D
    _check(dev, table, D, N, odd, qknorm=False)


@pytest.mark.parametrize("table", ["f64", "f32"])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("D", [2, 4, 64, 66, 300, 1024])
@pytest.mark.parametrize("N,scale", [(1, 1.0), (40, 1.0), (7, 1e-3), (40, 1e-7), (3, 1e-12)])
def test_the_norm_has_the_eps_of_its_type(dev, table, odd, D, N, scale):
    """2^-52, beside heads of any size: other ones' squares vanish beside 2^-23 already."""
    _check(dev, table, D, N, odd, qknorm=True, scale=scale)


def test_a_float64_model_over_pages(dev, monkeypatch):
    """GPT(...).double() in ragged chunks: logits within 1e-10 of the largest, as those of the other
    paths, of the float64 forward whose rotation is in float64 throughout, as the append's."""
    from diff_gpt.model.gpt import GPT
    from diff_gpt.model.paged import PagedKVCache
    from oracle import torch_ref as tr

    def rope(x, fc):
        re, im, c, s = x[..., 0::2], x[..., 1::2], fc[..., 0], fc[..., 1]
        return torch.stack([re * c - im * s, re * s + im * c], dim=-1).flatten(-2)

    monkeypatch.setattr(tr, "rope", rope)
    torch.manual_seed(3)
    kw = dict(vocab_size=128, n_embd=64, block_size=64, n_head=4, n_layer=3)
    model = GPT(use_checkpoint=False, attn_res_layers_per_block=2, **kw).double().to(dev).eval()
    params = {k: v.detach().cpu() for k, v in model.state_dict().items()}
    cfg = tr.ModelConfig(attn_res_layers_per_block=2, **kw)
    ids = torch.randint(0, 128, (3, 90), generator=torch.Generator().manual_seed(9))
    with torch.no_grad():
        ref = tr.forward(params, cfg, ids, None, model.freqs_cis.cpu())
    cache = PagedKVCache(3, 4, 16, 3, 30, 16, dtype=torch.float64, device=dev)
    for n in ([40, 1, 17], [1, 40, 0], [9, 9, 50], [1, 1, 1]):
        at = list(cache.lens)
        parts = [ids[b, a : a + c].tolist() for b, (a, c) in enumerate(zip(at, n))]
        most = max(n)
        got = model.forward_paged(torch.tensor([p + [0] * (most - len(p)) for p in parts], device=dev), cache, n).cpu()
        for b, c in enumerate(n):
            want = ref[b, at[b] : at[b] + c]
            assert bool(((got[b, :c] - want).abs() <= 1e-10 * ref.abs().max()).all())
