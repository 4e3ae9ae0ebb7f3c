"""How many splits a call over pages has, by the workspace it asks for: no GPU."""

import pytest

from diff_gpt import _native

P = 0x1000  # never followed


def _splits(B, H, Hkv, D, longest, weights, N=1, dtype=1, page=64):
    """Partial outputs and states of 4 bytes a value; with weights the rows' sums and scores follow."""
    width = -(-longest // page)
    rows = (P, P, 64 * Hkv * D, D, 64 * D, 64 * Hkv * D, D, 64 * D, 1000, page, P, width, width, P, 0)
    args = _native._PAGED_ATTENTION(B, N, H, Hkv, D, dtype, *rows, P, N * H * D, H * D, D, P, N * H * D, H * D, D, D**-0.5, longest,
                                    P if weights else 0, 0, 0)
    size = _native.lib().dg_paged_attention_workspace_size(args)
    R = B * N * H
    if weights:
        size -= (4 * R + 15) // 16 * 16 + 4 * R * (-(-width * page // 256) * 256)
    assert size % (R * (D + 2) * 4) in (0, (4 * B if B > 64 else 0))  # more rows are ordered there
    return max(1, size // (R * (D + 2) * 4))


@pytest.mark.parametrize("B,H,Hkv,D,longest", [(48, 16, 4, 128, 4096), (40, 12, 4, 128, 2049), (200, 4, 2, 64, 3001)])
def test_rows_that_nearly_fill_the_chip(B, H, Hkv, D, longest):
    """In two with the weights, whose launch joins them on the way, and whole without, where the
    join would be a launch more."""
    assert _splits(B, H, Hkv, D, longest, False) == 1
    assert _splits(B, H, Hkv, D, longest, True) == 2
    assert _splits(B, H, Hkv, D, 1500, True) == 1


def test_few_rows_are_split_either_way():
    for weights in (False, True):
        assert _splits(1, 4, 4, 16, 2100, weights) == _splits(1, 4, 4, 32, 2100, weights) == 8
        assert _splits(1, 16, 4, 128, 20000, weights) > 8
        assert _splits(1, 16, 4, 128, 200, weights) == 1
