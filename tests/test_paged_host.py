"""Refusals of the paged cache's operators and of draft verification, without a GPU: every one of
these calls returns before it would launch anything."""

import ctypes

import pytest
import torch

from diff_gpt import _native
from diff_gpt.model.paged import append_paged, attention_paged, evict_paged
from diff_gpt.sampler.drafts import verify_drafts

NUL = ctypes.c_void_p(0)
FAKE = ctypes.c_void_p(0x1000)
EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -4


def _rows(k=0x1000, v=0x1000, pages=4, page=16, table=0x1000, width=3, lens=0x1000):
    return (ctypes.c_int64 * 15)(k, v, 64, 16, 16, 64, 16, 16, pages, page, table, width, width, lens, 0)


def _st(*x):
    return (ctypes.c_int64 * 3)(*(x or (16, 16, 16)))


def _error():
    return _native.lib().dg_last_error()


def _append(B=1, N=1, H=1, Hkv=1, D=16, dtype=0, rows=None, q=FAKE, k=FAKE, freqs=FAKE, fdtype=0, freqs_rows=10):
    return _native.lib().dg_paged_append(B, N, H, Hkv, D, dtype, _rows() if rows is None else rows, q, _st(), q, _st(),
                                         k, _st(), k, _st(), freqs, D, freqs_rows, fdtype, None, 1, NUL)


@pytest.mark.parametrize("kw,code,word", [
    (dict(B=-1), EINVAL, b"negative"), (dict(D=5), EUNSUPPORTED, b"head_dim"), (dict(D=1026), EUNSUPPORTED, b"head_dim"),
    (dict(dtype=9), EUNSUPPORTED, b"dtype"), (dict(fdtype=1), EUNSUPPORTED, b"freqs"), (dict(H=70000), EINVAL, b"heads"),
    (dict(q=NUL), EINVAL, b"NULL"), (dict(k=NUL), EINVAL, b"NULL"), (dict(freqs=NUL), EINVAL, b"freqs"),
    (dict(freqs_rows=0), EINVAL, b"freqs"), (dict(rows=_rows(k=0)), EINVAL, b"NULL"), (dict(rows=_rows(lens=0)), EINVAL, b"NULL"),
    (dict(rows=_rows(table=0)), EINVAL, b"NULL"), (dict(rows=_rows(pages=0)), EINVAL, b"pages"),
    (dict(rows=_rows(page=12)), EINVAL, b"power of two"), (dict(rows=_rows(page=0)), EINVAL, b"power of two"),
    (dict(rows=_rows(width=0)), EINVAL, b"2^30"), (dict(rows=_rows(page=1 << 20, width=1025)), EINVAL, b"2^30"),
    (dict(B=1 << 20, N=1 << 10, D=1024), EINVAL, b"workgroups"),
])
def test_append_refusals(kw, code, word):
    assert _append(**kw) == code and word in _error()


def test_empty_calls_are_fine():
    assert _append(B=0, q=NUL) == 0 and _append(N=0, q=NUL) == 0
    assert _attend(B=0, q=NUL) == 0 and _attend(N=0) == 0
    assert _evict(B=0, weights=NUL) == 0
    assert _verify(B=0, target=NUL) == 0


def _attend(B=1, N=1, H=2, Hkv=1, D=16, dtype=0, rows=None, q=FAKE, scale=1.0, longest=10, weights=None, ws=None, ws_bytes=0):
    return _native.lib().dg_paged_attention(B, N, H, Hkv, D, dtype, _rows() if rows is None else rows, q, _st(), q, _st(),
                                            scale, longest, weights, 0, 0, ws, ws_bytes, NUL)


@pytest.mark.parametrize("kw,code,word", [
    (dict(N=-1), EINVAL, b"negative"), (dict(dtype=4), EUNSUPPORTED, b"dtype"), (dict(D=0), EUNSUPPORTED, b"head_dim"),
    (dict(D=1025), EUNSUPPORTED, b"head_dim"), (dict(H=3, Hkv=2), EINVAL, b"heads"), (dict(Hkv=0), EINVAL, b"heads"),
    (dict(scale=0.0), EINVAL, b"scale"), (dict(scale=float("nan")), EINVAL, b"scale"), (dict(scale=3e38), EINVAL, b"scale"),
    (dict(N=1 << 30, H=2), EINVAL, b"2^30"), (dict(q=NUL), EINVAL, b"NULL"), (dict(rows=_rows(v=0)), EINVAL, b"NULL"),
    (dict(longest=0), EINVAL, b"longest"), (dict(longest=49), EINVAL, b"longest"), (dict(rows=_rows(page=3)), EINVAL, b"power"),
    (dict(weights=FAKE), EWORKSPACE, b"workspace"), (dict(weights=FAKE, ws=FAKE, ws_bytes=7), EWORKSPACE, b"workspace"),
    (dict(weights=FAKE, ws=ctypes.c_void_p(0x1004), ws_bytes=1 << 20), EINVAL, b"aligned"),
    (dict(rows=_rows(page=1 << 20, width=1 << 10), longest=1 << 30), EWORKSPACE, b"workspace"),
    (dict(B=1 << 24, Hkv=1), EINVAL, b"workgroups"),
])
def test_attention_refusals(kw, code, word):
    assert _attend(**kw) == code and word in _error()


def test_workspace_covers_every_kernel():
    size = _native.lib().dg_paged_attention_workspace_size
    assert size(0, 1, 1, 1, 16, 0, 100, 100, 0) == 0 and size(1, 1, 3, 2, 16, 0, 100, 100, 0) == 0
    assert size(64, 1, 16, 4, 128, 1, 256, 256, 0) == 0  # no kernel splits so few positions
    one = size(1, 1, 4, 4, 64, 1, 100000, 100000, 0)
    # with weights the rows' sums, and few rows' scores, as well
    assert one > 0 and size(1, 1, 4, 4, 64, 1, 100000, 100000, 1) >= max(one + 16, 4 * 4 * 100096)
    assert size(1, 16, 4, 4, 64, 1, 100, 100, 1) == 4 * 4 * 16  # the sums of more than 8 rows
    assert size(1, 1, 4, 4, 300, 3, 100, 100, 1) == 32
    assert size(1, 1 << 30, 4, 2, 64, 3, 100, 100, 1) == 0 and size(1, 1, 1, 1, 64, 0, 100, 0, 1) == 0


def _evict(B=1, Hkv=1, D=16, dtype=0, rows=None, weights=FAKE, keep=8, recent=2, to_width=1, to=FAKE):
    return _native.lib().dg_paged_evict(B, Hkv, D, dtype, _rows() if rows is None else rows, weights, 48, 48, keep, recent, to,
                                        to_width, to_width, FAKE, FAKE, FAKE, NUL)


@pytest.mark.parametrize("kw,code,word", [
    (dict(Hkv=0), EINVAL, b"size"), (dict(D=2000), EUNSUPPORTED, b"head_dim"), (dict(dtype=-1), EUNSUPPORTED, b"dtype"),
    (dict(keep=0, recent=0), EINVAL, b"keep"), (dict(recent=9), EINVAL, b"keep"), (dict(recent=-1), EINVAL, b"keep"),
    (dict(weights=NUL), EINVAL, b"NULL"), (dict(to=NUL), EINVAL, b"NULL"), (dict(keep=17), EINVAL, b"into"),
    (dict(to_width=0), EINVAL, b"into"), (dict(rows=_rows(page=5)), EINVAL, b"power"),
    (dict(rows=_rows(k=0x1001)), EINVAL, b"aligned"), (dict(B=1 << 23), EINVAL, b"threads"),
])
def test_evict_refusals(kw, code, word):
    assert _evict(**kw) == code and word in _error()


def _verify(B=1, N=2, V=100, dtype=0, target=FAKE, tokens=FAKE, uniforms=FAKE, noise=FAKE, inv=1.0, ws=None, ws_bytes=0):
    return _native.lib().dg_verify_drafts(B, N, V, dtype, target, V, V, None, 0, 0, tokens, uniforms, noise, V, None, inv,
                                          FAKE, FAKE, FAKE, ws, ws_bytes, NUL)


@pytest.mark.parametrize("kw,code,word", [
    (dict(B=-1), EINVAL, b"negative"), (dict(N=-1), EINVAL, b"drafts"), (dict(N=65), EINVAL, b"drafts"),
    (dict(V=0), EINVAL, b"vocabulary"), (dict(V=1 << 30), EINVAL, b"vocabulary"), (dict(dtype=7), EUNSUPPORTED, b"dtype"),
    (dict(inv=-1.0), EINVAL, b"temperature"), (dict(inv=float("nan")), EINVAL, b"temperature"),
    (dict(inv=1e-40), EINVAL, b"temperature"), (dict(target=NUL), EINVAL, b"NULL"), (dict(tokens=NUL), EINVAL, b"NULL"),
    (dict(uniforms=NUL), EINVAL, b"random"), (dict(noise=NUL), EINVAL, b"random"),
    (dict(target=ctypes.c_void_p(0x1002)), EINVAL, b"aligned"), (dict(V=50000), EWORKSPACE, b"workspace"),
    (dict(V=50000, ws=ctypes.c_void_p(0x1008), ws_bytes=1 << 20), EINVAL, b"aligned"),
    (dict(B=1 << 24, V=50000, ws=FAKE, ws_bytes=1 << 40), EINVAL, b"threads"),
])
def test_verify_refusals(kw, code, word):
    assert _verify(**kw) == code and word in _error()


def test_cpu_tensors_are_refused():
    x, pages = torch.zeros(1, 1, 1, 16), torch.zeros(2, 16, 1, 16)
    table, n = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm"):
        append_paged(x, x, x, torch.zeros(4, 8, 2), pages, pages, table, n)
    with pytest.raises(RuntimeError, match="ROCm"):
        attention_paged(x, pages, pages, table, n)
    with pytest.raises(RuntimeError, match="ROCm"):
        evict_paged(pages, pages, table, n, torch.zeros(1, 1, 16), 4, 2, table)
    with pytest.raises(RuntimeError, match="ROCm"):
        verify_drafts(torch.zeros(1, 2, 5), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 1), torch.ones(1, 5))
