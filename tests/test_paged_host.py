"""Refusals of the paged cache's operators and of draft verification, without a GPU: every one of
these calls returns before it would launch anything."""

import pytest
import torch

from diff_gpt import _native
from diff_gpt.model.paged import append_paged, attention_paged, evict_paged
from diff_gpt.sampler.drafts import verify_drafts

EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -4


def _rows(k=0x1000, v=0x1000, pages=4, page=16, table=0x1000, width=3, lens=0x1000):
    return k, v, 64, 16, 16, 64, 16, 16, pages, page, table, width, width, lens, 0


ST = (16, 16, 16)
P = 0x1000  # never followed


def _error():
    return _native.lib().dg_last_error()


def _append(B=1, N=1, H=1, Hkv=1, D=16, dtype=0, rows=_rows(), q=P, k=P, freqs=P, fdtype=0, freqs_rows=10):
    args = _native._PAGED_APPEND(B, N, H, Hkv, D, dtype, *rows, q, *ST, q, *ST, k, *ST, k, *ST, freqs, D, freqs_rows, fdtype, 0, 1)
    return _native.lib().dg_paged_append(args, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(B=-1), EINVAL, b"negative"), (dict(D=5), EUNSUPPORTED, b"head_dim"), (dict(D=1026), EUNSUPPORTED, b"head_dim"),
    (dict(dtype=9), EUNSUPPORTED, b"dtype"), (dict(fdtype=1), EUNSUPPORTED, b"freqs"), (dict(H=70000), EINVAL, b"heads"),
    (dict(q=0), EINVAL, b"NULL"), (dict(k=0), EINVAL, b"NULL"), (dict(freqs=0), EINVAL, b"freqs"),
    (dict(freqs_rows=0), EINVAL, b"freqs"), (dict(rows=_rows(k=0)), EINVAL, b"NULL"), (dict(rows=_rows(lens=0)), EINVAL, b"NULL"),
    (dict(rows=_rows(table=0)), EINVAL, b"NULL"), (dict(rows=_rows(pages=0)), EINVAL, b"pages"),
    (dict(rows=_rows(page=12)), EINVAL, b"power of two"), (dict(rows=_rows(page=0)), EINVAL, b"power of two"),
    (dict(rows=_rows(width=0)), EINVAL, b"2^30"), (dict(rows=_rows(page=1 << 20, width=1025)), EINVAL, b"2^30"),
    (dict(B=1 << 20, N=1 << 10, D=1024), EINVAL, b"workgroups"),
    (dict(B=(1 << 31) - 1, N=(1 << 31) - 1, H=0xffff, Hkv=0xffff), EINVAL, b"workgroups"),
])
def test_append_refusals(kw, code, word):
    assert _append(**kw) == code and word in _error()


def test_null_structs_are_refused():
    L = _native.lib()
    assert L.dg_paged_append(None, None) == L.dg_paged_evict(None, None) == EINVAL
    assert L.dg_paged_attention(None, None, 0, None) == L.dg_verify_drafts(None, None, 0, None) == EINVAL
    assert L.dg_paged_attention_workspace_size(None) == L.dg_verify_drafts_workspace_size(None) == 0
    assert _append(B=1 << 32) == _attend(N=1 << 32) == _evict(B=1 << 32) == _verify(B=1 << 32) == EINVAL


def test_empty_calls_are_fine():
    assert _append(B=0, q=0) == 0 and _append(N=0, q=0) == 0
    assert _attend(B=0, q=0) == 0 and _attend(N=0) == 0
    assert _evict(B=0, weights=0) == 0
    assert _verify(B=0, target=0) == 0


def _attention_args(B=1, N=1, H=2, Hkv=1, D=16, dtype=0, rows=_rows(), q=P, scale=1.0, longest=10, weights=0):
    return _native._PAGED_ATTENTION(B, N, H, Hkv, D, dtype, *rows, q, *ST, q, *ST, scale, longest, weights, 0, 0)


def _attend(ws=None, ws_bytes=0, **kw):
    return _native.lib().dg_paged_attention(_attention_args(**kw), ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(N=-1), EINVAL, b"negative"), (dict(dtype=4), EUNSUPPORTED, b"dtype"), (dict(D=0), EUNSUPPORTED, b"head_dim"),
    (dict(D=1025), EUNSUPPORTED, b"head_dim"), (dict(H=3, Hkv=2), EINVAL, b"heads"), (dict(Hkv=0), EINVAL, b"heads"),
    (dict(scale=0.0), EINVAL, b"scale"), (dict(scale=float("nan")), EINVAL, b"scale"), (dict(scale=3e38), EINVAL, b"scale"),
    (dict(N=1 << 30, H=2), EINVAL, b"2^30"), (dict(q=0), EINVAL, b"NULL"), (dict(rows=_rows(v=0)), EINVAL, b"NULL"),
    (dict(longest=0), EINVAL, b"longest"), (dict(longest=49), EINVAL, b"longest"), (dict(rows=_rows(page=3)), EINVAL, b"power"),
    (dict(weights=P), EWORKSPACE, b"workspace"), (dict(weights=P, ws=P, ws_bytes=7), EWORKSPACE, b"workspace"),
    (dict(weights=P, ws=0x1004, ws_bytes=1 << 20), EINVAL, b"aligned"),
    (dict(rows=_rows(page=1 << 20, width=1 << 10), longest=1 << 30), EWORKSPACE, b"workspace"),
    (dict(B=1 << 24, Hkv=1), EINVAL, b"workgroups"),
    (dict(B=(1 << 31) - 1, N=128, H=(1 << 31) - 1, Hkv=(1 << 31) - 1), EINVAL, b"workgroups"),
    (dict(B=1 << 30, N=1, H=1 << 20, Hkv=1 << 20, weights=P), EINVAL, b"workgroups"),
])
def test_attention_refusals(kw, code, word):
    assert _attend(**kw) == code and word in _error()


def test_workspaces():
    def size(**kw):
        cap = kw.pop("cap", 48)
        return _native.lib().dg_paged_attention_workspace_size(
            _attention_args(**{**dict(rows=_rows(width=-(-cap // 16)), longest=cap), **kw}))

    assert size(B=0) == 0 and size(H=3, Hkv=2) == 0 and size(longest=0) == 0 and size(rows=_rows(k=0)) == 0
    assert size(B=64, H=16, Hkv=4, D=128, dtype=1, cap=256) == 0  # so few positions are not split
    one = size(H=4, Hkv=4, D=64, dtype=1, cap=100000)
    # with weights the rows' sums (4 of them, 16 bytes) and few rows' scores as well
    assert one > 0 and size(H=4, Hkv=4, D=64, dtype=1, cap=100000, weights=P) == one + 16 + 4 * 4 * 100096
    assert size(N=16, H=4, Hkv=4, D=64, dtype=1, weights=P) == 4 * 4 * 16
    assert size(H=4, Hkv=4, D=300, dtype=3, weights=P) == 4 * 8


def _evict(B=1, Hkv=1, D=16, dtype=0, rows=_rows(), weights=P, keep=8, recent=2, to_width=1, to=P):
    args = _native._PAGED_EVICT(B, Hkv, D, dtype, *rows, weights, 48, 48, keep, recent, to, to_width, to_width, P, P, P)
    return _native.lib().dg_paged_evict(args, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(Hkv=0), EINVAL, b"size"), (dict(D=2000), EUNSUPPORTED, b"head_dim"), (dict(dtype=-1), EUNSUPPORTED, b"dtype"),
    (dict(keep=0, recent=0), EINVAL, b"keep"), (dict(recent=9), EINVAL, b"keep"), (dict(recent=-1), EINVAL, b"keep"),
    (dict(weights=0), EINVAL, b"NULL"), (dict(to=0), EINVAL, b"NULL"), (dict(keep=17), EINVAL, b"into"),
    (dict(to_width=0), EINVAL, b"into"), (dict(rows=_rows(page=5)), EINVAL, b"power"),
    (dict(rows=_rows(k=0x1001)), EINVAL, b"aligned"), (dict(B=1 << 23), EINVAL, b"threads"),
    (dict(B=(1 << 31) - 1, Hkv=(1 << 31) - 1), EINVAL, b"threads"),
])
def test_evict_refusals(kw, code, word):
    assert _evict(**kw) == code and word in _error()


def _verify(B=1, N=2, V=100, dtype=0, target=P, tokens=P, uniforms=P, noise=P, inv=1.0, ws=None, ws_bytes=0):
    args = _native._VERIFY_DRAFTS(B, N, V, dtype, target, V, V, 0, 0, 0, tokens, uniforms, noise, V, 0, inv, P, P, P)
    return _native.lib().dg_verify_drafts(args, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(B=-1), EINVAL, b"negative"), (dict(N=-1), EINVAL, b"drafts"), (dict(N=65), EINVAL, b"drafts"),
    (dict(V=0), EINVAL, b"vocabulary"), (dict(V=1 << 30), EINVAL, b"vocabulary"), (dict(dtype=7), EUNSUPPORTED, b"dtype"),
    (dict(inv=-1.0), EINVAL, b"temperature"), (dict(inv=float("nan")), EINVAL, b"temperature"),
    (dict(inv=1e-40), EINVAL, b"temperature"), (dict(target=0), EINVAL, b"NULL"), (dict(tokens=0), EINVAL, b"NULL"),
    (dict(uniforms=0), EINVAL, b"random"), (dict(noise=0), EINVAL, b"random"),
    (dict(target=0x1002), EINVAL, b"aligned"), (dict(V=50000), EWORKSPACE, b"workspace"),
    (dict(V=50000, ws=0x1008, ws_bytes=1 << 20), EINVAL, b"aligned"),
    (dict(B=1 << 24, V=50000, ws=P, ws_bytes=1 << 40), EINVAL, b"threads"),
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
