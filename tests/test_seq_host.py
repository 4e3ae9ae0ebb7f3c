"""Packed layouts, tree masks and the refusals of the scoring operators, without a GPU."""

import ctypes

import pytest
import torch

from diff_gpt import _native
from diff_gpt.model.packed import PackedLayout, attention_packed
from diff_gpt.model.token_logprobs import token_logprobs
from diff_gpt.model.tree import attention_tree, tree_depths, tree_masks
from seq_cases import some_tree, tree_seen

NUL = ctypes.c_void_p(0)
FAKE = ctypes.c_void_p(0x1000)


def _covered(q_lens, k_lens, group):
    """Every (query, head) row of every sequence, from the plan's tiles."""
    tiles, counts = _native.packed_plan(q_lens, k_lens, group)
    assert tiles.shape == (counts[0], 8) and counts[0] % 8 == 0
    assert counts[1] == int((tiles[:, 5] > 0).sum()) and counts[2] == max(tiles[:, 5].tolist(), default=0)
    rows = []
    for q0, lq, k0, lk, row0, n, *_ in tiles.tolist():
        if n == 0:
            continue
        assert 0 <= row0 and row0 + n <= lq * group
        rows += [(q0, k0, lq, lk, r) for r in range(row0, row0 + n)]
    return rows


@pytest.mark.parametrize("group", [1, 2, 3, 8])
@pytest.mark.parametrize("q_lens,k_lens", [([1], [1]), ([0, 0], [0, 5]), ([3, 0, 300, 17], [3, 9, 400, 17]),
                                           ([128, 127, 129, 64, 32, 33], [0, 127, 1000, 64, 31, 7]),
                                           (list(range(1, 90)), list(range(1, 90)))])
def test_plan_covers_every_row_once(q_lens, k_lens, group):
    want, q0, k0 = [], 0, 0
    for a, b in zip(q_lens, k_lens):
        want += [(q0, k0, a, b, r) for r in range(a * group)]
        q0, k0 = q0 + a, k0 + b
    assert sorted(_covered(q_lens, k_lens, group)) == sorted(want)


def test_plan_refusals():
    def plan(lq, lk, group=1, cap=0, tiles=None):
        n = len(lq)
        counts = (ctypes.c_int64 * 3)()
        return _native.lib().dg_packed_plan(n, (ctypes.c_int64 * n)(*lq), (ctypes.c_int64 * n)(*lk), group, tiles, cap,
                                            counts)

    assert plan([1], [1]) == 0
    assert plan([-1], [1]) == -1 and b"negative" in _native.lib().dg_last_error()
    assert plan([1], [-1]) == -1
    assert plan([1], [1], group=0) == -1
    assert plan([2**31], [1]) == -1
    assert plan([2**30, 2**30], [1, 1]) == -1 and b"2^31" in _native.lib().dg_last_error()
    assert plan([2**30 + 1], [1]) == -1 and plan([2**29], [1], group=4) == -1
    assert plan([1], [2**30]) == 0
    assert plan([1], [2**30 + 1]) == -1 and b"2^30" in _native.lib().dg_last_error()
    assert plan([1000], [1000], cap=1, tiles=FAKE) == -1 and b"room" in _native.lib().dg_last_error()


def test_layout_refusals():
    with pytest.raises(RuntimeError, match="ROCm"):
        PackedLayout([1], device="cpu")
    with pytest.raises(ValueError, match="lengths"):
        PackedLayout([1, 2], [1], device="cuda")
    with pytest.raises(ValueError, match="negative"):
        PackedLayout([1, -2], device="cuda")
    with pytest.raises(ValueError, match="group"):
        PackedLayout([], group=0, device="cuda")


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64])
def test_tree_masks_name_the_ancestors(n):
    parents = some_tree(n, seed=n)
    masks = tree_masks(parents, device="cpu")
    seen = tree_seen(parents)
    got = torch.stack([(masks >> m) & 1 for m in range(n)], dim=1).bool()
    assert torch.equal(got, seen)
    assert tree_depths(parents) == [int(s.sum()) - 1 for s in seen]


@pytest.mark.parametrize("parents", [[], [0], [-2], [-1, 1], [-1] * 65])
def test_tree_refusals(parents):
    with pytest.raises(ValueError):
        tree_masks(parents, device="cpu")
    with pytest.raises(ValueError):
        tree_depths(parents)


def test_host_tensors_are_refused():
    class Layout:
        group, total_q, total_k, tiles, counts = 1, 2, 2, torch.zeros(8, 8, dtype=torch.int32), None

    x = torch.zeros(2, 1, 16)
    with pytest.raises(RuntimeError, match="ROCm"):
        attention_packed(x, x, x, Layout())
    with pytest.raises(RuntimeError, match="ROCm"):
        attention_tree(x[None], x[None], x[None], 0)
    with pytest.raises(RuntimeError, match="ROCm"):
        token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))


def _st(b=16, t=16, h=16):
    return ctypes.pointer(_native.Stride3(b, t, h))


def _packed(Nq=4, Nk=4, H=1, Hkv=1, D=16, dtype=0, p=FAKE, scale=1.0, tiles=FAKE, counts=(8, 1, 4)):
    counts = None if counts is None else (ctypes.c_int64 * 3)(*counts)
    return _native.lib().dg_attention_packed(Nq, Nk, H, Hkv, D, dtype, p, 16, 16, p, 16, 16, p, 16, 16, p, 16, 16, scale,
                                             tiles, counts, NUL)


def _tree(B=1, N=2, H=1, Hkv=1, Tcap=8, D=16, dtype=0, p=FAKE, scale=1.0, length=3, lens=NUL, ws=NUL, ws_bytes=0):
    return _native.lib().dg_attention_tree(B, N, H, Hkv, Tcap, D, dtype, p, _st(), p, _st(), p, _st(), p, _st(), scale,
                                           length, lens, NUL, 0, ws, ws_bytes, NUL)


@pytest.mark.parametrize("kw,rc", [(dict(Nq=-1), -1), (dict(dtype=9), -2), (dict(D=0), -2), (dict(D=1025), -2),
                                   (dict(H=3, Hkv=2), -1), (dict(Hkv=0), -1), (dict(scale=0.0), -1),
                                   (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(p=NUL), -1),
                                   (dict(tiles=NUL), -1), (dict(counts=None), -1), (dict(counts=(-8, 0, 0)), -1),
                                   (dict(counts=(1, 1, 1)), -1), (dict(counts=(8, 9, 1)), -1),
                                   (dict(counts=(8, 1, 129)), -1), (dict(Nq=0), 0), (dict(counts=(0, 0, 0)), 0), (dict(counts=(8, 0, 0)), 0),
                                   (dict(counts=(8, 1, 0)), 0), (dict(counts=(8, 0, 5), D=7), 0),
                                   (dict(H=0), 0)])
def test_packed_refusals(kw, rc):
    assert _packed(**kw) == rc


@pytest.mark.parametrize("kw,rc", [(dict(B=-1), -1), (dict(dtype=9), -2), (dict(D=0), -2), (dict(D=1025), -2),
                                   (dict(N=0), -1), (dict(N=65, Tcap=100), -1), (dict(Tcap=1), -1), (dict(H=3, Hkv=2), -1),
                                   (dict(scale=-1.0), -1), (dict(length=-1), -1), (dict(length=7), -1), (dict(p=NUL), -1),
                                   (dict(B=0), 0), (dict(H=0), 0), (dict(Tcap=2**30 + 1), -1), (dict(Tcap=2**30), -4),
                                   (dict(Tcap=5000), -4), (dict(Tcap=5000, ws=FAKE, ws_bytes=16), -4)])
def test_tree_entry_refusals(kw, rc):
    assert _tree(**kw) == rc


def test_tree_workspace_size():
    size = _native.lib().dg_attention_tree_workspace_size
    assert size(1, 1, 4, 4, 64, 16, 0) == 0  # one split
    assert size(1, 1, 4, 4, 100000, 16, 0) > 0
    assert size(1, 65, 4, 4, 100000, 16, 0) == 0 and size(0, 1, 4, 4, 100000, 16, 0) == 0
    assert size(1, 1, 4, 3, 100000, 16, 0) == 0
    assert size(1, 1, 4, 4, 2**30, 16, 0) > 0 and size(1, 1, 4, 4, 2**30 + 1, 16, 0) == 0


@pytest.mark.parametrize("kw,rc", [(dict(M=-1), -1), (dict(V=0), -1), (dict(dtype=9), -2), (dict(top=-1), -1),
                                   (dict(top=65), -1), (dict(V=3, top=4), -1), (dict(p=NUL), -1), (dict(V=2**31), -1),
                                   (dict(M=0), 0)])
def test_logprobs_refusals(kw, rc):
    a = dict(M=2, V=100, dtype=0, p=FAKE, top=0) | kw
    p = a["p"]
    assert _native.lib().dg_token_logprobs(a["M"], a["V"], a["dtype"], p, a["V"], p, p, p, a["top"], p, p, NUL) == rc


@pytest.mark.parametrize("counts,Hkv,D,rc", [((8 * (2**21 - 1), 8 * (2**21 - 1), 128), 8, 64, -1), ((2**24, 2**24, 1), 1, 64, -1),
                                             ((2**23, 2**23, 40), 1, 7, -1), ((2**31 - 8, 5, 1), 2**20, 64, -1)])
def test_packed_launches_past_the_grid(counts, Hkv, D, rc):
    """More workgroups than a launch of 2^32 - 1 threads has: refused before anything runs."""
    assert _packed(H=Hkv, Hkv=Hkv, D=D, counts=counts) == rc
    assert b"workgroups" in _native.lib().dg_last_error()


@pytest.mark.parametrize("kw", [dict(B=2**20, H=16, Hkv=16), dict(B=2**23, N=64, H=1, Tcap=64, length=0, D=7),
                                dict(B=2**24, H=4, Hkv=4, dtype=3), dict(B=2**22, N=32, H=4, Hkv=1, Tcap=64)])
def test_tree_launches_past_the_grid(kw):
    """Rows times key heads times row blocks of 32: 2^24 and more."""
    assert _tree(**kw) == -1
    assert b"workgroups" in _native.lib().dg_last_error()


@pytest.mark.parametrize("M,V,top,dtype", [(2**28 + 1, 2, 0, 1), (2**31 - 1, 256, 16, 0), (2**26, 64, 17, 0), (2**26, 1024, 0, 2),
                                           (2**24, 5000, 1, 1), (2**23, 20000, 0, 0), (2**22, 40000, 0, 1), (2**22, 300000, 0, 0),
                                           (2**26, 64, 0, 3)])
def test_logprobs_launches_past_the_grid(M, V, top, dtype):
    assert _native.lib().dg_token_logprobs(M, V, dtype, FAKE, V, FAKE, FAKE, FAKE, top, FAKE, FAKE, NUL) == -1
    assert b"launch" in _native.lib().dg_last_error()


def test_scales_that_overflow_in_log2_units():
    """Accepted, a scale of 3e38 was infinite times log2(e), and a score of 0 NaN."""
    assert _packed(scale=3e38) == -1 and b"scale" in _native.lib().dg_last_error()
    assert _tree(scale=2.4e38) == -1 and b"scale" in _native.lib().dg_last_error()
