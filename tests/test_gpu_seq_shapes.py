"""Which workgroups trees over a cache run on: rows of a workgroup, split or not, exactly."""

import pytest
import torch

from diff_gpt import _native
from diff_gpt.model.tree import attention_tree, tree_masks
from seq_cases import TDT, attend64, close, some_tree, tree_seen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D,B,N,Hkv,G,Tcap,rows,split", [
    ("f32", 16, 2, 60, 1, 3, 70, 32, False), ("bf16", 32, 3, 40, 2, 2, 300, 32, False),
    ("f32", 64, 2, 50, 1, 3, 90, 32, False), ("bf16", 64, 3, 41, 2, 4, 1000, 32, False),
    ("f16", 128, 3, 64, 2, 1, 900, 32, False), ("bf16", 256, 2, 9, 1, 1, 100, 32, False),
    ("f16", 64, 40, 64, 4, 3, 700, 32, False),
    ("f32", 128, 60, 64, 4, 1, 100, 64, True), ("f32", 100, 60, 64, 4, 1, 100, 64, True),
    ("f32", 128, 130, 50, 2, 1, 300, 64, False),
    ("bf16", 64, 65, 33, 4, 1, 1300, 64, True), ("bf16", 56, 65, 33, 4, 1, 1300, 64, True),
    ("f16", 64, 40, 64, 4, 3, 1000, 64, True),
    ("bf16", 128, 64, 50, 4, 3, 700, 64, False), ("f16", 136, 64, 50, 4, 3, 700, 64, False),
    ("bf16", 64, 300, 50, 1, 2, 1200, 64, False), ("f16", 256, 300, 50, 1, 2, 1200, 64, False),
    # 128 rows only where few tiles have many keys, so that all of them are split
    ("f16", 128, 128, 45, 1, 2, 2500, 128, True), ("bf16", 64, 250, 37, 1, 3, 1300, 128, True),
    ("f16", 96, 128, 45, 1, 2, 2500, 128, True), ("bf16", 256, 128, 45, 1, 2, 2500, 128, True),
    ("f16", 64, 255, 64, 1, 2, 1180, 128, True)])
def test_tree_workgroups(dev, dtype, D, B, N, Hkv, G, Tcap, rows, split):
    lens = [(131 * (b + 1)) % (Tcap - N + 1) for b in range(B)]
    g = torch.Generator(device=dev).manual_seed(B)
    q = torch.randn(B, N, Hkv * G, D, generator=g, device=dev).to(TDT[dtype])
    k, v = torch.randn(2, B, Hkv, Tcap, D, generator=g, device=dev).to(TDT[dtype]).transpose(2, 3)
    parents = some_tree(N, seed=B)
    y = attention_tree(q, k, v, torch.tensor(lens, dtype=torch.int32, device=dev), tree_masks(parents))
    ran = [_native.kernel_before(), _native.last_kernel()] if split else [_native.last_kernel()]
    assert ran == [f"seq_mfma_tree_{rows}", "seq_join_kernel"][: 1 + split]
    for b in {0, B // 2, B - 1}:
        n = lens[b]
        seen = torch.cat([torch.ones(N, n, dtype=torch.bool), tree_seen(parents)], dim=1).to(dev)
        ref, mag = attend64(q[b], k[b, : n + N], v[b, : n + N], seen)
        close(y[b], ref, mag, dtype, n + N, float(v[b].abs().max()))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [(1, 1), (3, 2), (24, 3)])
def test_tree_workgroups_of_any_shape(dev, dtype, rows):
    """Heads of 65 dims: the kernel for any shape, with splits and without."""
    N, G = rows
    for Tcap, split in ((200, False), (6000, True)):
        g = torch.Generator(device=dev).manual_seed(N)
        q = torch.randn(2, N, 2 * G, 65, generator=g, device=dev).to(TDT[dtype])
        k, v = torch.randn(2, 2, 2, Tcap, 65, generator=g, device=dev).to(TDT[dtype]).transpose(2, 3)
        y = attention_tree(q, k, v, Tcap - N)
        ran = [_native.kernel_before(), _native.last_kernel()] if split else [_native.last_kernel()]
        assert ran == ["seq_tile_kernel", "seq_join_kernel"][: 1 + split]
        seen = torch.cat([torch.ones(N, Tcap - N, dtype=torch.bool), tree_seen(range(-1, N - 1))], dim=1).to(dev)
        for b in range(2):
            ref, mag = attend64(q[b], k[b], v[b], seen)
            close(y[b], ref, mag, dtype, Tcap, float(v[b].abs().max()))
