"""Pages, tables and 64-bit answers of the paged cache's tests."""

import random

import torch

from seq_cases import TDT, attend64


class Pool:
    """Rows of ``lens`` cached positions and ``counts`` tokens behind them in pages of S of one
    pool: positions hold random numbers, everything else (other pages, the places behind a
    row's end) NaN; pages are in no order, a row's table ends in ids that the pool lacks."""

    def __init__(self, dev, dtype, lens, counts, Hkv, D, S, seed=0, spare=2, head_major=True):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.lens, self.counts, self.S = lens, counts, S
        need = [-(-(a + b) // S) for a, b in zip(lens, counts)]
        total = sum(need) + spare
        ids = list(range(total))
        rng.shuffle(ids)
        self.pages_of = [[ids.pop() for _ in range(n)] for n in need]
        self.free = ids
        width = max(1, *need) + 1
        bad = [-1, total, 2**31 - 1, -(2**31)]
        self.table_host = [p + [bad[(i + len(p)) % 4] for i in range(width - len(p))] for p in self.pages_of]
        self.k_rows, self.v_rows = [], []
        shape = (total, Hkv, S, D) if head_major else (total, S, Hkv, D)
        k = torch.full(shape, float("nan"), dtype=torch.float64)
        v = torch.full(shape, float("nan"), dtype=torch.float64)
        kk, vv = (x.transpose(1, 2) if head_major else x for x in (k, v))
        for b, (a, c) in enumerate(zip(lens, counts)):
            n = a + c
            kr, vr = (torch.randn(n, Hkv, D, generator=g, dtype=torch.float64).to(TDT[dtype]) for _ in range(2))
            self.k_rows.append(kr.to(dev))
            self.v_rows.append(vr.to(dev))
            for t in range(0, n, S):
                m = min(S, n - t)
                kk[self.pages_of[b][t // S], :m] = kr[t : t + m].double()
                vv[self.pages_of[b][t // S], :m] = vr[t : t + m].double()
        k, v = k.to(TDT[dtype]).to(dev), v.to(TDT[dtype]).to(dev)
        self.k, self.v = (x.transpose(1, 2) if head_major else x for x in (k, v))
        self.table = torch.tensor(self.table_host, dtype=torch.int32, device=dev)
        self.lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.new = torch.tensor(counts, dtype=torch.int32, device=dev)


def attend_rows(q, pool):
    """y (B, N, H, D) and its |v| companion (attend64), and each row's (Hkv, positions) weights and
    the sum of |q||k| that their error is relative to."""
    B, N, H, D = q.shape
    y, a = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    weights, most = [], 0.0
    for b, (at, n) in enumerate(zip(pool.lens, pool.counts)):
        k, v = pool.k_rows[b], pool.v_rows[b]
        Hkv = k.size(1)
        w = torch.zeros(Hkv, at + n, dtype=torch.float64, device=q.device)
        if n:
            seen = torch.arange(at + n, device=q.device)[None] <= at + torch.arange(n, device=q.device)[:, None]
            y[b, :n], a[b, :n] = attend64(q[b, :n], k, v, seen)
            for h in range(H):
                kh = k[:, h // (H // Hkv)].double()
                s = (q[b, :n, h].double() @ kh.t().contiguous()) * D**-0.5
                s = s.masked_fill(~seen, float("-inf"))
                p = torch.exp(s - s.amax(-1, keepdim=True))
                w[h // (H // Hkv)] += (p / p.sum(-1, keepdim=True)).sum(0)
                most = max(most, float((q[b, :n, h].double().abs() @ kh.abs().t().contiguous()).max()) * D**-0.5)
        weights.append(w)
    return y, a, weights, most
