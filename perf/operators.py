"""Timing cases of the scoring operators: what it takes to give the likelihoods of many
series of different lengths, and of candidate continuations over cached prompts.

Each case is a dict of plain values; ``op`` says which operator it takes:

  packed   causal attention over packed sequences of different lengths, the query heads
           in groups that share a key head; with ``past`` the sequences' first keys are
           cached ones that have no queries
  tree     a few tokens per row (a tree of candidates, or the one token of a decode step)
           over the row's cache of its own length and over the tokens' own keys, each
           token seeing itself and its ancestors
  logprobs the log probability of a given token per row of logits, the row's entropy and
           its most likely alternatives

``run`` with ``own`` false computes them from elementary torch operations in fp32; with
``own`` true it calls the framework.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DEV = "cuda"
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # 32 series of up to 138 tokens (the small model's window) scored together: the
        # smallest packed batch, bound by latency
        dict(name="packed_small_f32", op="packed", rows=32, low=2, high=138, past=0, heads=4, kv=4, dim=16,
             dtype="f32", ragged=1),
        # a whole panel of series at head_dim 32 (n_embd 128, 4 heads), no length twice
        dict(name="packed_series_bf16", op="packed", rows=512, low=17, high=276, past=0, heads=4, kv=4, dim=32,
             dtype="bf16", ragged=2),
        # longer prompts of very different lengths at the wider model's heads (8 x 64)
        dict(name="packed_ragged_bf16", op="packed", rows=64, low=100, high=2048, past=0, heads=8, kv=8, dim=64,
             dtype="bf16", ragged=3),
        # a few of the longest prompts, 16 query heads on 4 key heads of 128
        dict(name="packed_long_bf16", op="packed", rows=6, low=2000, high=7168, past=0, heads=16, kv=4, dim=128,
             dtype="bf16", ragged=4),
        # chunks of ragged length behind cached keys, 8 query heads on 2 key heads
        dict(name="packed_chunk_f16", op="packed", rows=48, low=1, high=300, past=3000, heads=8, kv=2, dim=64,
             dtype="f16", ragged=5),
        # one decode step of 64 rows whose caches differ in length, grouped heads
        dict(name="step_bf16", op="tree", rows=64, nodes=1, low=1, high=4096, room=64, heads=16, kv=4, dim=128,
             dtype="bf16", ragged=6),
        # trees of 31 scenario tokens over 32 cached series of the small model
        dict(name="tree_scenarios_f32", op="tree", rows=32, nodes=31, low=16, high=138, room=138, heads=4, kv=4,
             dim=16, dtype="f32", ragged=7),
        # drafted trees of 24 tokens over long prompts, grouped heads
        dict(name="tree_draft_bf16", op="tree", rows=16, nodes=24, low=1000, high=7168, room=64, heads=16, kv=4,
             dim=128, dtype="bf16", ragged=8),
        # the widest tree over two very long caches: few rows, the keys' axis has to be split
        dict(name="tree_long_f16", op="tree", rows=2, nodes=64, low=100001, high=131000, room=72, heads=8, kv=2,
             dim=64, dtype="f16", ragged=9),
        # one step's 32 rows of the small vocabulary
        dict(name="logprobs_small_f32", op="logprobs", rows=32, vocab=256, top=5, dtype="f32"),
        # 256 windows of 138 tokens scored at once
        dict(name="logprobs_series_bf16", op="logprobs", rows=35328, vocab=256, top=8, dtype="bf16"),
        # prompts over a large vocabulary of odd size: no row but the first is aligned
        dict(name="logprobs_vocab_bf16", op="logprobs", rows=2048, vocab=49999, top=20, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; odd more often than not."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n | 1 if rng.random() < 0.6 else n))


def draw(rng):
    op = rng.choice(["packed", "packed", "packed", "tree", "tree", "tree", "logprobs", "logprobs"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    ragged = rng.randrange(1 << 20)
    if op == "logprobs":
        if rng.random() < 0.4:
            return dict(op=op, rows=_spread(rng, 1, 35000), vocab=64 * rng.randint(1, 16), top=rng.randint(0, 16),
                        dtype=dtype)
        return dict(op=op, rows=_spread(rng, 1, 500), vocab=_spread(rng, 2000, 131072), top=rng.randint(0, 32),
                    dtype=dtype)
    dim = rng.choice([16, 32, 64, 64, 128, 128])
    kv = rng.randint(1, 8) if dim >= 64 else rng.randint(1, 4)
    heads = kv * rng.choice([1, 1, 2, 3, 4]) if dim >= 64 else kv
    if op == "packed":
        high = _spread(rng, 32, 3000 if dim >= 64 else 500)
        rows = _spread(rng, 1, max(2, min(256, 40000 // high)))
        past = rng.choice([0, 0, 0, _spread(rng, 10, 2000)])
        return dict(op=op, rows=rows, low=rng.randint(1, high), high=high, past=past, heads=heads, kv=kv, dim=dim,
                    dtype=dtype, ragged=ragged)
    high = _spread(rng, 64, 20000)
    rows = _spread(rng, 1, max(2, min(64, 100000 // high)))
    return dict(op=op, rows=rows, nodes=rng.choice([1, 1, rng.randint(2, 64)]), low=rng.randint(0, high), high=high,
                room=64 + rng.randint(0, 40), heads=heads, kv=kv, dim=dim, dtype=dtype, ragged=ragged)


def _lengths(case):
    """The rows' lengths, and for packed ones those of their cached keys."""
    rng = random.Random(case["ragged"])
    lens = [rng.randint(case["low"], case["high"]) for _ in range(case["rows"])]
    past = [rng.randint(0, case["past"]) if case.get("past") else 0 for _ in lens]
    return lens, past


def _parents(case):
    """One tree for the rows: node n hangs on an earlier node, or (-1) on the cached row."""
    rng = random.Random(case["ragged"] + 1)
    return [rng.randint(max(-1, n - 6), n - 1) if n else -1 for n in range(case["nodes"])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _randn(g, dtype, *shape, scale=1.0):
    return torch.empty(shape, dtype=torch.float32, device=_DEV).normal_(0.0, scale, generator=g).to(dtype)


def _starts(lens):
    return torch.tensor([0, *lens], dtype=torch.int64).cumsum(0).to(_DEV)


@torch.no_grad()
def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    st = {"case": case}
    if own:
        pkg = str(Path(__file__).resolve().parent.parent / "diff-gpt_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
    if case["op"] == "logprobs":
        M, V = case["rows"], case["vocab"]
        # a softcapped head's logits: up to 15 either way
        st["logits"] = (15.0 * torch.tanh(_randn(g, torch.float32, M, V, scale=0.2))).to(dtype)
        st["ids"] = torch.randint(0, V, (M,), generator=g, device=_DEV)
        return st
    H, Hkv, D = case["heads"], case["kv"], case["dim"]
    lens, past = _lengths(case)
    if case["op"] == "packed":
        k_lens = [a + b for a, b in zip(lens, past)]
        n, nk = sum(lens), sum(k_lens)
        # q, k and v are column slices of one projection's rows, as the layers have them
        # (keys behind cached ones are gathered into rows of their own)
        if nk == n:
            rows = _randn(g, dtype, n, (H + 2 * Hkv) * D)
            st["q"] = rows[:, : H * D].view(n, H, D)
            st["k"] = rows[:, H * D : (H + Hkv) * D].view(n, Hkv, D)
            st["v"] = rows[:, (H + Hkv) * D :].view(n, Hkv, D)
        else:
            st["q"] = _randn(g, dtype, n, H, D)
            st["k"] = _randn(g, dtype, nk, Hkv, D)
            st["v"] = _randn(g, dtype, nk, Hkv, D)
        st["q_starts"], st["k_starts"] = _starts(lens), _starts(k_lens)
        st["longest"] = max(lens), max(k_lens)
        if own:
            from diff_gpt.model.packed import PackedLayout

            st["layout"] = PackedLayout(lens, k_lens, group=H // Hkv, device=_DEV)
        return st
    B, N = case["rows"], case["nodes"]
    cap = max(lens) + max(N, case["room"])
    # one layer's pages of a cache, (B, Hkv, positions, D), seen as (B, positions, Hkv, D)
    pages = torch.empty(2, B, Hkv, cap, D, dtype=dtype, device=_DEV)
    for page in pages.view(2 * B, Hkv, cap, D):
        page.copy_(_randn(g, dtype, Hkv, cap, D))
    st["k"], st["v"] = pages[0].transpose(1, 2), pages[1].transpose(1, 2)
    st["q"] = _randn(g, dtype, B, N, H, D)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=_DEV)
    # which nodes a node sees: itself and its ancestors, one bit each
    masks = []
    for n, p in enumerate(_parents(case)):
        masks.append((1 << n) | (masks[p] if p >= 0 else 0))
    st["masks"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device=_DEV)
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _softmax_rows(s, seen):
    """exp(s - max) over the seen entries and its sums; rows that see nothing give zeros."""
    s = torch.where(seen, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _packed_plain(st):
    """The sequences padded to the longest one, as one batch of masked products."""
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    S, H, Hkv, D = case["rows"], case["heads"], case["kv"], case["dim"]
    qs, ks = st["q_starts"], st["k_starts"]
    Lq, Lk = st["longest"]
    nq, nk = (qs[1:] - qs[:-1])[:, None], (ks[1:] - ks[:-1])[:, None]
    iq, ik = torch.arange(Lq, device=_DEV)[None], torch.arange(Lk, device=_DEV)[None]
    qp = q[(qs[:-1, None] + iq).clamp(max=q.size(0) - 1)].float()  # (S, Lq, H, D)
    kp = k[(ks[:-1, None] + ik).clamp(max=k.size(0) - 1)].float()
    vp = v[(ks[:-1, None] + ik).clamp(max=v.size(0) - 1)].float()
    G = H // Hkv
    qp = qp.view(S, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * Lq, D)
    kp = kp.permute(0, 2, 3, 1).contiguous()  # (S, Hkv, D, Lk)
    vp = vp.permute(0, 2, 1, 3).contiguous()
    seen = (ik[:, None] <= iq[:, :, None] + (nk - nq)[:, :, None]) & (ik < nk)[:, None]  # (S, Lq, Lk)
    s = torch.matmul(qp, kp).mul_(D**-0.5).view(S, Hkv, G, Lq, Lk)
    p = _softmax_rows(s, seen[:, None, None]).view(S, Hkv, G * Lq, Lk)
    y = torch.matmul(p, vp).view(S, Hkv, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(S, Lq, H, D)
    row = torch.arange(q.size(0), device=_DEV)
    seq = torch.searchsorted(qs, row, right=True) - 1
    return y[seq, row - qs[seq]].to(q.dtype)


def _tree_plain(st):
    case, q = st["case"], st["q"]
    B, N, H, Hkv, D = case["rows"], case["nodes"], case["heads"], case["kv"], case["dim"]
    G, T = H // Hkv, st["k"].size(1)
    lens = st["lens"].long()[:, None, None]
    qp = q.float().view(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, D)
    kp = st["k"].float().permute(0, 2, 3, 1).contiguous()
    vp = st["v"].float().permute(0, 2, 1, 3).contiguous()
    t = torch.arange(T, device=_DEV)[None, None]
    node = t - lens  # (B, 1, T): which node's key a position holds
    bits = (st["masks"][None, :, None] >> node.clamp(0, 63)) & 1
    seen = (node < 0) | ((node < N) & (bits == 1))  # (B, N, T)
    s = torch.matmul(qp, kp).mul_(D**-0.5).view(B, Hkv, G, N, T)
    p = _softmax_rows(s, seen[:, None, None]).view(B, Hkv, G * N, T)
    y = torch.matmul(p, vp).view(B, Hkv, G, N, D).permute(0, 3, 1, 2, 4)
    return y.reshape(B, N, H, D).to(q.dtype)


def _logprobs_plain(st):
    x, ids, k = st["logits"].float(), st["ids"], st["case"]["top"]
    z = x - x.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    logs = z - torch.log(total)
    entropy = (torch.log(total) - (e * z).sum(-1, keepdim=True) / total).squeeze(-1)
    out = {"logprobs": logs.gather(-1, ids[:, None]).squeeze(-1), "entropy": entropy}
    if k:
        _, order = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lowest id first
        out["top_ids"] = order[:, :k].contiguous()
        out["top_logprobs"] = logs.gather(-1, out["top_ids"])
    return out


# ---------------------------------------------------------------------------
# the passes
# ---------------------------------------------------------------------------


@torch.no_grad()
def run(st):
    op = st["case"]["op"]
    if not own:
        return {"packed": _packed_plain, "tree": _tree_plain, "logprobs": _logprobs_plain}[op](st)
    if op == "packed":
        from diff_gpt.model.packed import attention_packed

        return attention_packed(st["q"], st["k"], st["v"], st["layout"])
    if op == "tree":
        from diff_gpt.model.tree import attention_tree

        return attention_tree(st["q"], st["k"], st["v"], st["lens"], st["masks"])
    from diff_gpt.model.token_logprobs import token_logprobs

    r = token_logprobs(st["logits"], st["ids"], top=st["case"]["top"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if st["case"]["top"]:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


def work(case):
    es = _BYTES[case["dtype"]]
    if case["op"] == "logprobs":
        M, V = case["rows"], case["vocab"]
        return {"bytes": M * V * es + M * (8 + 8 + 12 * case["top"]), "flops": 4 * M * V}
    H, Hkv, D = case["heads"], case["kv"], case["dim"]
    lens, past = _lengths(case)
    if case["op"] == "packed":
        n, nk = sum(lens), sum(lens) + sum(past)
        pairs = sum(a * (a + 1) // 2 + a * b for a, b in zip(lens, past))
        return {"bytes": (2 * n * H + 2 * nk * Hkv) * D * es, "flops": 4 * H * D * pairs}
    B, N = case["rows"], case["nodes"]
    keys = sum(lens) + B * N
    seen = 0
    depth = []
    for p in _parents(case):
        depth.append(1 + (depth[p] if p >= 0 else 0))
    seen = N * sum(lens) + B * sum(depth)
    return {"bytes": (2 * keys * Hkv + 2 * B * N * H) * D * es, "flops": 4 * H * D * seen}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------


def _attend(q, k, v, seen):
    """Softmax attention of (n, Hkv, G, D) queries over (t, Hkv, D) keys in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    y = torch.zeros_like(q)
    any_key = seen.any(-1)
    for h in range(k.size(1)):
        for g in range(q.size(2)):
            s = q[:, h, g] @ k[:, h].t().contiguous() / math.sqrt(q.size(-1))
            p = torch.softmax(s.masked_fill(~seen, float("-inf")), dim=-1)
            y[:, h, g] = torch.where(any_key[:, None], p @ v[:, h].contiguous(), 0.0)
    return y


@torch.no_grad()
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "logprobs":
        outs = []
        for x, ids in zip(st["logits"].split(512), st["ids"].split(512)):
            logs = torch.log_softmax(x.double(), dim=-1)
            p = logs.exp()
            outs.append((logs.gather(-1, ids[:, None])[:, 0], -(p * logs).sum(-1),
                         torch.topk(logs, case["top"], dim=-1).values if case["top"] else None))
        out = {"logprobs": torch.cat([o[0] for o in outs]), "entropy": torch.cat([o[1] for o in outs])}
        if case["top"]:
            out["top_ids"] = None
            out["top_logprobs"] = torch.cat([o[2] for o in outs])
        return out
    H, Hkv, D = case["heads"], case["kv"], case["dim"]
    lens, past = _lengths(case)
    if case["op"] == "packed":
        ys, a, b = [], 0, 0
        for n, m in zip(lens, past):
            i, j = torch.arange(n, device=_DEV)[:, None], torch.arange(n + m, device=_DEV)[None]
            q = st["q"][a : a + n].reshape(n, Hkv, H // Hkv, D)
            ys.append(_attend(q, st["k"][b : b + n + m], st["v"][b : b + n + m], j <= i + m).reshape(n, H, D))
            a, b = a + n, b + n + m
        return torch.cat(ys)
    N, parents = case["nodes"], _parents(case)
    among = torch.zeros(N, N, dtype=torch.bool)
    for n in range(N):
        at = n
        while at >= 0:
            among[n, at] = True
            at = parents[at]
    ys = []
    for r, n in enumerate(lens):
        seen = torch.cat([torch.ones(N, n, dtype=torch.bool), among], dim=1).to(_DEV)
        q = st["q"][r].reshape(N, Hkv, H // Hkv, D)
        ys.append(_attend(q, st["k"][r, : n + N], st["v"][r, : n + N], seen).reshape(N, H, D))
    return torch.stack(ys)
