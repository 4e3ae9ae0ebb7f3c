"""Timing cases of the operators of a paged cache: many series of different lengths that
decode together, each at its own pace, over pages that come from one pool.

Each case is a dict of plain values; ``op`` says which operator it takes:

  append  the rotation by position and the norm of every query and key head, and the new
          keys and values into the rows' pages
  attend  attention of the rows' newest tokens (one, or a chunk of different lengths) over
          their pages, the query heads in groups that share a key head; with ``weights`` the
          probabilities that each cached position was given are added up as well
  evict   of each row and key head the newest positions and those of the largest added-up
          weights, in order, into fewer pages
  verify  drafted tokens against the target model's probabilities: how many of them stand,
          and the token after them, from random numbers that are given

``run`` with ``own`` false computes them from elementary torch operations in fp32 (fp64 for
the probabilities that decide between tokens); with ``own`` true it calls the framework.
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
_EPS = 2.0**-23  # of the heads' norm


def listed():
    return [
        # one decode step's 32 rows of the small model: latency alone
        dict(name="append_small_f32", op="append", rows=32, new=1, low=2, high=138, heads=4, kv=4, dim=16, page=16,
             dtype="f32", ragged=1),
        # chunks of prompts of different lengths on their way into the pages, grouped heads
        dict(name="append_chunk_bf16", op="append", rows=24, new=700, low=0, high=3500, heads=16, kv=4, dim=128,
             page=64, dtype="bf16", ragged=2),
        # a decode step of the small model's rows
        dict(name="attend_small_f32", op="attend", rows=32, new=1, low=2, high=138, heads=4, kv=4, dim=16, page=16,
             weights=False, dtype="f32", ragged=3),
        # a decode step of 64 rows whose caches differ in length, grouped heads
        dict(name="attend_step_bf16", op="attend", rows=64, new=1, low=1, high=4096, heads=16, kv=4, dim=128, page=64,
             weights=False, dtype="bf16", ragged=4),
        # chunks of long prompts behind what is cached of them
        dict(name="attend_chunk_bf16", op="attend", rows=16, new=512, low=1000, high=7168, heads=16, kv=4, dim=128,
             page=16, weights=False, dtype="bf16", ragged=5),
        # eight drafted tokens a row over two very long caches: the keys' axis has to be split
        dict(name="attend_long_f16", op="attend", rows=2, new=8, low=100001, high=131000, heads=8, kv=2, dim=64,
             page=256, weights=False, dtype="f16", ragged=6),
        # a decode step that also adds up what each position is given
        dict(name="weights_step_bf16", op="attend", rows=48, new=1, low=100, high=4096, heads=16, kv=4, dim=128,
             page=64, weights=True, dtype="bf16", ragged=7),
        # a prompt's last chunk, whose weights choose what stays
        dict(name="weights_chunk_f16", op="attend", rows=8, new=200, low=500, high=4000, heads=8, kv=8, dim=64,
             page=32, weights=True, dtype="f16", ragged=8),
        # the small model's rows cut to 64 positions
        dict(name="evict_small_f32", op="evict", rows=32, low=40, high=200, keep=64, recent=16, kv=4, dim=16, page=16,
             dtype="f32", ragged=9),
        # long prompts cut to a quarter
        dict(name="evict_long_bf16", op="evict", rows=16, low=3000, high=8100, keep=2000, recent=250, kv=4, dim=128,
             page=64, dtype="bf16", ragged=10),
        # four drafts for each of 32 rows of the small vocabulary
        dict(name="verify_small_f32", op="verify", rows=32, drafts=4, vocab=256, certain=False, temperature=1.0,
             dtype="f32", ragged=11),
        # five drafts a row over a large vocabulary of odd size
        dict(name="verify_vocab_bf16", op="verify", rows=64, drafts=5, vocab=49999, certain=False, temperature=0.8,
             dtype="bf16", ragged=12),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; odd more often than not."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n | 1 if rng.random() < 0.6 else n))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "evict", "verify"])
    case = dict(op=op, dtype=rng.choice(["f32", "bf16", "bf16", "f16"]), ragged=rng.randrange(1 << 20))
    if op == "verify":
        drafts, vocab = rng.randint(1, 8), rng.choice([64 * rng.randint(1, 16), _spread(rng, 2000, 131072)])
        most = max(1, min(256, 15_000_000 // (drafts * vocab)))
        return dict(case, rows=_spread(rng, 1, most), drafts=drafts, vocab=vocab, certain=rng.random() < 0.25,
                    temperature=rng.choice([1.0, 1.0, 0.7, 1.3]))
    dim = rng.choice([16, 32, 64, 64, 80, 128, 128])
    kv = rng.randint(1, 8) if dim >= 64 else rng.randint(1, 4)
    heads = kv * rng.choice([1, 1, 2, 3, 4]) if dim >= 64 else kv
    case.update(kv=kv, dim=dim, page=rng.choice([8, 16, 16, 32, 64, 64, 128, 256]))
    if op == "evict":
        high = _spread(rng, 64, 8000)
        keep = rng.randint(max(1, high // 8), max(2, high * 3 // 4))
        return dict(case, rows=_spread(rng, 1, max(2, min(64, 100000 // high))), low=rng.randint(0, high), high=high,
                    keep=keep, recent=rng.randint(0, keep))
    case["heads"] = heads
    if op == "append":
        new = rng.choice([1, _spread(rng, 2, 600)])
        return dict(case, rows=_spread(rng, 1, max(2, min(96, 12000 // new))), new=new, low=0,
                    high=_spread(rng, 16, 3000))
    high = _spread(rng, 64, 20000)
    new = rng.choice([1, 1, rng.randint(2, 9), _spread(rng, 10, 500)])
    rows = _spread(rng, 1, max(2, min(64, 100000 // high, 3_000_000_000 // (new * high * heads * 64))))
    return dict(case, rows=rows, new=new, low=rng.randint(0, high), high=high, weights=rng.random() < 0.35)


def _lengths(case):
    """The rows' cached positions, and of each row how many new tokens (or drafts) it has."""
    rng = random.Random(case["ragged"])
    most = case["drafts"] if case["op"] == "verify" else case.get("new", 0)
    lens = [0 if case["op"] == "verify" else rng.randint(case["low"], case["high"]) for _ in range(case["rows"])]
    # one token in a decode step; chunks and drafts of different lengths, one row's of all
    counts = [most if most <= 1 or i == 0 else rng.randint((most + 1) // 2, most) for i in range(case["rows"])]
    return lens, counts


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _randn(g, dtype, *shape, scale=1.0):
    return torch.empty(shape, dtype=torch.float32, device=_DEV).normal_(0.0, scale, generator=g).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _exponential(g, *shape):
    return torch.empty(shape, dtype=torch.float32, device=_DEV).exponential_(1.0, generator=g)


def _pool(case, g, positions, seed, more=0):
    """Pages for rows of so many positions, and ``more`` further ones for each row: the pool,
    one layer's (pages, page, key heads, dim) keys and values, and tables of page ids in no
    order, -1 behind a row's last page."""
    S, rng = case["page"], random.Random(seed)
    need = [-(-n // S) for n in positions]
    total = sum(need) + more * len(need) + 2
    ids = list(range(total))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(n)] for n in need]
    width = max(1, *need) + 1
    tables = [_ints([t + [-1] * (width - len(t)) for t in table])]
    if more:
        tables.append(_ints([[ids.pop() for _ in range(more)] for _ in need]))
    pages = []
    for _ in range(2):
        page = torch.empty(total, case["kv"], S, case["dim"], dtype=_DTYPES[case["dtype"]], device=_DEV)
        for part in page.split(max(1, (1 << 26) // page[0].numel())):
            part.copy_(_randn(g, part.dtype, *part.shape))
        pages.append(page.transpose(1, 2))
    return pages[0], pages[1], tables


def _angles(case, positions):
    """The (positions, dim / 2, 2) cosines and sines of a rotation of base 10000, in the
    model's type."""
    inv = 10000.0 ** (-torch.arange(0, case["dim"], 2, dtype=torch.float64) / case["dim"])
    a = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], dim=-1).to(_DEV).to(_DTYPES[case["dtype"]])


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
    lens, counts = _lengths(case)
    B = case["rows"]
    if case["op"] == "verify":
        N, V = case["drafts"], case["vocab"]
        # a softcapped head's logits, and a smaller model's that come near them
        raw = _randn(g, torch.float32, B, N + 1, V, scale=0.3)
        st["target"] = (15.0 * torch.tanh(raw)).to(dtype)
        near = raw[:, :N] + _randn(g, torch.float32, B, N, V, scale=0.05)
        draft = (15.0 * torch.tanh(near)).to(dtype)
        race = torch.softmax(draft.float() / case["temperature"], dim=-1) / _exponential(g, B, N, V)
        st["tokens"] = (draft if case["certain"] else race).argmax(-1)  # as the drafting model drew them
        st["draft"] = None if case["certain"] else draft
        st["uniforms"] = torch.empty(B, N, dtype=torch.float32, device=_DEV).uniform_(0.0, 1.0, generator=g)
        st["noise"] = _exponential(g, B, V)
        st["counts"] = _ints(counts)
        return st
    st["lens"] = _ints(lens)
    if case["op"] == "evict":
        st["k"], st["v"], (st["table"], st["to"]) = _pool(case, g, lens, seed, more=-(-case["keep"] // case["page"]))
        # what a prompt's positions were given: most next to nothing, many nothing at all
        x = _randn(g, torch.float32, B, case["kv"], st["table"].size(1) * case["page"])
        st["weights"] = torch.where(x > 0.3, torch.exp(2.0 * x) - 1.0, 0.0)
        return st
    N, H, Hkv, D = case["new"], case["heads"], case["kv"], case["dim"]
    st["k"], st["v"], (st["table"],) = _pool(case, g, [a + b for a, b in zip(lens, counts)], seed)
    st["counts"] = None if N == 1 else _ints(counts)
    if case["op"] == "append":
        # q, k and v are column slices of one projection's rows, as the layers have them
        rows = _randn(g, dtype, B, N, (H + 2 * Hkv) * D)
        st["q"] = rows[..., : H * D].view(B, N, H, D)
        st["k_new"] = rows[..., H * D : (H + Hkv) * D].view(B, N, Hkv, D)
        st["v_new"] = rows[..., (H + Hkv) * D :].view(B, N, Hkv, D)
        st["freqs"] = _angles(case, max(lens) + N)
        return st
    st["q"] = _randn(g, dtype, B, N, H, D)
    if case["weights"]:
        st["weights"] = _randn(g, torch.float32, B, Hkv, st["table"].size(1) * case["page"]).abs_()
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _counts(st):
    B, N = st["q"].shape[:2]
    return torch.full((B,), N, device=_DEV) if st["counts"] is None else st["counts"].long()


def _rotated(x, cs):
    """Pairs of neighbouring dims turned by their angle, and the head's norm."""
    x, cs = x.float(), cs.float()
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = cs[..., 0], cs[..., 1]
    y = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    return y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS)


def _append_plain(st):
    q, S = st["q"], st["case"]["page"]
    B, N = q.shape[:2]
    at = st["lens"].long()[:, None] + torch.arange(N, device=_DEV)  # (B, N)
    cs = st["freqs"][at][:, :, None]
    valid = torch.arange(N, device=_DEV) < _counts(st)[:, None]
    y = torch.where(valid[..., None, None], _rotated(q, cs), 0.0).to(q.dtype)
    k = _rotated(st["k_new"], cs).to(q.dtype)
    b, n = valid.nonzero(as_tuple=True)
    p = at[b, n]
    page = st["table"].long()[b, p // S]
    st["k"][page, p % S] = k[b, n]
    st["v"][page, p % S] = st["v_new"][b, n]
    return y, st["k"], st["v"]


def _attend_plain(st):
    case, q = st["case"], st["q"]
    B, N, H, Hkv, D = case["rows"], case["new"], case["heads"], case["kv"], case["dim"]
    G, T = H // Hkv, st["table"].size(1) * case["page"]
    ids = st["table"].long().clamp(min=0)
    kp = st["k"][ids].reshape(B, T, Hkv, D).permute(0, 2, 3, 1).float().contiguous()
    vp = st["v"][ids].reshape(B, T, Hkv, D).permute(0, 2, 1, 3).float().contiguous()
    qp = q.float().view(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, D)
    n, t = torch.arange(N, device=_DEV), torch.arange(T, device=_DEV)
    valid = n < _counts(st)[:, None]  # (B, N)
    seen = (t <= st["lens"].long()[:, None, None] + n[:, None]) & valid[..., None]  # (B, N, T)
    s = torch.matmul(qp, kp).mul_(D**-0.5).view(B, Hkv, G, N, T)
    s = s.masked_fill_(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    y = torch.matmul(p.view(B, Hkv, G * N, T), vp).view(B, Hkv, G, N, D)
    y = y.permute(0, 3, 1, 2, 4).reshape(B, N, H, D).to(q.dtype)
    return (y, st["weights"] + p.sum((2, 3))) if case["weights"] else y


def _evict_plain(st):
    case = st["case"]
    S, keep, recent = case["page"], case["keep"], case["recent"]
    lens, T = st["lens"].long(), st["table"].size(1) * case["page"]
    B, Hkv = case["rows"], case["kv"]
    t = torch.arange(T, device=_DEV)
    w = torch.where(t < lens[:, None] - recent, 0.0, float("inf"))[:, None] + st["weights"]
    w = torch.where((t < lens[:, None])[:, None], w, float("-inf"))
    _, order = torch.sort(w, dim=-1, descending=True, stable=True)  # ties: the earlier position
    new = lens.clamp(max=keep)
    n = torch.arange(keep, device=_DEV)
    some = (n < new[:, None])[:, None].expand(B, Hkv, keep)
    order = torch.cat([order, order.new_zeros(B, Hkv, max(0, keep - T))], dim=-1)[..., :keep]
    kept = torch.where(some, order, T).sort(-1).values
    at = torch.where(some, kept, 0)
    weights = torch.zeros(B, Hkv, st["to"].size(1) * S, device=_DEV)
    weights[..., :keep] = torch.where(some, st["weights"].gather(-1, at), 0.0)
    b, h, j = some.nonzero(as_tuple=True)
    p = at[b, h, j]
    src, dst = st["table"].long()[b, p // S], st["to"].long()[b, j // S]
    for pages in (st["k"], st["v"]):
        pages[dst, j % S, h] = pages[src, p % S, h]
    return new.int(), weights, torch.where(some, kept, -1).int(), st["k"], st["v"]


def _verify_plain(st):
    case, tokens = st["case"], st["tokens"]
    B, N, T = case["rows"], case["drafts"], case["temperature"]
    counts = st["counts"].long()

    def probabilities(x):
        x = x.double() / T
        e = torch.exp(x - x.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)

    p = probabilities(st["target"])
    px = p[:, :N].gather(-1, tokens[..., None])[..., 0]
    if st["draft"] is None:
        qx = torch.ones_like(px)
    else:
        q = probabilities(st["draft"])
        qx = q.gather(-1, tokens[..., None])[..., 0]
    stands = (st["uniforms"].double() * qx < px) & (torch.arange(N, device=_DEV) < counts[:, None])
    accepted = torch.cumprod(stands.long(), dim=-1).sum(-1)
    b = torch.arange(B, device=_DEV)
    rest, last = p[b, accepted], accepted == counts
    at = accepted.clamp(max=N - 1)
    if st["draft"] is None:
        less = rest.scatter(-1, tokens[b, at][:, None], 0.0)
    else:
        less = (rest - q[b, at]).clamp_(min=0.0)
    rest = torch.where((last | ~(less > 0).any(-1))[:, None], rest, less)
    drawn = (rest / st["noise"].double()).argmax(-1)
    out = torch.cat([tokens, tokens.new_zeros(B, 1)], dim=1)
    n = torch.arange(N + 1, device=_DEV)
    out = torch.where(n < accepted[:, None], out, torch.where(n == accepted[:, None], drawn[:, None], -1))
    logs = torch.log(p.gather(-1, out.clamp(min=0)[..., None])[..., 0])
    return {"accepted": accepted, "tokens": out, "logprobs": torch.where(out >= 0, logs, 0.0).float()}


# ---------------------------------------------------------------------------
# the passes
# ---------------------------------------------------------------------------


@torch.no_grad()
def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "evict": _evict_plain, "verify": _verify_plain}[op](st)
    if op == "verify":
        from diff_gpt.sampler.drafts import verify_drafts

        return verify_drafts(st["target"], st["tokens"], st["uniforms"], st["noise"], draft=st["draft"],
                             counts=st["counts"], temperature=case["temperature"])._asdict()
    from diff_gpt.model import paged

    if op == "append":
        y = paged.append_paged(st["q"], st["k_new"], st["v_new"], st["freqs"], st["k"], st["v"], st["table"],
                               st["lens"], counts=st["counts"])
        return y, st["k"], st["v"]
    if op == "evict":
        r = paged.evict_paged(st["k"], st["v"], st["table"], st["lens"], st["weights"], case["keep"], case["recent"],
                              st["to"])
        return r.lengths, r.weights, r.kept, st["k"], st["v"]
    if not case["weights"]:
        return paged.attention_paged(st["q"], st["k"], st["v"], st["table"], st["lens"], counts=st["counts"])
    weights = st["weights"].clone()  # the call adds to them
    y = paged.attention_paged(st["q"], st["k"], st["v"], st["table"], st["lens"], counts=st["counts"], weights=weights)
    return y, weights


def work(case):
    es = _BYTES[case["dtype"]]
    B = case["rows"]
    lens, counts = _lengths(case)
    if case["op"] == "verify":
        N, V = case["drafts"], case["vocab"]
        rows = (N + 1) * B + (0 if case["certain"] else N * B)
        return {"bytes": rows * V * es + B * V * 4 + B * (N + 1) * 24, "flops": 4 * rows * V}
    Hkv, D = case["kv"], case["dim"]
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        return {"bytes": Hkv * (4 * sum(lens) + kept * (4 * D * es + 8)), "flops": Hkv * sum(lens)}
    H, new = case["heads"], sum(counts)
    if case["op"] == "append":
        return {"bytes": (2 * H + 4 * Hkv) * D * es * new + D * es * new, "flops": 6 * (H + Hkv) * D * new}
    keys = sum(a + b for a, b in zip(lens, counts))
    pairs = sum(a * b + b * (b + 1) // 2 for a, b in zip(lens, counts))
    extra = 8 * Hkv * keys if case["weights"] else 0
    return {"bytes": (2 * keys * Hkv + 2 * new * H) * D * es + extra, "flops": 4 * H * D * pairs}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------


def _row_pages(st, pages, b, n):
    """Positions 0 .. n - 1 of row b."""
    S = st["case"]["page"]
    return pages[st["table"][b, : -(-n // S)].long()].flatten(0, 1)[:n]


def _append_exact(st):
    case = st["case"]
    lens, counts = _lengths(case)
    y = torch.zeros_like(st["q"], dtype=torch.float64)
    k, v = st["k"].double(), st["v"].double()
    for b, (at, n) in enumerate(zip(lens, counts)):
        f = st["freqs"][at : at + n].double()
        z = torch.complex(f[..., 0], f[..., 1])[:, None]
        pos = torch.arange(at, at + n, device=_DEV)
        where = st["table"][b].long()[pos // case["page"]], pos % case["page"]
        for x, out in ((st["q"], None), (st["k_new"], k)):
            r = torch.view_as_real(torch.view_as_complex(x[b, :n].double().unflatten(-1, (-1, 2)).contiguous()) * z)
            r = r.flatten(-2)
            r = r / torch.sqrt(r.square().sum(-1, keepdim=True) / case["dim"] + _EPS)
            if out is None:
                y[b, :n] = r
            else:
                out[where] = r
        v[where] = st["v_new"][b, :n].double()
    return y, k, v


def _attend_exact(st):
    case, q = st["case"], st["q"]
    lens, counts = _lengths(case)
    H, G, D = case["heads"], case["heads"] // case["kv"], case["dim"]
    y = torch.zeros_like(q, dtype=torch.float64)
    weights = st["weights"].double() if case["weights"] else None
    for b, (at, n) in enumerate(zip(lens, counts)):
        k, v = (_row_pages(st, x, b, at + n) for x in (st["k"], st["v"]))
        ahead = torch.arange(at + n, device=_DEV)[None] > at + torch.arange(n, device=_DEV)[:, None]
        for h in range(H):
            s = q[b, :n, h].double() @ k[:, h // G].double().t().contiguous() / math.sqrt(D)
            p = torch.softmax(s.masked_fill(ahead, float("-inf")), dim=-1)
            y[b, :n, h] = p @ v[:, h // G].double().contiguous()
            if weights is not None:
                weights[b, h // G, : at + n] += p.sum(0)
    return y if weights is None else (y, weights)


def _evict_exact(st):
    case = st["case"]
    lens, _ = _lengths(case)
    S, keep, recent = case["page"], case["keep"], case["recent"]
    weights = torch.zeros(case["rows"], case["kv"], st["to"].size(1) * S, dtype=torch.float64, device=_DEV)
    k, v = st["k"].double(), st["v"].double()
    for b, n in enumerate(lens):
        for h in range(case["kv"]):
            w = st["weights"][b, h, :n]
            if n > keep:
                old = w[: n - recent].tolist()
                best = sorted(range(len(old)), key=lambda i: (-old[i], i))[: keep - recent]
                kept = sorted(best) + list(range(n - recent, n))
            else:
                kept = list(range(n))
            if not kept:
                continue
            src = torch.tensor(kept, device=_DEV)
            dst = torch.arange(len(kept), device=_DEV)
            weights[b, h, : len(kept)] = w[src].double()
            for pages, out in ((st["k"], k), (st["v"], v)):
                out[st["to"][b].long()[dst // S], dst % S, h] = pages[st["table"][b].long()[src // S], src % S, h].double()
    return None, weights, None, k, v


def _verify_exact(st):
    case = st["case"]
    _, counts = _lengths(case)
    N, T = case["drafts"], case["temperature"]
    logprobs = torch.zeros(case["rows"], N + 1, dtype=torch.float64, device=_DEV)
    for b, count in enumerate(counts):
        logs = torch.log_softmax(st["target"][b].double() / T, dim=-1)
        drafted = None if st["draft"] is None else torch.softmax(st["draft"][b].double() / T, dim=-1)
        for i in range(count + 1):
            rest = logs[i].exp()
            if i < count:
                x = int(st["tokens"][b, i])
                q = 1.0 if drafted is None else float(drafted[i, x])
                if float(st["uniforms"][b, i]) * q < float(rest[x]):
                    logprobs[b, i] = logs[i, x]
                    continue
                less = rest.clone()
                if drafted is None:
                    less[x] = 0.0
                else:
                    less = torch.clamp(rest - drafted[i], min=0.0)
                rest = less if float(less.max()) > 0.0 else rest
            logprobs[b, i] = logs[i, torch.argmax(rest / st["noise"][b].double())]
            break
    return {"accepted": None, "tokens": None, "logprobs": logprobs}


@torch.no_grad()
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"append": _append_exact, "attend": _attend_exact, "evict": _evict_exact, "verify": _verify_exact}[case["op"]](st)
