"""The operators of verifying trees of drafted tokens and of evicting positions from a paged cache by their accumulated attention weight, as
they are measured: which rows of a step see each other, attention over pages of 16 and 32 bits, the attention weights summed by cached
position, the positions that stay, the rows of the pages that move together, and the drafts that the model accepts.

A cache is two arrays [pages, kv_heads, page_size, dim], keys and values, and a page table [slots, pages of a slot].  A sequence's step has
`rows` rows, the last of its context's positions.  Row i sees every position before the step and, of the step's rows, those whose bit is set
in its mask (bit j % 32 of word j // 32 for row j): in a tree its ancestors and itself, without masks itself and the rows before it.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
F32, F64, I32, I64 = torch.float32, torch.float64, torch.int32, torch.int64
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------------- the cases
def listed() -> list[dict]:
    return [
        # one request of an 8B decoder, a tree of eight drafts over a short context: the smallest call, latency counts; its masks are made on the way
        dict(name="tree_1x8", kind="tree", seqs=1, rows=8, ctx=1000, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16", shape="wide", masks=True),
        # eight requests of it with full trees
        dict(name="tree_8x64", kind="tree", seqs=8, rows=64, ctx=4100, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16", shape="wide",
             masks=False),
        # one request of a 70B decoder with a long context
        dict(name="tree_1x26_32k", kind="tree", seqs=1, rows=26, ctx=32000, heads=64, kv_heads=8, dim=128, page=64, dtype="bfloat16", shape="wide",
             masks=False),
        # float16 on pages of 16 positions, sixteen requests of unequal lengths, their masks made on the way
        dict(name="tree_16x13_f16", kind="tree", seqs=16, rows=13, ctx=2001, heads=32, kv_heads=4, dim=128, page=16, dtype="float16", shape="deep",
             masks=True),
        # a float32 cache
        dict(name="tree_4x21_f32", kind="tree", seqs=4, rows=21, ctx=1500, heads=16, kv_heads=4, dim=64, page=64, dtype="float32", shape="wide",
             masks=False),
        # one request decodes a token, and the weights of its positions are summed
        dict(name="weigh_1x4096", kind="weigh", seqs=1, rows=1, ctx=4096, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16"),
        # a full batch of a 70B decoder over long contexts: the bytes of the cache
        dict(name="weigh_64x8192", kind="weigh", seqs=64, rows=1, ctx=8192, heads=64, kv_heads=8, dim=128, page=64, dtype="bfloat16"),
        # the last 32 tokens of a prompt, portion of it, look back on the whole
        dict(name="observe_32_16k", kind="weigh", seqs=1, rows=32, ctx=16384, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16"),
        # one layer of one request is cut to half
        dict(name="evict_1x4096", kind="evict", seqs=1, ctx=4096, budget=2048, first=4, recent=512, kv_heads=8, dim=128, page=64, dtype="bfloat16"),
        # one layer of sixteen requests
        dict(name="evict_16x8192", kind="evict", seqs=16, ctx=8192, budget=4096, first=4, recent=1000, kv_heads=8, dim=128, page=64, dtype="bfloat16"),
        # one request's drafts are accepted in 36 layers, with a vocabulary of 151936
        dict(name="accept_1x26", kind="accept", seqs=1, rows=26, ctx=2001, arrays=72, vocab=151936, kv_heads=8, dim=128, page=64, dtype="bfloat16",
             shape="wide"),
        # sixteen requests' full trees in 32 layers
        dict(name="accept_16x64", kind="accept", seqs=16, rows=64, ctx=600, arrays=64, vocab=128256, kv_heads=8, dim=128, page=64, dtype="bfloat16",
             shape="wide"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """a number in lo ... hi, spread over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 8), (64, 8), (32, 4), (16, 4), (16, 16), (12, 3), (8, 1), (4, 2)]


def draw(rng) -> dict:
    kind = rng.choice(["tree", "tree", "tree", "tree", "weigh", "weigh", "weigh", "evict", "evict", "accept", "accept"])
    dim = rng.choice([128, 128, 128, 64, 96, 256, 80])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    page = rng.choice([64, 64, 16, 32, 128, 48, 100, 0])              # 0: one page of a fixed length for each sequence
    heads, kv = rng.choice(HEADS)
    shape = rng.choice(["wide", "wide", "deep"])
    if kind in ("tree", "weigh"):
        seqs = _log(rng, 1, 16 if kind == "tree" else 64)
        rows = _log(rng, 1, 128 if dtype != "float32" else 32) if kind == "tree" else rng.choice([1, 1, _log(rng, 2, 64)])
        most = min(32768, 300_000_000 // (seqs * kv * dim), 12_000_000_000 // (seqs * heads * dim * rows))
        c = dict(kind=kind, seqs=seqs, rows=rows, ctx=rows + _log(rng, 1, max(64, most)) - 1, heads=heads, kv_heads=kv, dim=dim, page=page, dtype=dtype)
        return dict(c, shape=shape, masks=rng.random() < 0.3) if kind == "tree" else c
    if kind == "evict":
        seqs = _log(rng, 1, 16)
        ctx = _log(rng, 100, min(32768, 250_000_000 // (seqs * kv * dim)))
        budget = max(2, int(ctx * rng.uniform(0.2, 0.9)))
        recent = int(budget * rng.uniform(0.0, 0.6))
        return dict(kind=kind, seqs=seqs, ctx=ctx, budget=budget, first=rng.choice([0, 1, 4]) if budget - recent > 4 else 0, recent=recent, kv_heads=kv,
                    dim=dim, page=page, dtype=dtype)
    seqs, rows = _log(rng, 1, 16), _log(rng, 1, 64)
    return dict(kind=kind, seqs=seqs, rows=rows, ctx=rows + _log(rng, 1, 500), arrays=rng.choice([2, 24, 64]), vocab=_log(rng, 1000, 151936),
                kv_heads=min(kv, 8), dim=dim, page=page, dtype=dtype, shape=shape)


# ---------------------------------------------------------------------------------------------------- inputs
class _Gen:
    """tensors of one case, in the order in which they are asked for"""

    def __init__(self, seed: int):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 6271 + 29)

    def normal(self, *shape, std=1.0, dtype=F32):
        return (torch.randn(*shape, generator=self.g, device=DEV) * std).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=DEV)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def _rows(c) -> list[int]:
    """rows of every sequence's step: of several, unequal ones"""
    n = c.get("rows", 0)
    return [max(1, n - (n // 4) * (i % 3)) for i in range(c["seqs"])] if n else [0] * c["seqs"]


def _contexts(c) -> list[int]:
    """positions of every sequence with the step's: the last one has the most"""
    span = max(0, c["ctx"] - c.get("rows", 1))
    return [c["ctx"] - (41 * i * i) % (span // 4 + 1) for i in range(c["seqs"] - 1, -1, -1)]


def _trees(c, seed: int) -> list[list[int]]:
    """every sequence's parents: row 0 is the last token that was accepted, the others hang on a row before them"""
    r = random.Random(seed * 31 + c["rows"])
    out = []
    for n in _rows(c):
        p = [-1]
        for i in range(1, n):
            p.append(r.randrange(max(0, i - 3), i) if c["shape"] == "deep" else r.randrange(max(0, (i - 1) // 3 - 2), (i + 2) // 3))
        out.append(p)
    return out


def _starts(rows: list[int]) -> list[int]:
    s = [0]
    for n in rows:
        s.append(s[-1] + n)
    return s


def _pages(g: _Gen, c, arrays: int) -> tuple:
    """(arrays of pages, page table, slots): a cache filled by earlier steps, its pages in any order"""
    most = max(_contexts(c))
    ps = c["page"] or most + 37
    per = -(-most // ps)
    used = c["seqs"] * per
    table = g.perm(used).view(c["seqs"], per).to(I32)
    slots = g.perm(c["seqs"]).to(I32)
    shape, dt = (used, c["kv_heads"], ps, c["dim"]), TYPES[c["dtype"]]
    pages = torch.empty(arrays, *shape, dtype=dt, device=DEV)
    flat = pages.view(-1)
    for at in range(0, flat.numel(), 1 << 27):
        n = min(1 << 27, flat.numel() - at)
        flat[at:at + n] = g.normal(n)
    return pages, table, slots


def prepare(case: dict, seed: int) -> dict:
    c = {k: v for k, v in case.items() if k != "name"}
    g, kind = _Gen(seed), c["kind"]
    ctx, rows = _contexts(c), _rows(c)
    s = dict(case=c)
    pages, s["table"], s["slots"] = _pages(g, c, c.get("arrays", 2))
    s["pages"], s["k_cache"], s["v_cache"] = pages, pages[0], pages[1]
    s["ctx"], s["max_ctx"] = _i32(ctx), max(ctx)
    if kind != "evict":
        s["first"], s["max_rows"] = _i32(_starts(rows)), max(rows)
        T = sum(rows)
    if kind in ("tree", "accept"):
        trees = _trees(c, seed)
        s["parents"] = _i32([p for t in trees for p in t])
        words = -(-s["max_rows"] // 32)
        s["masks"], s["depths"] = torch.empty(T, words, dtype=I32, device=DEV), torch.empty(T, dtype=I32, device=DEV)
    if kind in ("tree", "weigh"):
        dt = TYPES[c["dtype"]]
        s["q"] = g.normal(T, c["heads"], c["dim"], std=1.5, dtype=dt)
        s["out"] = torch.empty_like(s["q"])
        if kind == "weigh":
            s["lse"] = torch.empty(T, c["heads"], dtype=F32, device=DEV)
            s["weights"] = g.uniform(c["seqs"], c["kv_heads"], s["max_ctx"]) ** 8
        elif not c["masks"]:
            s["masks"], s["depths"] = _masks_plain(s)
    elif kind == "evict":
        # sums of many steps' weights: most positions have little, a few have most
        s["weights"] = -torch.log(g.uniform(c["seqs"], c["kv_heads"], s["max_ctx"]).clamp(min=1e-7)) ** 3
        s["kept"] = (torch.empty(c["seqs"], c["kv_heads"], c["budget"], dtype=I32, device=DEV), torch.empty(c["seqs"], dtype=I32, device=DEV))
    else:
        V = c["vocab"]
        s["tokens"] = (g.uniform(T) * V).to(I32)
        x = g.normal(T, V, std=2.0)
        # seven of ten rows go on to one of their drafts
        r = random.Random(seed)
        at, tok, base = [], [], 0
        tokens = s["tokens"].tolist()
        for t in trees:
            for i, p in enumerate(t):
                if p >= 0 and r.random() < 0.7:
                    at.append(base + p)
                    tok.append(tokens[base + i])
            base += len(t)
        if at:
            x[torch.tensor(at, device=DEV), torch.tensor(tok, device=DEV)] += 12.0
        s["logits"] = x.to(torch.bfloat16)
        s["committed"] = _i32([m - n for m, n in zip(ctx, rows)])
        s["accepted"] = (torch.empty(c["seqs"], s["max_rows"], dtype=I32, device=DEV), torch.empty(c["seqs"], dtype=I32, device=DEV),
                         torch.empty(c["seqs"], dtype=I32, device=DEV))
    return s


# ---------------------------------------------------------------------------------------------------- the plain forms
def _ancestors(s):
    """[sequences, rows, rows]: whether row j is row i or one that it hangs on; with one more sequence and row for those that do not exist"""
    first, parents, R = s["first"].long(), s["parents"].long(), s["max_rows"]
    T = parents.shape[0]
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(first[1:].contiguous(), t, right=True)
    i = t - first[seq]
    up = torch.zeros(first.shape[0] - 1, R, R, dtype=F64, device=DEV)
    has = parents >= 0
    up[seq[has], i[has], parents[has]] = 1.0
    reach = torch.linalg.inv(torch.eye(R, dtype=F64, device=DEV) - up)          # 1 + up + up^2 + ...: a forest has one way from a row to another
    return reach.round() > 0.5, seq, i


def _masks_plain(s):
    reach, seq, i = _ancestors(s)
    R = s["max_rows"]
    words = -(-R // 32)
    mine = torch.nn.functional.pad(reach[seq, i], (0, 32 * words - R)).unflatten(1, (words, 32)).to(I64)
    masks = (mine << torch.arange(32, device=DEV)).sum(-1)
    masks = torch.where(masks >= 1 << 31, masks - (1 << 32), masks).to(I32)
    return masks, (reach[seq, i].sum(1) - 1).to(I32)


def _scores_plain(s, seen_step):
    """(scores [S, H, rep R, keys], rows that exist [S, R], positions of the step's rows in the queries): float32, -infinity where unseen"""
    c = s["case"]
    H, rep, R = c["kv_heads"], c["heads"] // c["kv_heads"], s["max_rows"]
    first, ctx = s["first"].long(), s["ctx"].long()
    pages = s["table"].long()[s["slots"].long()]
    k = s["k_cache"][pages].transpose(1, 2).flatten(2, 3).to(F32)                                         # [S, H, keys, D]
    n = first[1:] - first[:-1]
    i = torch.arange(R, device=DEV)
    live = i < n[:, None]
    at = (first[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].to(F32).unflatten(2, (H, rep)).permute(0, 2, 3, 1, 4).flatten(2, 3)                     # [S, H, rep R, D]
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(c["dim"]))
    j = torch.arange(k.shape[2], device=DEV) - (ctx - n)[:, None]                                         # a key's row in the step
    inside = (j >= 0) & (j < n[:, None])
    mine = seen_step.gather(2, j.clamp(0, R - 1)[:, None].expand(-1, R, -1))
    seen = torch.where(inside[:, None], mine, (j < 0)[:, None])                                           # [S, R, keys]
    return x.unflatten(2, (rep, R)).masked_fill(~seen[:, None, None], -math.inf), live, pages


def _attend_plain(s, seen_step):
    x, live, pages = _scores_plain(s, seen_step)
    v = s["v_cache"][pages].transpose(1, 2).flatten(2, 3).to(F32)
    top = x.amax(-1, keepdim=True).clamp(min=-3e38)
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    o = (w.flatten(2, 3) @ v).unflatten(2, w.shape[2:4]) / total
    lse = (top + torch.log(total))[..., 0]
    out = o.permute(0, 3, 1, 2, 4)[live].flatten(1, 2).to(s["q"].dtype)
    return out, lse.permute(0, 3, 1, 2)[live].flatten(1, 2), w / total, live


def _tree_plain(s):
    c = s["case"]
    masks, depths = _masks_plain(s) if c["masks"] else (s["masks"], s["depths"])
    R, first = s["max_rows"], s["first"].long()
    at = (first[:-1, None] + torch.arange(R, device=DEV)).clamp(max=masks.shape[0] - 1)
    j = torch.arange(R, device=DEV)
    seen = (masks.long()[at][:, :, j // 32] >> (j % 32)) & 1 > 0
    out = _attend_plain(s, seen)[0]
    return [out, masks, depths] if c["masks"] else out


def _weigh_plain(s):
    R = s["max_rows"]
    i = torch.arange(R, device=DEV)
    seen = (i <= i[:, None]).expand(s["case"]["seqs"], R, R)
    out, lse, p, live = _attend_plain(s, seen)
    p = p.masked_fill(~live[:, None, None, :, None], 0.0).sum((2, 3))                                       # [S, H, keys]
    s["weights"][s["slots"].long()] += p[..., :s["weights"].shape[2]]
    return [out, lse, s["weights"]]


def _gone_to_front(pages, row_at, to, live):
    """pages [arrays, pages, H, ps, ...]: position `to` of a sequence's pages becomes what `row_at` was; [S, H, m] with their page and row each"""
    (sp, sr), (dp, dr) = row_at, to
    h = torch.arange(pages.shape[2], device=DEV)[:, None].expand_as(sp)
    got = pages[:, sp, h, sr]
    pages[:, dp[live], h[live], dr[live]] = got[:, live]


def _evict_plain(s):
    c = s["case"]
    S, H, B = c["seqs"], c["kv_heads"], c["budget"]
    slots, ctx, w = s["slots"].long(), s["ctx"].long(), s["weights"]
    P = w.shape[2]
    x = w[slots]
    j = torch.arange(P, device=DEV)
    there = (j < ctx[:, None])[:, None]
    always = ((j < c["first"]) | (j >= (ctx - c["recent"])[:, None]))[:, None] & there
    key = torch.where(always, math.inf, torch.where(there, x, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1][..., :B]
    counts = ctx.clamp(max=B)
    live = (torch.arange(B, device=DEV) < counts[:, None])[:, None].expand(S, H, B)
    kept = torch.sort(torch.where(live, order[..., :B] if P >= B else torch.nn.functional.pad(order, (0, B - P)), P), dim=-1)[0]
    kept = torch.where(live, kept, -1)
    ps = s["k_cache"].shape[2]
    table = s["table"].long()[slots]
    i = torch.arange(B, device=DEV).expand(S, H, B)

    def place(pos):
        pos = pos.clamp(min=0, max=P - 1)
        return table.gather(1, (pos // ps).flatten(1)).view(S, H, B), pos % ps

    _gone_to_front(s["pages"], place(kept), place(i), live)
    moved = x.gather(2, kept.clamp(min=0))
    new = torch.where((j < ctx[:, None])[:, None], 0.0, x)
    new[..., :B] = torch.where(live, moved, new[..., :B])[..., :P]
    w[slots] = new
    return [kept.to(I32), counts.to(I32), s["pages"], w]


def _accept_plain(s):
    c = s["case"]
    S, R = c["seqs"], s["max_rows"]
    first, tokens, parents = s["first"].long(), s["tokens"].long(), s["parents"].long()
    x = s["logits"].to(F32)
    v = torch.arange(c["vocab"], device=DEV)
    chosen = torch.where(x == x.amax(1, keepdim=True), v, c["vocab"]).amin(1)          # of equal ones the lowest
    reach, seq, i = _ancestors(s)
    t = torch.arange(tokens.shape[0], device=DEV)
    up = torch.where(parents >= 0, first[seq] + parents, t)
    fits = (parents >= 0) & (tokens == chosen[up])
    twin = (seq[:, None] == seq) & (parents[:, None] == parents) & (t < t[:, None]) & fits       # a sibling before that fits as well
    fits = (fits & ~twin.any(1)) | (i == 0)
    ok = torch.zeros(S, R, dtype=torch.bool, device=DEV)
    ok[seq, i] = fits
    taken = (ok[:, None] | ~reach).all(2)                                              # all of its ancestors, itself among them
    alive = torch.arange(R, device=DEV) < (first[1:] - first[:-1])[:, None]
    taken &= alive
    counts = taken.sum(1)
    r = torch.arange(R, device=DEV)
    rows = torch.sort(torch.where(taken, r, R), dim=1)[0]
    last = rows.gather(1, (counts - 1)[:, None])[:, 0]
    nxt = chosen[first[:-1] + last]
    rows = torch.where(rows < R, rows, -1)
    ps, H = s["pages"].shape[3], s["pages"].shape[2]
    table, base = s["table"].long()[s["slots"].long()], s["committed"].long()[:, None]

    def place(pos):
        pos = pos.clamp(min=0, max=table.shape[1] * ps - 1)
        return [y[:, None].expand(S, H, R) for y in (table.gather(1, pos // ps), pos % ps)]

    _gone_to_front(s["pages"], place(base + rows.clamp(min=0)), place(base + r), (rows >= 0)[:, None].expand(S, H, R))
    return [rows.to(I32), counts.to(I32), nxt.to(I32), s["pages"]]


# ---------------------------------------------------------------------------------------------------- the framework's calls
def _arr(t):
    from pygpukit_b200.core import dtypes
    from pygpukit_b200.core.array import GPUArray
    return None if t is None else GPUArray(tuple(t.shape), getattr(dtypes, str(t.dtype).replace("torch.", "")), ptr=t.data_ptr(), source=t)


def _held(s, *names):
    """the package's arrays over the state's tensors: a program holds them, so that they are made with a state's first pass"""
    held = s.setdefault("held", {})
    for n in names:
        if n not in held:
            held[n] = [_arr(t) for t in s[n]] if n in ("kept", "accepted", "pages") else _arr(s[n])
    return [held[n] for n in names]


def _tree_own(s):
    from pygpukit_b200 import ops
    q, k_cache, v_cache, out, table, slots, ctx, first, parents, masks, depths = _held(
        s, "q", "k_cache", "v_cache", "out", "table", "slots", "ctx", "first", "parents", "masks", "depths")
    if s["case"]["masks"]:
        ops.tree_masks(parents, first, s["max_rows"], masks=masks, depths=depths)
    ops.sdpa_paged(q, k_cache, v_cache, out, table, slots, ctx, s["max_ctx"], row_starts=first, max_rows=s["max_rows"], masks=masks)
    return [s["out"], s["masks"], s["depths"]] if s["case"]["masks"] else s["out"]


def _weigh_own(s):
    from pygpukit_b200 import ops
    q, k_cache, v_cache, out, table, slots, ctx, first, lse, weights = _held(
        s, "q", "k_cache", "v_cache", "out", "table", "slots", "ctx", "first", "lse", "weights")
    starts = first if s["case"]["rows"] > 1 else None
    ops.sdpa_paged(q, k_cache, v_cache, out, table, slots, ctx, s["max_ctx"], row_starts=starts, max_rows=s["max_rows"], lse=lse)
    ops.weigh_paged(q, k_cache, lse, weights, table, slots, ctx, s["max_ctx"], row_starts=starts, max_rows=s["max_rows"])
    return [s["out"], s["lse"], s["weights"]]


def _evict_own(s):
    from pygpukit_b200 import ops
    c = s["case"]
    pages, table, slots, ctx, weights, kept = _held(s, "pages", "table", "slots", "ctx", "weights", "kept")
    ops.select_rows(weights, slots, ctx, c["budget"], first=c["first"], recent=c["recent"], out=tuple(kept))
    ops.move_rows_paged(pages, table, slots, kept[0], kept[1], weights=weights, context_lens=ctx)
    return [*s["kept"], s["pages"], s["weights"]]


def _accept_own(s):
    from pygpukit_b200 import ops
    pages, table, slots, logits, tokens, parents, first, committed, accepted = _held(
        s, "pages", "table", "slots", "logits", "tokens", "parents", "first", "committed", "accepted")
    ops.accept_tree(logits, tokens, parents, first, s["max_rows"], out=tuple(accepted))
    ops.move_rows_paged(pages, table, slots, accepted[0], accepted[1], starts=committed)
    return [*s["accepted"], s["pages"]]


_PLAIN = dict(tree=_tree_plain, weigh=_weigh_plain, evict=_evict_plain, accept=_accept_plain)
_OWN = dict(tree=_tree_own, weigh=_weigh_own, evict=_evict_own, accept=_accept_own)


def run(state: dict):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------- the work
def work(case: dict) -> dict:
    c, kind = case, case["kind"]
    size, D, H = TYPES[c["dtype"]].itemsize, c["dim"], c["kv_heads"]
    rows, ctx = _rows(c), _contexts(c)
    if kind in ("tree", "weigh"):
        Hq, T = c["heads"], sum(rows)
        seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(rows, ctx))
        b, f = 2 * T * Hq * D * size + 2 * sum(ctx) * H * D * size, 4 * seen * Hq * D
        if kind == "tree":
            return dict(bytes=b + T * 4 * -(-max(rows) // 32) + (8 * T if c["masks"] else 0), flops=f)
        return dict(bytes=b + 4 * T * Hq + 8 * sum(ctx) * H, flops=f)
    if kind == "evict":
        kept = sum(min(m, c["budget"]) for m in ctx)
        # a position that stays where it is costs nothing: of the first ones, none before the first that goes
        return dict(bytes=4 * sum(ctx) * H + 4 * kept * H + 4 * kept * D * H * size + 4 * sum(ctx) * H + 4 * kept * H, flops=0)
    T = sum(rows)
    return dict(bytes=T * c["vocab"] * 2 + 8 * T + c["seqs"] * (4 * max(rows) + 8), flops=T * c["vocab"])


# ---------------------------------------------------------------------------------------------------- 64 bits
def _exact_attend(s, masks):
    """outputs, logarithms of the softmax's sums, weights by position, from loops over sequences and heads"""
    c = s["case"]
    D, H, rep, ps = c["dim"], c["kv_heads"], c["heads"] // c["kv_heads"], s["k_cache"].shape[2]
    first, ctx, slots, table = s["first"].tolist(), s["ctx"].tolist(), s["slots"].tolist(), s["table"].cpu().tolist()
    out = torch.empty(s["q"].shape, dtype=F64, device=DEV)
    lse = torch.empty(s["q"].shape[:2], dtype=F64, device=DEV)
    weights = s["weights"].to(F64) if "weights" in s else None
    for i, (m, slot) in enumerate(zip(ctx, slots)):
        at = torch.tensor(table[slot][:-(-m // ps)], device=DEV)
        k, v = (x[at].to(F64).permute(1, 0, 2, 3).reshape(H, -1, D)[:, :m] for x in (s["k_cache"], s["v_cache"]))
        q = s["q"][first[i]:first[i + 1]].to(F64)
        n = q.shape[0]
        hidden = torch.zeros(n, m, dtype=torch.bool, device=DEV)
        hidden[:, m - n:] = ~masks[i] if masks is not None else torch.ones(n, n, device=DEV).triu(1).bool()
        for h in range(c["heads"]):
            x = torch.einsum("td,jd->tj", q[:, h], k[h // rep]) / math.sqrt(D)
            x[hidden] = -math.inf
            z = torch.logsumexp(x, 1)
            p = torch.exp(x - z[:, None])
            out[first[i]:first[i + 1], h] = p @ v[h // rep]
            lse[first[i]:first[i + 1], h] = z
            if weights is not None:
                weights[slot, h // rep, :m] += p.sum(0)
    return out, lse, weights


def exact(case: dict, seed: int):
    c, kind = case, case["kind"]
    if kind == "evict":
        return None                                     # whole numbers and rows as they were
    s = prepare(case, seed)
    if kind == "tree":
        masks = []
        for parents in _trees(c, seed):
            m = torch.zeros(len(parents), len(parents), dtype=torch.bool)
            for i, p in enumerate(parents):
                if p >= 0:
                    m[i] = m[p]
                m[i, i] = True
            masks.append(m.to(DEV))
        out = _exact_attend(s, masks)[0]
        return [out, None, None] if c["masks"] else out
    if kind == "weigh":
        return list(_exact_attend(s, None))
    return None
