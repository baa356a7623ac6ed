"""The operators of decoding on a paged cache held in four bits, and of beam search, as they are measured: keys and values appended (the
rotation on the way) and read back, attention of decoded tokens, of a few rows and of prompts over that cache, the selection of beams, and
the reordering of what belongs to a beam.

The cache stands for values s (c - z): codes c of four bits, and per group of 32 elements of a head's row one 16-bit word, a bfloat16 scale s
of four significant bits (bits 4 to 14) above a zero point z (bits 0 to 3).  A page of one head holds page_size rows of D / 2 bytes of codes,
then page_size rows of D / 32 words; the 32-bit word t (D / 32) + g of a row holds elements 32 g + 8 t ... + 7, the first in the lowest bits.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------------- the cases
def listed() -> list[dict]:
    return [
        # eight requests of an 8B decoder bring one token each: the smallest call, latency counts
        dict(name="append_decode_8", kind="append", seqs=8, rows=1, ctx=4100, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16",
             rot=128, pairs=False),
        # three prompts side by side, of unequal odd lengths
        dict(name="append_prompts_3200", kind="append", seqs=3, rows=1333, ctx=1333, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16",
             rot=128, pairs=False),
        # one request of an 8B decoder, one token over a few thousand positions
        dict(name="decode_1x4096", kind="attend", seqs=1, rows=1, ctx=4096, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16",
             window=0, softcap=0.0, sinks=False),
        # a full batch of a 70B decoder over long contexts: the bytes of the cache
        dict(name="decode_64x8192", kind="attend", seqs=64, rows=1, ctx=8192, heads=64, kv_heads=8, dim=128, page=64, dtype="bfloat16",
             window=0, softcap=0.0, sinks=False),
        # a token-major model's float32 rows behind a window, with learned sinks and a tanh cap
        dict(name="decode_8x2000_f32", kind="attend", seqs=8, rows=1, ctx=2000, heads=16, kv_heads=4, dim=128, page=64, dtype="float32",
             window=1024, softcap=50.0, sinks=True),
        # drafts of five tokens verified for eight requests
        dict(name="verify_8x5", kind="attend", seqs=8, rows=5, ctx=3001, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16",
             window=0, softcap=0.0, sinks=False),
        # a whole prompt
        dict(name="prompt_2000", kind="attend", seqs=1, rows=2000, ctx=2000, heads=32, kv_heads=8, dim=128, page=64, dtype="bfloat16",
             window=0, softcap=0.0, sinks=False),
        # a portion of a long prompt
        dict(name="portion_512_16k", kind="attend", seqs=1, rows=512, ctx=16384, heads=32, kv_heads=4, dim=128, page=64, dtype="bfloat16",
             window=0, softcap=0.0, sinks=False),
        # one request with four beams, the token-major models' float32 logits
        dict(name="beam_1x4", kind="beam", groups=1, beams=4, n=8, vocab=32768, dtype="float32", finished=0),
        # sixteen requests with eight beams over a large vocabulary
        dict(name="beam_16x8", kind="beam", groups=16, beams=8, n=16, vocab=151936, dtype="float32", finished=3),
        # the recurrent states of sixteen layers follow four requests' eight beams (a 128 x 128 state for each of 16 heads)
        dict(name="reorder_32x16", kind="reorder", groups=4, beams=8, arrays=16, floats=262144),
        # the partly filled pages of 32 layers that two beams go on from
        dict(name="pages_24x64", kind="pages", pairs=24, arrays=64, pages=256, bytes=36864),
    ]


def _log(rng, lo: int, hi: int, step: int = 1) -> int:
    """a multiple of `step` in lo .. hi, spread over its logarithm"""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


HEADS = [(32, 8), (64, 8), (32, 4), (16, 4), (16, 16), (12, 3), (8, 1), (4, 2)]


def draw(rng) -> dict:
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "few", "prompt", "prompt", "beam", "beam", "reorder", "pages"])
    dim = rng.choice([128, 128, 128, 64, 96, 256])
    page = rng.choice([64, 64, 16, 32, 128, 48])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    heads, kv = rng.choice(HEADS)
    extra = dict(window=rng.choice([0, 0, 0, 128, 1000]), softcap=rng.choice([0.0, 0.0, 30.0]), sinks=rng.random() < 0.3)
    if kind == "append":
        seqs = _log(rng, 1, 64)
        rows = rng.choice([1, 1, _log(rng, 2, 4000 // seqs)])
        return dict(kind="append", seqs=seqs, rows=rows, ctx=rows + _log(rng, 1, 3000) - 1, heads=heads, kv_heads=kv, dim=dim, page=page,
                    dtype=dtype, rot=rng.choice([dim, dim, dim // 2]), pairs=rng.random() < 0.3)
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        return dict(kind="attend", seqs=seqs, rows=1, ctx=_log(rng, 1, min(32768, 400_000_000 // (seqs * kv * dim))), heads=heads, kv_heads=kv,
                    dim=dim, page=page, dtype=dtype, **extra)
    if kind == "few":
        seqs, rows = _log(rng, 1, 16), _log(rng, 2, 16)
        return dict(kind="attend", seqs=seqs, rows=rows, ctx=_log(rng, rows, 4000), heads=heads, kv_heads=kv, dim=dim, page=page, dtype=dtype,
                    **extra)
    if kind == "prompt":
        seqs, rows = rng.choice([1, 1, 2, 3]), _log(rng, 17, 1000)
        if dtype == "float32":
            rows = min(rows, 300)
        ctx = rows + rng.choice([0, 0, _log(rng, 1, 4000)])
        rows = max(17, min(rows, 30_000_000_000 // (seqs * heads * dim * ctx)))
        return dict(kind="attend", seqs=seqs, rows=rows, ctx=max(rows, ctx), heads=heads, kv_heads=kv, dim=dim, page=page, dtype=dtype, **extra)
    if kind == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        return dict(kind="beam", groups=_log(rng, 1, 128 // beams), beams=beams, n=rng.choice([beams, 2 * beams, 2 * beams]),
                    vocab=_log(rng, 1000, 151936), dtype=dtype, finished=rng.choice([0, 0, 1]))
    if kind == "reorder":
        beams = rng.choice([2, 3, 4, 8])
        return dict(kind="reorder", groups=_log(rng, 1, 16), beams=beams, arrays=rng.choice([1, 5, 16]), floats=_log(rng, 100, 100000, 2))
    return dict(kind="pages", pairs=_log(rng, 1, 60), arrays=rng.choice([2, 8, 48]), pages=200, bytes=_log(rng, 288, 36864, 144))


# ---------------------------------------------------------------------------------------------------- inputs
class _Gen:
    """tensors of one case, in the order in which they are asked for"""

    def __init__(self, seed: int):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 7919 + 17)

    def normal(self, *shape, std=1.0, dtype=F32):
        return (torch.randn(*shape, generator=self.g, device=DEV) * std).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=DEV)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _contexts(c) -> list[int]:
    """positions of every sequence behind the step: the last one has the most"""
    span = max(0, c["ctx"] - c["rows"])
    return [c["ctx"] - (37 * i * i) % (span // 4 + 1) for i in range(c["seqs"] - 1, -1, -1)]


def _rows(c) -> list[int]:
    """rows of every sequence: with several prompts side by side of unequal length"""
    return [max(1, c["rows"] - (c["rows"] // 5) * (i % 3)) for i in range(c["seqs"])]


def _parents(c) -> list[list[int]]:
    """what a step of beam search leaves: a few beams go on from the best ones, the others from themselves"""
    r = random.Random(c["beams"] * 1009 + c["groups"])
    return [[k if r.random() < 0.5 else r.randrange(c["beams"]) for k in range(c["beams"])] for _ in range(c["groups"])]


def _pairs(c) -> tuple[list[int], list[int]]:
    r = random.Random(c["pairs"])
    rows = r.sample(range(c["pages"]), 2 * c["pairs"])
    return rows[:c["pairs"]], rows[c["pairs"]:]


def _cache(g: _Gen, c) -> tuple:
    """(K pages, V pages, page table, slots): a cache filled by earlier steps, its pages in any order"""
    ctx, ps, D, H = _contexts(c), c["page"], c["dim"], c["kv_heads"]
    per = -(-max(ctx) // ps)
    used = c["seqs"] * per
    table = g.perm(used).view(c["seqs"], per).to(torch.int32)
    slots = g.perm(c["seqs"]).to(torch.int32)
    chan = 0.3 + 2.0 * g.uniform(2, 1, H, 1, D) ** 3            # channels of unequal size, as keys have them
    mean = g.normal(2, 1, H, 1, D, std=0.4)
    out = []
    for side in range(2):
        pages = torch.empty(used, H, ps, D * 9 // 16, dtype=torch.uint8, device=DEV)
        step = max(1, 32_000_000 // (H * ps * D))
        for p in range(0, used, step):
            n = min(step, used - p)
            x = (g.normal(n, H, ps, D) * chan[side] + mean[side]).to(torch.bfloat16).to(F32)
            code, word = _encode(x)
            flat = pages[p:p + n].view(n, H, -1)
            flat[:, :, :ps * D // 2] = code.reshape(n, H, -1)
            flat[:, :, ps * D // 2:] = word.reshape(n, H, -1)
        out.append(pages)
    return (*out, table, slots)


def prepare(case: dict, seed: int) -> dict:
    c = {k: v for k, v in case.items() if k != "name"}
    g, kind = _Gen(seed), c["kind"]
    s = dict(case=c)
    if kind in ("append", "attend"):
        dt, D = TYPES[c["dtype"]], c["dim"]
        rows, ctx = _rows(c), _contexts(c)
        T = sum(rows)
        s["k_cache"], s["v_cache"], s["table"], s["slots"] = _cache(g, c)
        slots = s["slots"].tolist()
        s["q"] = g.normal(T, c["heads"], D, dtype=dt)
        if kind == "append":
            s["k"], s["v"] = g.normal(T, c["kv_heads"], D, std=1.5, dtype=dt), g.normal(T, c["kv_heads"], D, dtype=dt)
            pos = [p for n, m in zip(rows, ctx) for p in range(m - n, m)]
            s["row_slots"] = torch.tensor([x for n, x in zip(rows, slots) for _ in range(n)], dtype=torch.int32, device=DEV)
            s["positions"] = torch.tensor(pos, dtype=torch.int32, device=DEV)
            inv = 5e5 ** (-torch.arange(0, c["rot"], 2, dtype=F64, device=DEV) / c["rot"])
            a = torch.arange(c["ctx"], dtype=F64, device=DEV)[:, None] * inv
            s["cos"], s["sin"] = (torch.cat([f(a), f(a)], 1).to(F32).contiguous() for f in (torch.cos, torch.sin))
            s["k_rows"], s["v_rows"] = (torch.empty(T, c["kv_heads"], D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        else:
            s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
            first = [0]
            for n in rows:
                first.append(first[-1] + n)
            s["first"] = torch.tensor(first, dtype=torch.int32, device=DEV)
            s["max_rows"], s["max_ctx"] = max(rows), max(ctx)
            s["sinks"] = g.normal(c["heads"]) if c["sinks"] else None
            s["out"] = torch.empty_like(s["q"])
    elif kind == "beam":
        B, K, V = c["groups"], c["beams"], c["vocab"]
        x = g.normal(B * K, V, std=2.0)
        top = (g.uniform(B * K, 12) * V).long()
        x.scatter_add_(1, top, 4.0 + 6.0 * g.uniform(B * K, 12))
        s["logits"] = x.to(TYPES[c["dtype"]])
        s["scores"] = -torch.cumsum(2.0 * g.uniform(B, K), 1)
        s["finished"] = (g.uniform(B, K) < 0.15 * c["finished"]).to(torch.int32) if c["finished"] else None
        s["picked"] = (torch.empty(B, c["n"], dtype=F32, device=DEV), torch.empty(B, c["n"], dtype=torch.int32, device=DEV),
                       torch.empty(B, c["n"], dtype=torch.int32, device=DEV))
    elif kind == "reorder":
        s["rows"] = g.normal(c["arrays"], c["groups"] * c["beams"], c["floats"])
        s["parents"] = torch.tensor(_parents(c), dtype=torch.int32, device=DEV)
    else:
        s["rows"] = torch.randint(0, 256, (c["arrays"], c["pages"], c["bytes"]), generator=g.g, device=DEV, dtype=torch.uint8)
        s["src"], s["dst"] = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in _pairs(c))
    return s


# ---------------------------------------------------------------------------------------------------- the plain forms
def _encode(x):
    """float32 rows [..., D] -> (codes [..., D / 2], group words [..., D / 16]) as bytes"""
    D = x.shape[-1]
    y = x.unflatten(-1, (D // 32, 32))
    lo, hi = y.amin(-1).clamp(max=0.0), y.amax(-1).clamp(min=0.0)
    bits = ((hi - lo) / torch.full_like(hi, 15.0)).view(torch.int32)      # a quotient, rounded once: often four bits already
    bits = (bits + 0xFFFFF) & ~0xFFFFF                         # up to four significant bits
    scale = bits.view(F32)
    scale = torch.where(scale < 2.0 ** -40, torch.zeros_like(scale), scale)
    div = torch.where(scale == 0, torch.ones_like(scale), scale)
    zero = torch.where(scale == 0, torch.zeros_like(scale), torch.round(-lo / div))
    code = (torch.round(y / div[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8)
    code = torch.where(scale[..., None] == 0, torch.zeros_like(code), code)
    n = code.unflatten(-1, (4, 4, 2)).transpose(-3, -4)        # [..., t, g, byte, nibble]
    word = ((scale.view(torch.int32) >> 16) | zero.to(torch.int32)).to(torch.int16)
    return (n[..., 0] | (n[..., 1] << 4)).flatten(-3), word.view(torch.uint8)


def _values(pages, D):
    """pages [..., page, 9 D / 16] of bytes -> the float32 values [..., page, D] that they stand for"""
    ps = pages.shape[-2]
    flat = pages.flatten(-2)
    code = flat[..., :ps * D // 2].unflatten(-1, (ps, 4, D // 32, 4))
    word = flat[..., ps * D // 2:].contiguous().view(torch.int16).unflatten(-1, (ps, D // 32)).to(torch.int32)
    nib = torch.stack([code & 15, code >> 4], -1).transpose(-3, -4).flatten(-3)        # [..., page, g, 32]
    scale = ((word & 0x7FF0) << 16).view(F32)
    return ((nib.to(F32) - (word & 15).to(F32)[..., None]) * scale[..., None]).flatten(-2)


def _turn(x, cos, sin, pairs):
    """rows [T, H, D] rotated over the first elements, in float32"""
    R = cos.shape[-1]
    h = R // 2
    y = x.to(F32)
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if pairs else (y[..., :h], y[..., h:R])
    c, s = cos[:, None, :h], sin[:, None, :h]
    u, v = a * c - b * s, b * c + a * s
    return torch.cat([torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1), y[..., R:]], -1)


def _append_plain(s):
    c, ps = s["case"], s["case"]["page"]
    D, pos = c["dim"], s["positions"].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    page = s["table"].long()[s["row_slots"].long(), pos // ps]
    row = pos % ps
    s["q"].copy_(_turn(s["q"], cos, sin, c["pairs"]).to(s["q"].dtype))
    return [s["q"], *(_store(cache, page, row, x, D) for cache, x in
                      ((s["k_cache"], _turn(s["k"], cos, sin, c["pairs"])), (s["v_cache"], s["v"].to(F32))))]


def _store(cache, page, row, x, D):
    """rows into their pages, and what they stand for there"""
    ps = cache.shape[-2]
    code, word = _encode(x)
    flat = cache.flatten(-2)
    codes, words = flat[..., :ps * D // 2].unflatten(-1, (ps, D // 2)), flat[..., ps * D // 2:].unflatten(-1, (ps, D // 16))
    codes[page, :, row] = code
    words[page, :, row] = word
    back = torch.cat([codes[page, :, row], words[page, :, row]], -1)[..., None, :]
    return _values(back, D)[..., 0, :].to(torch.bfloat16)


def _attend_plain(s):
    c = s["case"]
    D, H, rep = c["dim"], c["kv_heads"], c["heads"] // c["kv_heads"]
    S, R, first, ctx = c["seqs"], s["max_rows"], s["first"].long(), s["ctx"].long()
    pages = s["table"].long()[s["slots"].long()]
    k, v = (_values(x[pages], D).transpose(1, 2).flatten(2, 3) for x in (s["k_cache"], s["v_cache"]))      # [S, H, keys, D]
    n = first[1:] - first[:-1]
    i = torch.arange(R, device=DEV)
    live = i < n[:, None]
    at = (first[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].to(F32).unflatten(2, (H, rep)).permute(0, 2, 3, 1, 4).flatten(2, 3)                     # [S, H, rep R, D]
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    if c["softcap"] > 0:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    pos = (ctx - n)[:, None] + i                                                                          # [S, R]
    j = torch.arange(k.shape[2], device=DEV)
    seen = j <= pos[..., None]
    if c["window"] > 0:
        seen = seen & (j > pos[..., None] - c["window"])
    x = x.unflatten(2, (rep, R)).masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, H, rep, 1, 1)
        top = torch.maximum(top, sink)
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    o = (w.flatten(2, 3) @ v).unflatten(2, (rep, R)) / total
    return o.permute(0, 3, 1, 2, 4)[live].flatten(1, 2).to(s["q"].dtype)


def _beam_plain(s):
    c = s["case"]
    B, K, V = c["groups"], c["beams"], c["vocab"]
    x = s["logits"].to(F64).view(B, K, V)
    x = x - x.amax(-1, keepdim=True)
    x = s["scores"].to(F64)[..., None] + (x - torch.log(torch.exp(x).sum(-1, keepdim=True)))
    if s["finished"] is not None:
        done = s["finished"].bool()[..., None]
        pad = torch.arange(V, device=DEV) == 0
        x = torch.where(done, torch.where(pad, s["scores"].to(F64)[..., None], -math.inf), x)
    best, at = torch.sort(x.flatten(1), dim=1, descending=True, stable=True)
    best, at = best[:, :c["n"]], at[:, :c["n"]]
    return [best.to(F32), (at // V).to(torch.int32), (at % V).to(torch.int32)]


def _reorder_plain(s):
    c, x = s["case"], s["rows"]
    at = (s["parents"].long() + torch.arange(c["groups"], device=DEV)[:, None] * c["beams"]).flatten()
    x.copy_(x[:, at])
    return x


def _pages_plain(s):
    s["rows"][:, s["dst"].long()] = s["rows"][:, s["src"].long()]
    return s["rows"]


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
            held[n] = [_arr(t) for t in s[n]] if n in ("rows", "picked") else _arr(s[n])
    return [held[n] for n in names]


def _append_own(s):
    from pygpukit_b200 import ops
    k_cache, v_cache, table, slots, pos = _held(s, "k_cache", "v_cache", "table", "row_slots", "positions")
    q, k, v, cos, sin, k_rows, v_rows = _held(s, "q", "k", "v", "cos", "sin", "k_rows", "v_rows")
    ops.rope_append_paged_int4(q, k, v, cos, sin, k_cache, v_cache, table, slots, pos, interleaved=s["case"]["pairs"])
    ops.kv_read_paged_int4(k_cache, table, slots, pos, out=k_rows)
    ops.kv_read_paged_int4(v_cache, table, slots, pos, out=v_rows)
    return [s["q"], s["k_rows"], s["v_rows"]]


def _attend_own(s):
    from pygpukit_b200 import ops
    c = s["case"]
    q, k_cache, v_cache, out, table, slots, ctx, first, sinks = _held(s, "q", "k_cache", "v_cache", "out", "table", "slots", "ctx", "first", "sinks")
    ops.sdpa_paged_int4(q, k_cache, v_cache, out, table, slots, ctx, s["max_ctx"], row_starts=first if c["rows"] > 1 else None,
                        max_rows=s["max_rows"], window=c["window"], softcap=c["softcap"], sinks=sinks)
    return s["out"]


def _beam_own(s):
    from pygpukit_b200 import ops
    logits, scores, finished, picked = _held(s, "logits", "scores", "finished", "picked")
    ops.beam_select(logits, scores, s["case"]["n"], finished=finished, pad_token=0, out=tuple(picked))
    return list(s["picked"])


def _reorder_own(s):
    from pygpukit_b200 import ops
    rows, parents = _held(s, "rows", "parents")
    ops.reorder_rows(rows, parents)
    return s["rows"]


def _pages_own(s):
    from pygpukit_b200 import ops
    rows, src, dst = _held(s, "rows", "src", "dst")
    ops.copy_rows(rows, src, dst)
    return s["rows"]


_PLAIN = dict(append=_append_plain, attend=_attend_plain, beam=_beam_plain, reorder=_reorder_plain, pages=_pages_plain)
_OWN = dict(append=_append_own, attend=_attend_own, beam=_beam_own, reorder=_reorder_own, pages=_pages_own)


def run(state: dict):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------- the work
def work(case: dict) -> dict:
    c, kind = case, case["kind"]
    if kind in ("append", "attend"):
        size = TYPES[c["dtype"]].itemsize
        D, H, Hq = c["dim"], c["kv_heads"], c["heads"]
        rows, ctx = _rows(c), _contexts(c)
        T = sum(rows)
        if kind == "append":
            # q read and written, k and v read, the rows in four bits written, and read again for 16-bit rows
            return dict(bytes=T * (2 * Hq * D * size + 2 * H * D * size + 2 * 2 * H * D * 9 // 16 + 2 * H * D * 2 + 4 * c["rot"] + 8),
                        flops=T * (6 * (Hq + H) * c["rot"] // 2 + 8 * 2 * H * D))
        keys = seen = 0
        for n, m in zip(rows, ctx):
            w = c["window"] if c["window"] > 0 else m
            keys += min(m, n - 1 + w)
            seen += sum(min(p + 1, w) for p in range(m - n, m))
        return dict(bytes=2 * T * Hq * D * size + 2 * keys * H * D * 9 // 16, flops=4 * seen * Hq * D)
    if kind == "beam":
        rows = c["groups"] * c["beams"] * (1.0 - 0.15 * c["finished"])
        return dict(bytes=rows * c["vocab"] * TYPES[c["dtype"]].itemsize + c["groups"] * c["n"] * 12, flops=4 * rows * c["vocab"])
    if kind == "reorder":
        reads = sum(len({p for k, p in enumerate(ps) if p != k}) for ps in _parents(c))
        writes = sum(p != k for ps in _parents(c) for k, p in enumerate(ps))
        return dict(bytes=max(1, reads + writes) * c["arrays"] * c["floats"] * 4, flops=0)
    return dict(bytes=2 * c["pairs"] * c["arrays"] * c["bytes"], flops=0)


# ---------------------------------------------------------------------------------------------------- 64 bits
def _exact_attend(s):
    c = s["case"]
    D, H, rep = c["dim"], c["kv_heads"], c["heads"] // c["kv_heads"]
    first, ctx, slots = s["first"].tolist(), s["ctx"].tolist(), s["slots"].tolist()
    out = torch.empty(s["q"].shape, dtype=F64, device=DEV)
    ps = c["page"]
    table = s["table"].cpu().tolist()
    for i, (m, slot) in enumerate(zip(ctx, slots)):
        pages = torch.tensor(table[slot][:-(-m // ps)], device=DEV)
        kv = []
        for cache in (s["k_cache"], s["v_cache"]):
            x = cache[pages].reshape(len(pages), H, -1).to(torch.int64)
            w = x[..., :ps * D // 2].view(len(pages), H, ps, D // 8, 4)
            w = (w * torch.tensor([1, 256, 65536, 1 << 24], device=DEV)).sum(-1)
            meta = x[..., ps * D // 2:].view(len(pages), H, ps, D // 32, 2)
            meta = meta[..., 0] + 256 * meta[..., 1]
            e = torch.arange(D, device=DEV)
            code = torch.bitwise_right_shift(w[..., (e % 32) // 8 * (D // 32) + e // 32], 4 * (e % 8)) & 15
            scale = torch.where(meta == 0, torch.zeros((), dtype=F64, device=DEV),
                                torch.ldexp(1.0 + ((meta >> 4) & 7).to(F64) / 8.0, (meta >> 7) - 127))
            val = (code - (meta & 15)[..., e // 32]).to(F64) * scale[..., e // 32]
            kv.append(val.permute(1, 0, 2, 3).reshape(H, -1, D)[:, :m])
            del x, w, code, val
        q = s["q"][first[i]:first[i + 1]].to(F64)
        n = q.shape[0]
        p = torch.arange(m - n, m, device=DEV)[:, None]
        j = torch.arange(m, device=DEV)[None]
        hidden = (j > p) | ((j <= p - c["window"]) if c["window"] > 0 else (j < 0))
        for h in range(c["heads"]):
            x = torch.einsum("td,jd->tj", q[:, h], kv[0][h // rep]) / math.sqrt(D)
            if c["softcap"] > 0:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            x[hidden] = -math.inf
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].to(F64).expand(n, 1)], 1)
            w = torch.softmax(x, 1)[:, :m]
            out[first[i]:first[i + 1], h] = w @ kv[1][h // rep]
    return out


def _exact_append(s):
    c = s["case"]
    pos = s["positions"].long()
    R, D = c["rot"], c["dim"]

    def turned(x):
        y = x.to(F64).clone()
        first = torch.arange(0, R, 2, device=DEV) if c["pairs"] else torch.arange(R // 2, device=DEV)
        second = first + (1 if c["pairs"] else R // 2)
        z = torch.complex(y[..., first], y[..., second])
        z = z * torch.complex(s["cos"][pos, :R // 2].to(F64), s["sin"][pos, :R // 2].to(F64))[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def held(x):
        """what a row stands for in four bits"""
        y = x.reshape(*x.shape[:-1], D // 32, 32)
        lo, hi = torch.minimum(y.min(-1)[0], torch.zeros((), device=DEV)), torch.maximum(y.max(-1)[0], torch.zeros((), device=DEV))
        m, e = torch.frexp((hi - lo) / 15.0)                    # 0.5 <= m < 1: sixteenths are four significant bits
        scale = torch.ldexp(torch.ceil(m * 16.0) / 16.0, e)
        scale[scale < 2.0 ** -40] = 0.0
        safe = torch.where(scale == 0, torch.ones_like(scale), scale)
        z = torch.round(-lo / safe)
        code = torch.clamp(torch.round(y / safe[..., None]) + z[..., None], 0.0, 15.0)
        return ((code - z[..., None]) * scale[..., None]).reshape(x.shape)

    # the keys are rotated and divided in float32 before they are rounded to four bits: an element next to a border may fall on either side
    return [turned(s["q"]), held(turned(s["k"])), held(s["v"].to(F64))]


def _exact_beam(s):
    c = s["case"]
    B, K, V = c["groups"], c["beams"], c["vocab"]
    x = s["logits"].cpu().to(F64).numpy().reshape(B, K, V)
    base = s["scores"].cpu().to(F64).numpy()
    done = s["finished"].cpu().numpy() if s["finished"] is not None else np.zeros((B, K), int)
    out = [np.zeros((B, c["n"])), np.zeros((B, c["n"]), np.int32), np.zeros((B, c["n"]), np.int32)]
    for b in range(B):
        found = []
        for k in range(K):
            if done[b, k]:
                found.append((-base[b, k], k, 0))
                found += [(math.inf, k, t) for t in range(1, min(V, c["n"] + 1))]
                continue
            r = x[b, k]
            peak = r.max()
            total = peak + math.log(math.fsum(np.exp(r - peak)))
            cut = np.partition(r, V - c["n"])[V - c["n"]] if V > c["n"] else -math.inf
            found += [(-(base[b, k] + (float(r[t]) - total)), k, int(t)) for t in np.flatnonzero(r >= cut)]
        found.sort()
        for i, (v, k, t) in enumerate(found[:c["n"]]):
            out[0][b, i], out[1][b, i], out[2][b, i] = -v, k, t
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":
        return _exact_append(s)
    if kind == "attend":
        return _exact_attend(s)
    if kind == "beam":
        return _exact_beam(s)
    if kind == "reorder":
        rows, K = s["rows"].to(F64), case["beams"]
        at = [gi * K + p for gi, ps in enumerate(_parents(case)) for p in ps]
        return torch.stack([rows[:, p] for p in at], 1)
    return None
