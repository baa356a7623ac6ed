"""The four-bit cache, attention over it and beam search in NumPy: the format in float32 as it is defined, everything else in float64."""
import math

import numpy as np

from pygpukit_b200.core.dtypes import bf16_bits_to_f32, f32_to_bf16_bits

F = np.float32
NAN_WORD = 0x7FC0


def rounded(x, dtype):
    """float32 -> the type's storage"""
    x = np.asarray(x, F)
    return f32_to_bf16_bits(x) if dtype == "bfloat16" else x.astype(np.float16 if dtype == "float16" else F)


def floats(a, dtype):
    return bf16_bits_to_f32(a) if dtype == "bfloat16" else np.asarray(a, F)


def encode(x):
    """float32 rows [..., D] -> (words of codes uint32 [..., D / 8], group words uint16 [..., D / 32])"""
    D = x.shape[-1]
    y = np.asarray(x, F).reshape(*x.shape[:-1], D // 32, 32)
    with np.errstate(all="ignore"):
        bad = ~(np.abs(y) < F(2.0 ** 56)).all(-1)
        y = np.where(bad[..., None], F(0), y)
        lo, hi = np.minimum(y.min(-1), F(0)), np.maximum(y.max(-1), F(0))
        bits = ((hi - lo) / F(15)).view(np.uint32)
        s = ((bits + np.uint32(0xFFFFF)) & np.uint32(0xFFF00000)).view(F)
        none = ~(s >= F(2.0 ** -40))
        s = np.where(none, F(1), s)
        z = np.rint(-lo / s)
        c = np.clip(np.rint(y / s[..., None]) + z[..., None], 0, 15).astype(np.uint32)
    dead = (none | bad)
    c = np.where(dead[..., None], np.uint32(0), c)
    word = (s.view(np.uint32) >> 16).astype(np.uint16) | z.astype(np.uint16)
    word = np.where(none, np.uint16(0), word)
    word = np.where(bad, np.uint16(NAN_WORD), word)
    G = D // 32
    out = np.zeros((*x.shape[:-1], 4 * G), np.uint32)
    for g in range(G):
        for t in range(4):
            for e in range(8):
                out[..., t * G + g] |= c[..., g, 8 * t + e] << np.uint32(4 * e)
    return out, word


def decode(words, groups):
    """the inverse, in float64"""
    G = groups.shape[-1]
    out = np.zeros((*groups.shape, 32))
    scale = ((groups.astype(np.uint32) & 0x7FF0) << 16).astype(np.uint32).view(F).astype(np.float64)
    for g in range(G):
        for t in range(4):
            for e in range(8):
                c = (words[..., t * G + g] >> np.uint32(4 * e)) & np.uint32(15)
                out[..., g, 8 * t + e] = (c.astype(np.int64) - (groups[..., g] & 15).astype(np.int64)) * scale[..., g]
    return out.reshape(*groups.shape[:-1], 32 * G)


def put(cache, page, head, row, words, groups):
    """one row into a cache uint8 [pages, heads, page_size, row bytes]"""
    ps, n = cache.shape[2], words.size * 4
    flat = cache[page, head].reshape(-1)
    flat[row * n:(row + 1) * n] = words.view(np.uint8)
    at = ps * n + row * groups.size * 2
    flat[at:at + groups.size * 2] = groups.view(np.uint8)


def get(cache, page, head, row):
    ps = cache.shape[2]
    D = cache.shape[3] // 9 * 16
    flat = cache[page, head].reshape(-1)
    at = ps * (D // 2) + row * (D // 16)
    return flat[row * (D // 2):(row + 1) * (D // 2)].copy().view(np.uint32), flat[at:at + D // 16].copy().view(np.uint16)


def rows_of(cache, table, slot, n):
    """what the first n positions of a slot stand for: float64 [n, heads, D], and the scale of every element"""
    ps, H, D = cache.shape[2], cache.shape[1], cache.shape[3] // 9 * 16
    pages = np.asarray(table[slot][:-(-n // ps)])
    flat = cache[pages].reshape(len(pages), H, -1)
    words = np.ascontiguousarray(flat[..., :ps * D // 2]).view(np.uint32).reshape(len(pages), H, ps, D // 8)
    groups = np.ascontiguousarray(flat[..., ps * D // 2:]).view(np.uint16).reshape(len(pages), H, ps, D // 32)
    scale = np.repeat(((groups.astype(np.uint32) & 0x7FF0) << 16).astype(np.uint32).view(F).astype(np.float64), 32, -1)
    def order(x):
        return x.transpose(0, 2, 1, 3).reshape(-1, H, D)[:n]
    return order(decode(words, groups)), order(scale)


def rotate(x, cos, sin, pairs):
    """float32 rows [T, H, D], angles of every row [T, R]: products and sums rounded one by one"""
    R = cos.shape[-1]
    y = np.asarray(x, F).copy()
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if pairs else (y[..., :R // 2], y[..., R // 2:R])
    c, s = cos[:, None, :R // 2].astype(F), sin[:, None, :R // 2].astype(F)
    u, v = a * c - b * s, b * c + a * s
    if pairs:
        y[..., 0:R:2], y[..., 1:R:2] = u, v
    else:
        y[..., :R // 2], y[..., R // 2:R] = u, v
    return y


def attention(q, k, v, scale_of, ctx, window, softcap, sinks, scale, keys=None):
    """q float64 [n, heads, D], k, v, scale_of [m, kv_heads, D], the rows being the last n of ctx positions; keys: how many are seen at
    most.  Returns (output, sum of weight x 15 x the value's scale, the largest sum of |q| |k| x scale) per row and head."""
    n, Hq, D = q.shape
    H = k.shape[1]
    out, spread, size = np.zeros((n, Hq, D)), np.zeros((n, Hq, D)), np.zeros((n, Hq))
    for i in range(n):
        pos = ctx - n + i
        j = np.arange(max(0, pos - window + 1) if window else 0, max(0, min(pos + 1, ctx, k.shape[0] if keys is None else keys)))
        if not len(j):
            continue
        for h in range(Hq):
            g = h // (Hq // H)
            x = (k[j, g] @ q[i, h]) * scale
            size[i, h] = (np.abs(k[j, g]) @ np.abs(q[i, h])).max() * scale
            if softcap:
                x = softcap * np.tanh(x / softcap)
            top = max(x.max(), sinks[h] if sinks is not None else -math.inf)
            w = np.exp(x - top)
            w /= w.sum() + (math.exp(sinks[h] - top) if sinks is not None else 0.0)
            out[i, h] = w @ v[j, g]
            spread[i, h] = w @ (15 * scale_of[j, g])
    return out, spread, size


HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}


def bound(ref, spread, size, D, dtype, softcap):
    """What an output may be off.  Its own rounding; a weight's: bfloat16 (half a step 2^-8) where rows are of that type, two such terms (2^-16) and an
    exponent of up to 72 in float32 (2^-18) where they are float16, three (2^-23) where they have 32 bits, on codes up to 15 scales; for rows of 16 bits
    32 float32 additions (truncated, 2^-23) of bytes up to 17 codes; and what the score is off moves a weight by as much, relatively, numerator and denominator:
    D + 8 float32 roundings of a sum of |q k|, the query's own representation (2^-22, two float16 terms; 2^-25 of the largest element below
    float16's range), the exponential (2^-21) and a tanh (2^-21 of the cap)."""
    weight = {"float32": 2.0 ** -23, "float16": 2.0 ** -16 + 2.0 ** -18 + 17 * 32 * 2.0 ** -23, "bfloat16": 2.0 ** -8 + 17 * 32 * 2.0 ** -23}[dtype]
    score = (D + 12) * 2.0 ** -24 * size + 2.0 ** -21 + (2.0 ** -21 * softcap if softcap else 0.0)
    return HALF_STEP[dtype] * np.abs(ref) + spread * (weight + 2 * score[..., None] + (D + 64) * 2.0 ** -24) + 1e-30


def select(logits, scores, n, finished=None, pad=0):
    """[groups, n] scores, beams, tokens in float64, ties to the lowest (beam, token)"""
    B, K = scores.shape
    V = logits.shape[-1]
    x = np.asarray(logits, np.float64).reshape(B, K, V)
    out = np.zeros((B, n)), np.zeros((B, n), np.int32), np.zeros((B, n), np.int32)
    for b in range(B):
        c = np.full((K, V), -np.inf)
        for k in range(K):
            if finished is not None and finished[b, k]:
                c[k, pad] = scores[b, k] if scores[b, k] == scores[b, k] else -np.inf
                continue
            r = x[b, k]
            top = r.max()
            if not scores[b, k] > -1e30 or not np.isfinite(top):
                continue
            c[k] = float(scores[b, k]) + (r - (top + math.log(math.fsum(np.exp(r - top)))))
        flat = c.reshape(-1)
        order = np.lexsort((np.arange(flat.size), -flat))[:n]
        out[0][b], out[1][b], out[2][b] = flat[order], order // V, order % V
    return out
