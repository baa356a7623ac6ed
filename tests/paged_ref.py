"""NumPy oracle in 64 bits of the operators on pages of 16 and 32 bits: attention under masks, weights by position, what stays, rows that move, trees."""
import numpy as np

from pygpukit_b200.core.dtypes import bf16_bits_to_f32, f32_to_bf16_bits

EPS = {"bfloat16": 2.0 ** -7, "float16": 2.0 ** -10, "float32": 2.0 ** -23}


def rounded(x, dtype):
    """as the arrays hold it (bfloat16: bits)"""
    x = np.asarray(x, np.float32)
    return f32_to_bf16_bits(x) if dtype == "bfloat16" else x.astype(dtype)


def floats(a, dtype):
    return (bf16_bits_to_f32(a) if dtype == "bfloat16" else np.asarray(a)).astype(np.float64)


def tree(rng, n, deep=False):
    """parents of a tree of n rows: row 0 the root"""
    p = [-1]
    for i in range(1, n):
        p.append(int(rng.integers(max(0, i - 2) if deep else 0, i)))
    return p


def ancestors(parents):
    n = len(parents)
    m = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            m[i] = m[p]
        m[i, i] = True
    return m


def words(masks, count):
    """rows of truth values as int32 words"""
    out = np.zeros((len(masks), 32 * count), np.uint8)
    for i, m in enumerate(masks):
        k = min(len(m), 32 * count)
        out[i, :k] = np.asarray(m)[:k]
    return np.packbits(out, axis=1, bitorder="little").view(np.int32)


class Pages:
    """a cache whose pages are in any order; rows that nobody wrote are NaN"""

    def __init__(self, rng, contexts, H, D, ps, dtype, spare=2, slots=None, std=1.0):
        S = len(contexts)
        self.H, self.D, self.ps, self.dtype, self.contexts = H, D, ps, dtype, list(contexts)
        per = max(1, -(-max([1, *contexts]) // ps))
        n_slots = (slots or S) + 1
        self.n_slots, self.positions = n_slots, per * ps
        self.pages = n_slots * per + spare
        self.table = rng.permutation(self.pages)[:n_slots * per].reshape(n_slots, per).astype(np.int32)
        self.slots = rng.permutation(n_slots)[:S].astype(np.int32)
        nan = rounded(np.full((self.pages, H, ps, D), np.nan), dtype)
        self.k, self.v = nan.copy(), nan.copy()
        for s, ctx in enumerate(contexts):
            for a in (self.k, self.v):
                self.put(a, s, range(ctx), rounded(rng.standard_normal((ctx, H, D)) * std, dtype))

    def put(self, a, s, positions, rows):
        for j, row in zip(positions, rows):
            a[self.table[self.slots[s], j // self.ps], :, j % self.ps] = row

    def rows(self, a, s, n):
        """[n, H, D] in 64 bits"""
        if n <= 0:
            return np.zeros((0, self.H, self.D))
        j = np.arange(n)
        return floats(a[self.table[self.slots[s], j // self.ps], :, j % self.ps], self.dtype)


def attention(pages, q, starts, masks=None, scale=None, keys=None):
    """(out, lse, what a weight's error is made of, weights by position [S, H, positions]) of steps whose rows see each other by masks (lists of rows of truth values)"""
    T, Hq, D = q.shape
    rep, scale = Hq // pages.H, scale or 1.0 / np.sqrt(D)
    out, lse, spread, size = np.zeros(q.shape), np.full((T, Hq), -np.inf), np.zeros(q.shape), np.zeros((T, Hq))
    weights = np.zeros((len(pages.contexts), pages.H, pages.positions))
    for s, ctx in enumerate(pages.contexts):
        a, b = starts[s], starts[s + 1]
        n = b - a
        k, v = pages.rows(pages.k, s, ctx), pages.rows(pages.v, s, ctx)
        end = ctx if keys is None else min(ctx, keys)
        for i in range(n):
            seen = np.zeros(ctx, bool)
            seen[:max(0, ctx - n)] = True
            for t in range(n):
                j = ctx - n + t
                if j >= 0:
                    seen[j] = t <= i if masks is None else (t < len(masks[a + i]) and bool(masks[a + i][t]))
            seen[end:] = False
            if not seen.any():
                continue
            at = np.flatnonzero(seen)
            for h in range(Hq):
                g = h // rep
                with np.errstate(all="ignore"):
                    x = scale * (k[at, g] @ q[a + i, h])
                    top = x.max()
                    w = np.exp(x - top)
                    out[a + i, h] = w @ v[at, g] / w.sum()
                    lse[a + i, h] = top + np.log(w.sum())
                    spread[a + i, h] = w @ np.abs(v[at, g]) / w.sum()
                    size[a + i, h] = scale * (np.abs(k[at, g]) @ np.abs(q[a + i, h])).max()
                    weights[s, g, at] += w / w.sum()
    return out, lse, spread, size, weights


def score_error(size, D):
    """how far a score may be off: D products added in float32, each addition truncated; the factor and the exponent's argument, rounded"""
    return size[..., None] * (D + 4) * 2.0 ** -23


def bound(out, spread, size, D, keys, dtype):
    """how far an output may be off.  A weight: its score's error (twice, the reference has it too), the exponential's 2 units, and its own rounding to the rows' type; sums of at most
    `keys` additions of float32; the output's rounding, half a unit"""
    e = EPS[dtype]
    weight = 2 * score_error(size, D) + 2.0 ** -21 + (e / 2 if dtype != "float32" else 0.0)
    sums = 2 * (keys / 16 + 64) * 2.0 ** -23
    small = keys * 2.0 ** -31 if dtype == "float16" else 0.0        # weights below 2^-14 of float16 come in steps of 2^-24, where the largest is 2^6
    return (weight + sums + small) * spread + e / 2 * np.abs(out) + 1e-30 + (2.0 ** -25 if dtype == "float16" else 0.0)


def select(weights, slots, contexts, budget, first, recent):
    S, H = len(contexts), weights.shape[1]
    kept, counts = np.full((S, H, budget), -1, np.int32), np.zeros(S, np.int32)
    for s, ctx in enumerate(contexts):
        if not 0 <= slots[s] < weights.shape[0]:
            continue
        ctx = min(max(0, ctx), weights.shape[2])
        counts[s] = n = min(ctx, budget)
        for h in range(H):
            w = weights[slots[s], h, :ctx].astype(np.float64)
            order = sorted(range(ctx), key=lambda j: (0 if j < first or j >= ctx - recent else 1, np.isnan(w[j]), -w[j] if not np.isnan(w[j]) else 0.0, j))
            kept[s, h, :n] = sorted(order[:n])
    return kept, counts


def accept(chosen, tokens, parents, starts, max_rows):
    S = len(starts) - 1
    rows, counts, nxt = np.full((S, max_rows), -1, np.int32), np.zeros(S, np.int32), np.full(S, -1, np.int32)
    for s in range(S):
        a, n = starts[s], min(starts[s + 1] - starts[s], max_rows)
        cur = 0 if n > 0 else -1
        while cur >= 0:
            rows[s, counts[s]] = cur
            counts[s] += 1
            nxt[s] = chosen[a + cur]
            cur = next((j for j in range(cur + 1, n) if parents[a + j] == cur and tokens[a + j] == nxt[s]), -1)
    return rows, counts, nxt
