"""Attention over the four-bit cache at the ends of its ranges: windows, contexts and caps of any size, long sums, weights that have fallen to zero; and
prompts whose tiles are made once, with pages, rows and values missing."""
import numpy as np
import pytest

from tests import kv4_ref as ref
from tests.test_gpu_int4_cache import Attend

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------- windows
WIDE = [  # (context, rows): a few, many, and many enough for tiles made once; rows before position 0 among them
    ([(3, 5), (70, 2), (1, 4)], "float32"),
    ([(3, 5), (70, 2), (1, 4)], "bfloat16"),
    ([(20, 60), (150, 40)], "bfloat16"),
    ([(100, 220), (300, 200)], "bfloat16"),
    ([(100, 220), (300, 200)], "float16"),
]


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30, 64])
@pytest.mark.parametrize("portions,dtype", WIDE, ids=str)
def test_windows_of_any_size(portions, dtype, window):
    """a window that reaches below position -2^31 is no window: rows before position 0 see nothing, the others everything"""
    a = Attend(portions, 8, 2, 128, 16, dtype, window=window, seed=50)
    got = a.run()
    a.check(got)
    for (ctx, n), at in zip(a.portions, a.starts):
        assert (got[at:at + max(0, n - ctx)] == 0).all() and (got[at + max(0, n - ctx):at + n] != 0).any(-1).all()
    if window > 2 ** 29:
        a.window = 0
        assert np.array_equal(a.run(), got)


# ---------------------------------------------------------------------------------------------------- long sums
class Shared(Attend):
    """64 decoded tokens over one slot's pages, of unequal contexts: sequences enough that few blocks share one's keys, and a warp adds thousands of them"""

    def __init__(self, ctx, D, rep, dtype, H=8, seed=60):
        super().__init__([(ctx, 1)], H * rep, H, D, 64, dtype, seed=seed)
        S = 64
        self.slots, self.portions = np.repeat(self.slots, S), [(ctx - 7 * i, 1) for i in range(S)]
        self.starts, self.T = np.arange(S + 1, dtype=np.int32), S
        factor = np.where(np.arange(S) % 2, 1.0, 0.02)[:, None, None]         # weights that differ, and all alike
        self.q = ref.rounded(np.random.default_rng(seed + 1).standard_normal((S, H * rep, D)) * factor, dtype)

    def rows(self, arr, h):
        """one head's values and scales"""
        got = ref.rows_of(arr[:, h:h + 1], self.c.table, self.slots[0], self.top)
        return tuple(x[:, 0] for x in got)

    def check(self, got, ignore=None):
        """`ignore`: a group of elements that is not compared"""
        q, rep = ref.floats(self.q, self.dtype).astype(np.float64), self.Hq // self.c.H
        seen = np.arange(self.top) < np.array([c for c, _ in self.portions])[:, None]
        keep = np.ones(self.D, bool)
        if ignore is not None:
            keep[32 * ignore:32 * ignore + 32] = False
        for h in (0, self.Hq - 1):
            (k, _), (v, s) = self.rows(self.c.k, h // rep), self.rows(self.c.v, h // rep)
            x = np.where(seen, q[:, h] @ k.T / np.sqrt(self.D), -np.inf)
            w = np.exp(x - x.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            size = np.where(seen, np.abs(q[:, h]) @ np.abs(k).T, 0).max(1) / np.sqrt(self.D)
            want, spread = w @ v[:, keep], w @ (15 * s[:, keep])
            off, tol = np.abs(got[:, h][:, keep] - want), ref.bound(want, spread, size, self.D, self.dtype, 0.0)
            print(f"worst {(off / tol).max():.3f} of the bound, rms {np.sqrt(np.mean(off ** 2)):.3e} of {np.sqrt(np.mean(want ** 2)):.3e}")
            assert (off <= tol).all()


@pytest.mark.parametrize("ctx,D,rep,dtype", [(65536, 64, 1, "float16"), (65536, 64, 1, "bfloat16"), (20011, 96, 2, "float32"), (30000, 128, 4, "float16")])
def test_sums_over_many_keys(ctx, D, rep, dtype):
    """the bound has 32 truncated additions, whatever the context"""
    a = Shared(ctx, D, rep, dtype)
    a.check(a.run(False))


@pytest.mark.parametrize("D,rep,dtype", [(64, 1, "float16"), (128, 2, "bfloat16"), (128, 4, "float32"), (256, 1, "float16")])
def test_maxima_that_grow_along_the_context(D, rep, dtype):
    """references move long after the first sums were put aside"""
    ctx = 9000
    a = Shared(ctx, D, rep, dtype)
    for h in range(8):
        x = (a.rows(a.c.k, h)[0] * (1 + 40 * np.arange(ctx) / ctx)[:, None]).astype(np.float32)
        words, groups = ref.encode(x)
        for page in range(-(-ctx // 64)):
            n = min(64, ctx - 64 * page)
            flat = a.c.k[a.c.table[a.slots[0], page], h].reshape(-1)
            flat[:n * D // 2] = words[64 * page:64 * page + n].reshape(-1).view(np.uint8)
            flat[32 * D:32 * D + n * D // 16] = np.ascontiguousarray(groups[64 * page:64 * page + n]).reshape(-1).view(np.uint8)
    a.c.upload()
    a.check(a.run(False))


@pytest.mark.parametrize("at", [0, 5990])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_a_value_that_is_nan_in_a_long_sum(dtype, at):
    a = Shared(6000, 128, 1, dtype)
    for h in range(8):
        page, row = a.c.table[a.slots[0], at // 64], at % 64
        words, groups = ref.get(a.c.v, page, h, row)
        groups[1] = ref.NAN_WORD
        ref.put(a.c.v, page, h, row, words, groups)
    a.c.upload()
    got = a.run(False)
    sees = np.array([c for c, _ in a.portions]) > at
    nan = np.zeros(got.shape, bool)
    nan[sees, :, 32:64] = True
    assert np.array_equal(np.isnan(got), nan)
    a.check(got, ignore=1)


@pytest.mark.parametrize("rows,dtype", [(1, "bfloat16"), (1, "float32"), (3, "float16"), (3, "float32"), (60, "bfloat16"), (250, "float16")])
@pytest.mark.parametrize("at", [40, 296])
def test_a_nan_under_a_weight_of_zero(rows, dtype, at):
    """A key whose score is some thousand below the largest is seen all the same: its value's NaN shows, as 0 NaN does, in whatever block of keys it lies"""
    a = Attend([(300, rows)], 4, 2, 128, 16, dtype, seed=65)
    one = np.sign(np.random.default_rng(66).standard_normal(128))
    a.q = ref.rounded(np.broadcast_to(one, a.q.shape), dtype)
    page, row = a.c.table[a.slots[0], at // 16], at % 16
    words, groups = ref.encode((-300 * one).astype(np.float32)[None])      # a score of -3394
    for h in (0, 1):
        ref.put(a.c.k, page, h, row, words[0], groups[0])
    words, groups = ref.get(a.c.v, page, 1, row)
    groups[2] = ref.NAN_WORD
    ref.put(a.c.v, page, 1, row, words, groups)
    a.c.upload()
    nan = np.zeros((a.T + 2, 4, 128), bool)
    nan[max(0, at - (300 - rows)):rows, 2:, 64:96] = True
    assert np.array_equal(np.isnan(a.run()), nan)


# ---------------------------------------------------------------------------------------------------- caps
@pytest.mark.parametrize("rows,dtype", [(1, "bfloat16"), (3, "float16"), (3, "float32"), (60, "bfloat16"), (60, "float16"), (250, "bfloat16")])
@pytest.mark.parametrize("cap", [1e-36, 1e-3, 0.5, 170.0, 180.0, 5000.0, 1e6, 1e30])
def test_caps_of_any_size(rows, dtype, cap):
    """Up to KV4_CAP_WIDE (256 units of log2 e: 177) a cap is off by 2^-21 of itself; above, by a score's 2^-20, which the score's own bound has"""
    a = Attend([(300, rows), (70, min(rows, 50))], 4, 2, 128, 16, dtype, softcap=cap, seed=70, scale=0.7)
    got = a.run()
    want, spread, size = a.exact()
    tol = ref.bound(want, spread, size, 128, dtype, cap if cap < 177 else 0.0)
    off = np.abs(got[:a.T] - want)
    print(f"worst {(off / tol).max():.3f} of the bound")
    assert (off <= tol).all()


# ---------------------------------------------------------------------------------------------------- prompts: what is not there, in both kinds of tiles
MANY = [  # rows of the longest sequence, elements, page, type, window: tiles made by the blocks, and (768 rows a key head) made once
    (40, 128, 16, "bfloat16", 0), (60, 64, 48, "float16", 90), (50, 96, 16, "bfloat16", 33),
    (200, 128, 16, "float16", 0), (210, 64, 80, "bfloat16", 150), (195, 96, 32, "float16", 0), (230, 128, 64, "bfloat16", 70),
]


def many(rows, D, PS, dtype, window, seed=80):
    return Attend([(300, rows), (260, 30), (19, 19)], 8, 2, D, PS, dtype, window=window, seed=seed)


def masked(a, there):
    """float64 outputs and their bound over the keys j of sequence s with there[s][j]"""
    want, tol = np.zeros((a.T, a.Hq, a.D)), np.zeros((a.T, a.Hq, a.D))
    rep = a.Hq // a.c.H
    for i, ((ctx, n), slot, at) in enumerate(zip(a.portions, a.slots, a.starts)):
        k, _ = ref.rows_of(a.c.k, a.c.table % a.c.pages, slot, ctx)
        v, s = ref.rows_of(a.c.v, a.c.table % a.c.pages, slot, ctx)
        q = ref.floats(a.q[at:at + n], a.dtype).astype(np.float64)
        pos, j = np.arange(ctx - n, ctx)[:, None], np.arange(ctx)
        seen = (j <= pos) & (j > pos - (a.window or ctx + 1)) & there[i]
        for h in range(a.Hq):
            x = np.where(seen, q[:, h] @ k[:, h // rep].T / np.sqrt(a.D), -np.inf)
            top = x.max(1, keepdims=True)
            w = np.where(seen, np.exp(x - np.where(np.isfinite(top), top, 0.0)), 0.0)
            w /= np.maximum(w.sum(1, keepdims=True), 1e-300)
            want[at:at + n, h] = w @ v[:, h // rep]
            size = np.where(seen, np.abs(q[:, h]) @ np.abs(k[:, h // rep]).T, 0).max(1) / np.sqrt(a.D)
            tol[at:at + n, h] = ref.bound(want[at:at + n, h], w @ (15 * s[:, h // rep]), size, a.D, a.dtype, 0.0)
    return want, tol


@pytest.mark.parametrize("rows,D,PS,dtype,window", MANY)
def test_prompts_over_pages_that_do_not_exist(rows, D, PS, dtype, window):
    a = many(rows, D, PS, dtype, window)
    there = [np.ones(c, bool) for c, _ in a.portions]
    for i, slot in enumerate(a.slots):
        for page, number in ((1, -5), (3, a.c.pages), (0, 2 ** 31 - 1)):      # the first page too: early rows see nothing
            if page < a.c.table.shape[1]:
                a.c.table[slot, page] = number
                there[i][page * PS:(page + 1) * PS] = False
    a.c.upload()
    got = a.run()
    want, tol = masked(a, there)
    assert (np.abs(got[:a.T] - want) <= tol).all() and (got[a.T:] == 77.0).all()


@pytest.mark.parametrize("rows,D,PS,dtype,window", MANY)
def test_prompts_over_stale_bytes(rows, D, PS, dtype, window):
    """whatever lies behind a context or before a window, NaN scales among it, leaves the output's bits alone"""
    a = many(rows, D, PS, dtype, window)
    clean = a.run()
    a.check(clean)
    used = np.zeros((a.c.pages, PS), bool)
    for (ctx, n), slot in zip(a.portions, a.slots):
        j = np.arange(max(0, ctx - n - window + 1) if window else 0, ctx)
        used[a.c.table[slot, j // PS], j % PS] = True
    for arr in (a.c.k, a.c.v):
        for page, row in zip(*np.nonzero(~used)):
            for h in range(2):
                words, groups = ref.get(arr, page, h, row)
                ref.put(arr, page, h, row, words, np.full_like(groups, ref.NAN_WORD))
    a.c.upload()
    assert np.array_equal(a.run(), clean)


@pytest.mark.parametrize("rows,D,PS,dtype,window", MANY)
@pytest.mark.parametrize("where", ["key", "value"])
def test_prompts_and_a_nan(where, rows, D, PS, dtype, window):
    """a NaN in the middle of the rows' own keys reaches the rows behind it, within its window, of its head's group; of a value, its elements alone"""
    a = many(rows, D, PS, dtype, window)
    at = 300 - rows + rows // 2
    arr = a.c.k if where == "key" else a.c.v
    page, row = a.c.table[a.slots[0], at // PS], at % PS
    words, groups = ref.get(arr, page, 1, row)
    groups[1] = ref.NAN_WORD
    ref.put(arr, page, 1, row, words, groups)
    a.c.upload()
    nan = np.zeros((a.T + 2, 8, D), bool)
    last = min(rows, rows // 2 + window) if window else rows
    if where == "key":
        nan[rows // 2:last, 4:] = True
    else:
        nan[rows // 2:last, 4:, 32:64] = True
    assert np.array_equal(np.isnan(a.run()), nan)


@pytest.mark.parametrize("rows,D,PS,dtype,window", MANY)
def test_prompts_of_fewer_rows_than_there_are(rows, D, PS, dtype, window):
    """rows from max_rows on, sequences without a slot and starts that reach outside: outputs stay, and nothing else changes"""
    a = many(rows, D, PS, dtype, window)
    full = a.run()
    few = rows - 3
    got = a.run(max_rows=few)
    keep = np.ones(a.T + 2, bool)
    keep[few:rows] = False
    assert np.array_equal(got[keep], full[keep]) and (got[few:rows] == 77.0).all()
    slots = a.slots.copy()
    for bad in (-1, 99):
        a.slots[1] = bad
        got = a.run()
        assert (got[rows:rows + 30] == 77.0).all() and np.array_equal(np.delete(got, np.s_[rows:rows + 30], 0), np.delete(full, np.s_[rows:rows + 30], 0))
    a.slots = slots
    a.starts = np.array([-4, rows, rows + 30, 2 ** 30], np.int32)
    got = a.run(max_rows=rows + 10)
    assert np.isfinite(got).all() and np.array_equal(got[rows:rows + 30], full[rows:rows + 30])
