"""Keys and values in four bits: rows into the paged cache (bit for bit) and back, and attention over it against float64."""
import math

import numpy as np
import pytest

from pygpukit_b200 import ops
from pygpukit_b200._lib import api
from pygpukit_b200.core.dtypes import bfloat16, float16, float32
from pygpukit_b200.core.factory import empty, from_numpy, zeros
from pygpukit_b200.core.stream import CudaGraph, Stream, synchronize, use_stream
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"bfloat16": bfloat16, "float16": float16, "float32": float32}


def i32(x):
    return from_numpy(np.ascontiguousarray(np.asarray(x, np.int32)))


def tables(n, R, theta=1e4):
    a = np.arange(n)[:, None] * theta ** (-np.arange(0, R, 2) / R)
    return tuple(np.ascontiguousarray(np.concatenate([f(a), f(a)], 1).astype(np.float32)) for f in (np.cos, np.sin))


class Cache:
    """a cache whose pages are in any order, every byte of it known"""

    def __init__(self, rng, slots, ctx, H, D, PS, spare=2, fill=True):
        self.rng, self.H, self.D, self.PS = rng, H, D, PS
        per = max(1, -(-ctx // PS))
        self.pages = slots * per + spare
        self.table = rng.permutation(self.pages)[:slots * per].reshape(slots, per).astype(np.int32)
        shape = (self.pages, H, PS, ops.int4_row_bytes(D))
        self.k, self.v = (rng.integers(0, 256, shape, dtype=np.uint8) for _ in range(2))
        if fill:
            for a in (self.k, self.v):
                x = rng.standard_normal((self.pages, H, PS, D)) * rng.uniform(0.2, 2.0, D) + rng.standard_normal(D) * 0.5
                words, groups = ref.encode(x.astype(np.float32))
                flat = a.reshape(self.pages, H, -1)
                flat[..., :PS * D // 2] = words.reshape(self.pages, H, -1).view(np.uint8)
                flat[..., PS * D // 2:] = groups.reshape(self.pages, H, -1).view(np.uint8)
        self.upload()

    def upload(self):
        self.kd, self.vd, self.td = from_numpy(self.k), from_numpy(self.v), from_numpy(self.table)


# ---------------------------------------------------------------------------------------------------- append and read
APPENDS = [  # heads, kv heads, D, page, rotated, neighbours, type
    (8, 2, 128, 64, 128, False, "bfloat16"),
    (32, 8, 128, 16, 64, False, "float32"),
    (4, 4, 64, 32, 64, True, "float16"),
    (3, 1, 96, 48, 96, False, "bfloat16"),
    (5, 5, 96, 16, 32, True, "float32"),
    (6, 3, 192, 80, 96, False, "float16"),
    (2, 1, 256, 64, 256, False, "bfloat16"),
    (0, 2, 128, 64, 128, True, "bfloat16"),
    (4, 2, 64, 16, 0, False, "float32"),
]


@pytest.mark.parametrize("T", [1, 7, 40, 600])
@pytest.mark.parametrize("form", range(len(APPENDS)))
def test_append_is_the_format_bit_for_bit(form, T):
    Hq, H, D, PS, R, pairs, dtype = APPENDS[form]
    rng = np.random.default_rng(100 * form + T)
    slots = min(T, 5)
    ctx = -(-T // slots) + 37
    c = Cache(rng, slots, ctx, H, D, PS, fill=False)
    slot = np.arange(T, dtype=np.int32) % slots
    pos = (np.arange(T, dtype=np.int32) // slots + 21).astype(np.int32)
    q, k, v = (rng.standard_normal((T, n, D)) * s for n, s in ((Hq, 1.0), (H, 2.0), (H, 0.01)))
    k[T // 2, :, :32] = 0.0                                        # a group of zeros
    k[0, 0, 32:64] = np.abs(k[0, 0, 32:64])                        # one side only
    v[0, 0, :32] = -np.abs(v[0, 0, :32])
    v[T // 2, 0, 3] = 300.0                                        # an outlier
    v[T - 1, :, 32:64] = 2.0 ** -45                                # below the smallest scale
    q, k, v = (ref.rounded(x, dtype) for x in (q, k, v))
    qd, kd, vd = from_numpy(q), from_numpy(k), from_numpy(v)
    cos = sin = None
    if R:
        cos, sin = tables(ctx + 30, R)
    ops.rope_append_paged_int4(qd if Hq else None, kd, vd, from_numpy(cos) if R else None, from_numpy(sin) if R else None, c.kd, c.vd, c.td, i32(slot), i32(pos),
                               interleaved=pairs)
    turn = (lambda x: ref.rotate(ref.floats(x, dtype), cos[pos], sin[pos], pairs)) if R else (lambda x: ref.floats(x, dtype))
    held = {}
    for name, cache, x in (("k", c.k, turn(k)), ("v", c.v, ref.floats(v, dtype))):
        words, groups = ref.encode(x)
        held[name] = ref.decode(words, groups)
        for t in range(T):
            for h in range(H):
                ref.put(cache, c.table[slot[t], pos[t] // PS], h, pos[t] % PS, words[t, h], groups[t, h])
    assert np.array_equal(c.kd.to_numpy(), c.k) and np.array_equal(c.vd.to_numpy(), c.v)
    if Hq:
        want = ref.rounded(turn(q), dtype)
        assert np.array_equal(qd.to_numpy().view(np.uint8), np.ascontiguousarray(want).view(np.uint8))
    for out in (None, float32, float16):
        o = None if out is None else empty((T, H, D), out)
        got = ops.kv_read_paged_int4(c.vd, c.td, i32(slot), i32(pos), out=o)
        name = "bfloat16" if out is None else out.name
        x = ref.floats(got.to_numpy(), name)
        # what a group stands for is a bfloat16 number: 16 bits hold it, float16 where it is in range
        assert np.array_equal(x, held["v"].astype(np.float16).astype(np.float32) if out is float16 else held["v"].astype(np.float32))
    # no further off than a step, which is a fifteenth of at most twice the largest magnitude, rounded up by an eighth at most
    x, s = ref.floats(v, dtype).astype(np.float64), np.repeat(np.abs(ref.decode(*ref.encode(ref.floats(v, dtype)))).reshape(T, H, -1, 32).max(-1), 32, -1)
    assert (np.abs(held["v"] - x) <= 0.16 * s + 2.0 ** -36).all()


def test_append_takes_rows_of_a_fused_projection():
    """Strided rows, on and off 16-byte boundaries: the same bytes as packed ones."""
    rng = np.random.default_rng(5)
    Hq, H, D, T = 4, 2, 128, 9
    cos, sin = (from_numpy(x) for x in tables(64, D))
    slot, pos = i32(np.arange(T) % 3), i32(np.arange(T) // 3 + 11)
    got = []
    for off, ld in ((0, (Hq + 2 * H) * D), (0, (Hq + 2 * H) * D + 3), (1, (Hq + 2 * H) * D + 8)):
        c = Cache(np.random.default_rng(1), 3, 32, H, D, 16, fill=False)
        rows = np.zeros((T, ld), np.float32)
        rows[:, off:off + (Hq + 2 * H) * D] = np.random.default_rng(2).standard_normal((T, (Hq + 2 * H) * D))
        x = from_numpy(ref.rounded(rows, "bfloat16"))
        base = x.device_ptr + 2 * off
        api.kv4_append(base, base + 2 * Hq * D, base + 2 * (Hq + H) * D, ld, ld, ld, cos.device_ptr, sin.device_ptr, 64, D, 0, c.kd.device_ptr, c.vd.device_ptr,
                       c.pages, 16, c.td.device_ptr, 3, c.table.shape[1], slot.device_ptr, pos.device_ptr, T, Hq, H, D, 2, None)
        got.append((c.kd.to_numpy(), c.vd.to_numpy(), x.to_numpy()[:, off:off + Hq * D]))
        assert np.array_equal(x.to_numpy()[:, off + Hq * D:], ref.rounded(rows, "bfloat16")[:, off + Hq * D:])
    for other in got[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(got[0], other))


def test_rows_that_are_no_position_are_skipped():
    rng = np.random.default_rng(6)
    Hq, H, D, PS = 2, 1, 64, 16
    c = Cache(rng, 3, 64, H, D, PS, fill=False)
    c.table[1, 2], c.table[2, 0] = c.pages, -1                      # pages that do not exist
    c.upload()
    slot = np.array([-1, 0, 3, 0, 0, 1, 2, 2 ** 31 - 1, 0, 1], np.int32)
    pos = np.array([3, -1, 3, 64, 2 ** 31 - 1, 40, 5, 0, 50, 20], np.int32)
    ok = np.zeros(10, bool)
    ok[9] = True                                                    # position 50 is behind the tables
    q = rng.standard_normal((10, Hq, D)).astype(np.float32)
    k = rng.standard_normal((10, H, D)).astype(np.float32)
    cos, sin = tables(50, D)
    qd = from_numpy(q)
    ops.rope_append_paged_int4(qd, from_numpy(k), from_numpy(k), from_numpy(cos), from_numpy(sin), c.kd, c.vd, c.td, i32(slot), i32(pos))
    words, groups = ref.encode(k)
    ref.put(c.v, c.table[1, 1], 0, 4, words[9, 0], groups[9, 0])
    words, groups = ref.encode(ref.rotate(k[9:], cos[20:21], sin[20:21], False))
    ref.put(c.k, c.table[1, 1], 0, 4, words[0, 0], groups[0, 0])
    assert np.array_equal(c.kd.to_numpy(), c.k) and np.array_equal(c.vd.to_numpy(), c.v)
    assert np.array_equal(qd.to_numpy()[~ok], q[~ok]) and not np.array_equal(qd.to_numpy()[ok], q[ok])
    got = ops.kv_read_paged_int4(c.kd, c.td, i32(slot), i32(pos), out=empty((10, H, D), float32)).to_numpy()
    assert (got[[0, 1, 2, 3, 4, 5, 6, 7]] == 0).all() and (got[9] != 0).any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 2.0 ** 56])
def test_what_is_not_finite_comes_back_as_nan_in_its_group_alone(bad):
    rng = np.random.default_rng(7)
    c = Cache(rng, 1, 16, 2, 128, 16, fill=False)
    k = rng.standard_normal((1, 2, 128)).astype(np.float32)
    k[0, 1, 70] = bad
    ops.rope_append_paged_int4(None, from_numpy(k), from_numpy(k), None, None, c.kd, c.vd, c.td, i32([0]), i32([3]))
    got = ops.kv_read_paged_int4(c.kd, c.td, i32([0]), i32([3]), out=empty((1, 2, 128), float32)).to_numpy()
    nan = np.zeros((1, 2, 128), bool)
    nan[0, 1, 64:96] = True
    assert np.array_equal(np.isnan(got), nan)


# ---------------------------------------------------------------------------------------------------- attention
FORMS = [  # heads, kv heads, D, page, type, options
    dict(Hq=8, H=2, D=128, PS=64, dtype="bfloat16"),
    dict(Hq=32, H=8, D=128, PS=16, dtype="bfloat16", window=90),
    dict(Hq=4, H=4, D=64, PS=32, dtype="float16", softcap=20.0),
    dict(Hq=16, H=1, D=96, PS=48, dtype="bfloat16", sinks=True),
    dict(Hq=6, H=2, D=192, PS=80, dtype="float32", window=33, sinks=True),
    dict(Hq=12, H=3, D=128, PS=128, dtype="float32", softcap=30.0),
    dict(Hq=24, H=2, D=256, PS=64, dtype="bfloat16"),
    dict(Hq=40, H=1, D=64, PS=64, dtype="float32"),
    dict(Hq=7, H=7, D=256, PS=16, dtype="float16", window=1, sinks=True),
    dict(Hq=8, H=2, D=128, PS=64, dtype="float16"),
    dict(Hq=32, H=4, D=96, PS=32, dtype="float16", window=70, sinks=True),
]


class Attend:
    """sequences of (context, rows) over a cache; row -1 of the output belongs to nobody"""

    def __init__(self, portions, Hq, H, D, PS, dtype, window=0, softcap=0.0, sinks=False, seed=0, scale=0.0):
        rng = np.random.default_rng(seed)
        self.rng = rng
        self.portions, self.dtype, self.window, self.softcap, self.scale = portions, dtype, window, softcap, scale
        self.Hq, self.D = Hq, D
        S = len(portions)
        self.top = max([c for c, _ in portions] + [1])
        self.c = Cache(rng, S + 1, self.top, H, D, PS)
        self.slots = rng.permutation(S + 1)[:S].astype(np.int32)
        self.starts = np.cumsum([0] + [n for _, n in portions]).astype(np.int32)
        self.T = int(self.starts[-1])
        self.q = ref.rounded(rng.standard_normal((self.T + 2, Hq, D)) * 1.5, dtype)
        self.sinks = rng.standard_normal(Hq).astype(np.float32) if sinks else None
        self.single = all(n == 1 for _, n in portions)

    def run(self, starts=None, **kw):
        q = from_numpy(self.q if starts is not False else self.q[:self.T])
        out = from_numpy(ref.rounded(np.full(self.q.shape if starts is not False else self.q[:self.T].shape, 77.0), self.dtype))
        ops.sdpa_paged_int4(q, self.c.kd, self.c.vd, out, self.c.td, i32(self.slots), i32([c for c, _ in self.portions]),
                            kw.pop("max_context", min(self.top, self.c.table.shape[1] * self.c.PS)), self.scale,
                            row_starts=None if starts is False else i32(self.starts), max_rows=kw.pop("max_rows", max(n for _, n in self.portions)),
                            window=self.window, softcap=self.softcap, sinks=from_numpy(self.sinks) if self.sinks is not None else None, **kw)
        return ref.floats(out.to_numpy(), self.dtype).astype(np.float64)

    def exact(self, keys=None):
        outs = []
        scale = self.scale or 1.0 / math.sqrt(self.D)
        for (ctx, n), slot, at in zip(self.portions, self.slots, self.starts):
            k, s = ref.rows_of(self.c.k, self.c.table, slot, max(1, ctx))
            v, s = ref.rows_of(self.c.v, self.c.table, slot, max(1, ctx))
            q = ref.floats(self.q[at:at + n], self.dtype).astype(np.float64)
            outs.append(ref.attention(q, k, v, s, ctx, self.window, self.softcap, self.sinks, scale, keys))
        return tuple(np.concatenate([o[i] for o in outs]) for i in range(3))

    def check(self, got, keys=None):
        want, spread, size = self.exact(keys)
        off = np.abs(got[:self.T] - want)
        tol = ref.bound(want, spread, size, self.D, self.dtype, self.softcap)
        worst = np.unravel_index(np.argmax(off / tol), off.shape)
        print(f"worst {off[worst]:.3e} of {tol[worst]:.3e}, rms {np.sqrt(np.mean(off ** 2)):.3e} of {np.sqrt(np.mean(want ** 2)):.3e}")
        assert (off <= tol).all()
        assert (got[self.T:] == 77.0).all()


@pytest.mark.parametrize("form", range(len(FORMS)))
def test_one_row_each(form):
    a = Attend([(c, 1) for c in (1, 2, 15, 16, 17, 63, 64, 65, 130, 401)], seed=form, **FORMS[form])
    a.check(a.run())
    assert np.array_equal(a.run(False), a.run()[:a.T])


@pytest.mark.parametrize("form", range(len(FORMS)))
def test_a_few_rows_each(form):
    a = Attend([(5, 5), (64, 3), (130, 2), (33, 1), (200, 7), (16, 4)], seed=20 + form, **FORMS[form])
    a.check(a.run())


@pytest.mark.parametrize("form", range(len(FORMS)))
def test_prompts_and_portions(form):
    a = Attend([(150, 150), (260, 70), (1, 1), (129, 33)], seed=40 + form, **FORMS[form])
    a.check(a.run())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("ctx", [3000, 9001])
def test_long_contexts(ctx, dtype):
    a = Attend([(ctx, 1), (ctx - 700, 1), (40, 1)], 8, 2, 128, 64, dtype, seed=ctx)
    a.check(a.run(False))


@pytest.mark.parametrize("Hq,H", [(1, 1), (9, 1), (16, 1), (17, 1), (33, 1), (64, 2), (130, 1)])
def test_groups_of_any_size(Hq, H):
    a = Attend([(70, 1), (200, 3)], Hq, H, 64, 16, "bfloat16", seed=Hq)
    a.check(a.run())


def test_rows_that_see_nothing():
    """contexts of 0 or fewer, fewer positions than rows, sequences without rows, keys cut off: zeros, or nothing at all"""
    a = Attend([(0, 1), (3, 5), (20, 0), (64, 2), (40, 1)], 4, 2, 128, 16, "bfloat16", seed=3)
    got = a.run()
    a.check(got)
    assert (got[0] == 0).all() and (got[1:3] == 0).all() and (got[3] != 0).any()
    a.check(a.run(max_context=30), keys=30)
    assert (a.run(max_context=0)[:a.T] == 0).all()
    a.window = 4
    got = a.run(max_context=30)
    assert (got[6] == 0).all()                                     # position 62: its window lies behind the keys
    a.check(got, keys=30)


def test_padding_keeps_its_outputs():
    a = Attend([(30, 2), (50, 3), (70, 1)], 4, 2, 64, 16, "float32", seed=4)
    full = a.run()
    slots = a.slots.copy()
    a.slots[1] = -1
    got = a.run()
    assert (got[2:5] == 77.0).all() and np.array_equal(got[:2], full[:2]) and np.array_equal(got[5:], full[5:])
    a.slots[1] = 99
    assert (a.run()[2:5] == 77.0).all()
    a.slots = slots
    got = a.run(max_rows=2)                                         # the third row is not asked for
    assert np.array_equal(got[[0, 1, 2, 3, 5]], full[[0, 1, 2, 3, 5]]) and (got[4] == 77.0).all()


def test_starts_that_reach_outside_stay_inside():
    a = Attend([(30, 2), (50, 3), (70, 1)], 4, 2, 64, 16, "float32", seed=4)
    a.starts = np.array([-1, 2, 5, 2 ** 30], np.int32)
    got = a.run(max_rows=8)
    assert np.isfinite(got).all()


def test_pages_that_do_not_exist_are_not_seen():
    a = Attend([(100, 1), (100, 3)], 4, 2, 128, 16, "bfloat16", seed=5)
    before = a.c.table.copy()
    for slot in a.slots:
        a.c.table[slot, 2] = -5
        a.c.table[slot, 4] = a.c.pages
    a.c.upload()
    got = a.run()
    # the same keys, moved together
    keep = np.r_[0:32, 48:64, 80:100]
    scale = 1.0 / math.sqrt(a.D)
    for (ctx, n), slot, at in zip(a.portions, a.slots, a.starts):
        k, _ = ref.rows_of(a.c.k, before, slot, ctx)
        v, s = ref.rows_of(a.c.v, before, slot, ctx)
        q = ref.floats(a.q[at:at + n], a.dtype).astype(np.float64)
        for i in range(n):
            seen = keep[keep <= ctx - n + i]
            w, sp, sz = ref.attention(q[i:i + 1], k[seen], v[seen], s[seen], len(seen), 0, 0.0, None, scale)
            assert (np.abs(got[at + i] - w[0]) <= ref.bound(w, sp, sz, a.D, a.dtype, 0.0)[0]).all()


def test_stale_bytes_are_not_seen():
    """whatever lies behind a context or before a window, NaN scales among it, leaves the output's bits alone"""
    for rows in (1, 3, 80):
        a = Attend([(100, min(rows, 100)), (333, rows)], 8, 2, 128, 64, "bfloat16", window=70, seed=6)
        clean = a.run()
        used = np.zeros((a.c.pages, 64), bool)
        for (ctx, n), slot in zip(a.portions, a.slots):
            j = np.arange(max(0, ctx - n - 69), ctx)
            used[a.c.table[slot, j // 64], j % 64] = True
        for arr in (a.c.k, a.c.v):
            for page, row in zip(*np.nonzero(~used)):
                for h in range(2):
                    words, groups = ref.get(arr, page, h, row)
                    ref.put(arr, page, h, row, words, np.full_like(groups, ref.NAN_WORD))
        a.c.upload()
        assert np.array_equal(a.run(), clean)


@pytest.mark.parametrize("rows", [1, 3, 60])
@pytest.mark.parametrize("where", ["key", "value", "query"])
def test_nan_reaches_who_sees_it(where, rows):
    a = Attend([(200, rows), (90, rows)], 4, 2, 128, 16, "bfloat16", seed=7)
    at = 200 - rows + rows // 2                                     # seen by the later half of the rows, and by one head's group
    nan = np.zeros((a.T + 2, a.Hq, a.D), bool)
    if where == "query":
        a.q[rows // 2, 1, 5] = 0x7FC0
        nan[rows // 2, 1] = True
    else:
        arr = a.c.k if where == "key" else a.c.v
        page, row = a.c.table[a.slots[0], at // 16], at % 16
        words, groups = ref.get(arr, page, 1, row)
        groups[2] = ref.NAN_WORD
        ref.put(arr, page, 1, row, words, groups)
        a.c.upload()
        nan[rows // 2:rows, 2:, :] = True
        if where == "value":
            nan[rows // 2:rows, 2:, :64] = False
            nan[rows // 2:rows, 2:, 96:] = False
    assert np.array_equal(np.isnan(a.run()), nan)


@pytest.mark.parametrize("factor", [1e-20, 1e15])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_queries_and_values_of_any_size(factor, dtype):
    """queries far outside float16, values at the ends of the scales: what counts is relative"""
    a = Attend([(70, 1), (90, 4)], 4, 2, 128, 16, dtype, seed=8)
    a.q = ref.rounded(ref.floats(a.q, dtype) * factor, dtype)
    a.scale = 1.0 / factor / math.sqrt(128)
    got = a.run()
    want, spread, size = a.exact()
    assert (np.abs(got[:a.T] - want) <= ref.bound(want, spread, size, 128, dtype, 0.0)).all()
    a = Attend([(70, 1), (90, 4)], 4, 2, 128, 16, dtype, seed=8)
    x = np.random.default_rng(1).standard_normal((a.c.pages, 2, 16, 128)) * (2.0 ** 50 if factor > 1 else 2.0 ** -34)
    words, groups = ref.encode(x.astype(np.float32))
    flat = a.c.v.reshape(a.c.pages, 2, -1)
    flat[..., :16 * 64] = words.reshape(a.c.pages, 2, -1).view(np.uint8)
    flat[..., 16 * 64:] = groups.reshape(a.c.pages, 2, -1).view(np.uint8)
    a.c.upload()
    a.check(a.run())


@pytest.mark.parametrize("rows", [1, 4, 30])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_scores_near_the_end_of_float32(rows, dtype):
    """|q . k| of 10^36 and an all-zero key: one key has all of the weight, and nothing becomes infinite"""
    a = Attend([(70, rows)], 4, 2, 128, 16, dtype, seed=9)
    a.q = ref.rounded(ref.floats(a.q, dtype) * 1e36 / 1.5, dtype)
    words, groups = ref.encode(np.zeros((1, 128), np.float32))
    for h in (0, 1):
        ref.put(a.c.k, a.c.table[a.slots[0], 0], h, 5, words[0], groups[0])
    a.c.upload()
    got, (want, spread, _) = a.run(), a.exact()
    assert (np.abs(got[:a.T] - want) <= ref.bound(want, spread, np.zeros(want.shape[:2]), 128, dtype, 0.0)).all()


@pytest.mark.parametrize("rows", [1, 30])
def test_scores_of_large_keys(rows):
    """float16 rows over keys of 2^40: scores of 2^42 among zeros"""
    a = Attend([(300, rows)], 4, 2, 128, 16, "float16", seed=10)
    x = np.random.default_rng(2).standard_normal((a.c.pages, 2, 16, 128)) * 2.0 ** 40
    x[:, :, 3] = 0.0
    words, groups = ref.encode(x.astype(np.float32))
    flat = a.c.k.reshape(a.c.pages, 2, -1)
    flat[..., :16 * 64] = words.reshape(a.c.pages, 2, -1).view(np.uint8)
    flat[..., 16 * 64:] = groups.reshape(a.c.pages, 2, -1).view(np.uint8)
    a.c.upload()
    got, (want, spread, _) = a.run(), a.exact()
    assert (np.abs(got[:a.T] - want) <= ref.bound(want, spread, np.zeros(want.shape[:2]), 128, "float16", 0.0)).all()


def test_scores_far_apart_and_all_the_same():
    """one key that takes all the weight, wherever it lies; and queries of zero, whose output is the mean"""
    for at in (0, 63, 64, 150, 299):
        a = Attend([(300, 1)], 2, 1, 64, 16, "float32", seed=9, scale=3.0)
        q = ref.floats(a.q, "float32")
        k, _ = ref.rows_of(a.c.k, a.c.table, a.slots[0], 300)
        q[0] = 40.0 * k[at, 0]
        a.q = q.astype(np.float32)
        a.check(a.run())
    a = Attend([(300, 1), (300, 5)], 2, 1, 64, 16, "float32", seed=9)
    a.q = np.zeros_like(a.q)
    a.check(a.run())


def test_the_same_call_gives_the_same_bits():
    for form in (0, 3, 5):
        for portions in ([(5000, 1), (70, 1)], [(900, 6), (70, 2)], [(400, 300)]):
            a = Attend(portions, seed=11, **FORMS[form])
            first = a.run()
            assert all(np.array_equal(a.run(), first) for _ in range(3))


# ---------------------------------------------------------------------------------------------------- streams, graphs, a run of them
def test_a_step_on_a_stream_captured_and_replayed():
    """append and attend on a stream of their own, captured, then replayed on the next positions: as eager calls on the same inputs"""
    rng = np.random.default_rng(12)
    S, Hq, H, D, PS = 3, 8, 2, 128, 16
    ctx0 = np.array([5, 40, 400], np.int32)
    cos, sin = (from_numpy(x) for x in tables(600, D))
    inputs = [[ref.rounded(rng.standard_normal((S, n, D)), "bfloat16") for n in (Hq, H, H)] for _ in range(4)]

    def step(c, arrays, slots, pos, ctx, out):
        q, k, v = arrays
        ops.rope_append_paged_int4(q, k, v, cos, sin, c.kd, c.vd, c.td, slots, pos)
        ops.sdpa_paged_int4(q, c.kd, c.vd, out, c.td, slots, ctx, c.table.shape[1] * PS)

    slots = i32([2, 0, 1])
    c = Cache(np.random.default_rng(13), S, 500, H, D, PS)
    eager = []
    for n, x in enumerate(inputs):
        out = empty((S, Hq, D), bfloat16)
        step(c, [from_numpy(a) for a in x], slots, i32(ctx0 + n), i32(ctx0 + n + 1), out)
        eager.append(out.to_numpy())
    want = c.kd.to_numpy()

    c = Cache(np.random.default_rng(13), S, 500, H, D, PS)
    s, g = Stream(), CudaGraph()
    arrays = [empty((S, n, D), bfloat16) for n in (Hq, H, H)]
    pos, ctx, out = i32(ctx0), i32(ctx0 + 1), empty((S, Hq, D), bfloat16)
    synchronize()
    with g.capture(s):
        step(c, arrays, slots, pos, ctx, out)
    for n, x in enumerate(inputs):
        with use_stream(s):
            for a, b in zip(arrays, x):
                a.copy_from_numpy(b)
            pos.copy_from_numpy(ctx0 + n)
            ctx.copy_from_numpy(ctx0 + n + 1)
            g.replay(s)
            assert np.array_equal(out.to_numpy(), eager[n])
    assert np.array_equal(c.kd.to_numpy(), want)


def test_two_calls_at_once_on_two_streams():
    a, b = Attend([(6000, 1)], 8, 2, 128, 64, "bfloat16", seed=14), Attend([(5000, 1), (30, 1)], 8, 2, 128, 64, "bfloat16", seed=15)
    want = a.run(False), b.run(False)
    s, t = Stream(), Stream()

    def held(x):
        return dict(q=from_numpy(x.q[:x.T]), out=zeros((x.T, x.Hq, x.D), bfloat16), slots=i32(x.slots), ctx=i32([c for c, _ in x.portions]))

    ha, hb = held(a), held(b)
    synchronize()
    for _ in range(20):
        for stream, x, h in ((s, a, ha), (t, b, hb)):
            with use_stream(stream):
                ops.sdpa_paged_int4(h["q"], x.c.kd, x.c.vd, h["out"], x.c.td, h["slots"], h["ctx"], x.top)
    s.synchronize()
    t.synchronize()
    for h, w in ((ha, want[0]), (hb, want[1])):
        assert np.array_equal(ref.floats(h["out"].to_numpy(), "bfloat16").astype(np.float64), w)


@pytest.mark.parametrize("rows,dtype", [(6, "bfloat16"), (6, "float16"), (60, "bfloat16"), (300, "bfloat16"), (300, "float16"), (5, "float32")])
def test_two_captured_calls_replayed_at_once(rows, dtype):
    """graphs of two calls, made before either ran, with what work memory they have: side by side on two streams, and then eager calls"""
    both = [Attend([(700, rows), (400, rows // 2), (90, 1)], 8, 2, 128, 64, dtype, seed=18 + i) for i in (0, 1)]
    held = [dict(q=from_numpy(x.q), out=zeros(x.q.shape, TYPES[dtype]), slots=i32(x.slots), ctx=i32([c for c, _ in x.portions]), starts=i32(x.starts)) for x in both]

    def call(x, h):
        ops.sdpa_paged_int4(h["q"], x.c.kd, x.c.vd, h["out"], x.c.td, h["slots"], h["ctx"], x.top, row_starts=h["starts"], max_rows=rows)

    streams, graphs = [Stream(), Stream()], [CudaGraph(), CudaGraph()]
    synchronize()
    for s, g, x, h in zip(streams, graphs, both, held):
        with g.capture(s):
            call(x, h)
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with use_stream(s):
                g.replay(s)
    for s in streams:
        s.synchronize()
    got = [h["out"].to_numpy()[:x.T] for x, h in zip(both, held)]
    for x, h, g in zip(both, held, got):
        x.check(x.run())
        call(x, h)
        synchronize()
        assert np.array_equal(h["out"].to_numpy()[:x.T], g)


def test_outputs_over_their_queries():
    """out may be Q: a block has read all of its rows before one of them is written"""
    for rows, dtype in ((1, "float32"), (4, "bfloat16"), (70, "bfloat16"), (250, "float16")):
        x = Attend([(900, rows), (300, rows)], 8, 2, 128, 64, dtype, seed=30 + rows)
        want, q = x.run(), from_numpy(x.q)
        ops.sdpa_paged_int4(q, x.c.kd, x.c.vd, q, x.c.td, i32(x.slots), i32([c for c, _ in x.portions]), x.top, row_starts=i32(x.starts), max_rows=rows)
        assert np.array_equal(ref.floats(q.to_numpy(), dtype).astype(np.float64)[:x.T], want[:x.T])


def test_offsets_past_32_bits():
    """a cache of more than 4 GB: the last page is where it should be"""
    H, D, PS = 16, 256, 64
    row = ops.int4_row_bytes(D)
    pages = (1 << 32) // (H * PS * row) + 40
    small = Cache(np.random.default_rng(16), 1, 100, H, D, PS, spare=0)
    from pygpukit_b200.core.array import GPUArray
    from pygpukit_b200.core.dtypes import uint8
    try:
        big = [GPUArray((pages, H, PS, row), uint8) for _ in range(2)]
    except RuntimeError:
        pytest.skip("no room for two caches of 4 GB")
    table = np.array([[pages - 2, pages - 1]], np.int32)
    n = H * PS * row
    for arr, src in zip(big, (small.k, small.v)):
        for i, p in enumerate(table[0]):
            part = GPUArray((n,), uint8, ptr=arr.device_ptr + int(p) * n, source=arr)
            part.copy_from_numpy(src[small.table[0, i]].reshape(-1))
    x = ref.rounded(np.random.default_rng(17).standard_normal((1, 2 * H, D)), "bfloat16")
    kv = ref.rounded(np.random.default_rng(18).standard_normal((1, H, D)), "bfloat16")
    outs = []
    for k, v, t in ((small.kd, small.vd, small.td), (*big, from_numpy(table))):
        ops.rope_append_paged_int4(None, from_numpy(kv), from_numpy(kv), None, None, k, v, t, i32([0]), i32([99]))
        out = zeros((1, 2 * H, D), bfloat16)
        ops.sdpa_paged_int4(from_numpy(x), k, v, out, t, i32([0]), i32([100]), 100)
        outs.append((out.to_numpy(), ops.kv_read_paged_int4(k, t, i32([0]), i32([99])).to_numpy()))
    assert np.array_equal(outs[0][0], outs[1][0]) and np.array_equal(outs[0][1], outs[1][1])
