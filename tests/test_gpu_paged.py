"""Attention over pages of 16 and 32 bits, trees among them, and the weights summed by position, against float64."""
import numpy as np
import pytest

from pygpukit_b200 import ops
from pygpukit_b200.core.dtypes import bfloat16, float16, float32
from pygpukit_b200.core.factory import from_numpy
from pygpukit_b200.core.stream import CudaGraph, Stream, synchronize, use_stream
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"bfloat16": bfloat16, "float16": float16, "float32": float32}


def i32(x):
    return from_numpy(np.ascontiguousarray(np.asarray(x, np.int32)))


class Step:
    """sequences (context, rows), their cache and queries; masks: "chain" (none), "tree", "any" (rows that see nothing of the step, and of an empty context nothing at all)"""

    def __init__(self, portions, Hq, H, D, ps, dtype, masks="chain", seed=0, std=1.0, spare_words=0):
        rng = np.random.default_rng(seed)
        self.portions, self.Hq, self.D, self.dtype = portions, Hq, D, dtype
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in portions])]).astype(np.int32)
        self.T, self.max_rows, self.max_ctx = int(self.starts[-1]), max(1, max(n for _, n in portions)), max(c for c, _ in portions)
        self.p = ref.Pages(rng, [c for c, _ in portions], H, D, ps, dtype, std=std)
        self.q = ref.rounded(rng.standard_normal((self.T, Hq, D)) * 1.5, dtype)
        self.masks, self.parents = None, []
        if masks != "chain":
            self.masks = []
            for _, n in portions:
                tree = ref.tree(rng, n, deep=seed % 2 == 0) if n else []
                self.parents += tree
                m = ref.ancestors(tree) if masks == "tree" else rng.random((n, n)) < 0.4
                if masks == "any" and n > 1:
                    m[rng.integers(n)] = False
                self.masks += list(m)
            self.words = -(-self.max_rows // 32) + spare_words
        self.weights = rng.random((self.p.n_slots, H, self.p.positions)).astype(np.float32)

    def arrays(self):
        p = self.p
        return dict(q=from_numpy(self.q), k=from_numpy(p.k), v=from_numpy(p.v), table=from_numpy(p.table), slots=i32(p.slots), ctx=i32([c for c, _ in self.portions]),
                    starts=i32(self.starts), masks=None if self.masks is None else from_numpy(ref.words(self.masks, self.words)),
                    out=from_numpy(ref.rounded(np.full(self.q.shape, 7.0), self.dtype)), lse=from_numpy(np.full((self.T, self.Hq), 7.0, np.float32)),
                    weights=from_numpy(self.weights))

    def call(self, a, weigh=True, max_ctx=None, scale=0.0):
        max_ctx = self.max_ctx if max_ctx is None else max_ctx
        kw = dict(row_starts=a["starts"], max_rows=self.max_rows, masks=a["masks"])
        ops.sdpa_paged(a["q"], a["k"], a["v"], a["out"], a["table"], a["slots"], a["ctx"], max_ctx, scale, lse=a["lse"], **kw)
        if weigh:
            ops.weigh_paged(a["q"], a["k"], a["lse"], a["weights"], a["table"], a["slots"], a["ctx"], max_ctx, scale, **kw)

    def run(self, **kw):
        a = self.arrays()
        self.call(a, **kw)
        return self.read(a)

    def read(self, a):
        return ref.floats(a["out"].to_numpy(), self.dtype), a["lse"].to_numpy().astype(np.float64), a["weights"].to_numpy()

    def check(self, got, max_ctx=None, scale=None):
        out, lse, weights = got
        q = ref.floats(self.q, self.dtype)
        want, want_lse, spread, size, by = ref.attention(self.p, q, self.starts, self.masks, scale, max_ctx)
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(out), nan)
        fine = np.isfinite(want)
        assert np.array_equal(out[~fine & ~nan], want[~fine & ~nan])
        tol = ref.bound(want, spread, size, self.D, self.max_ctx, self.dtype)
        off = np.abs(out - want)[fine]
        print(f"worst {(off / tol[fine]).max(initial=0):.3f} of the bound, rms {np.sqrt(np.mean(off ** 2)) if off.size else 0:.2e} of {np.sqrt(np.mean(want[fine] ** 2)) if off.size else 0:.2e}")
        assert (off <= tol[fine]).all()
        none = want_lse == -np.inf
        assert np.array_equal(lse == -np.inf, none) and (out[none] == 0).all()
        ok = np.isfinite(want_lse)
        err = ref.score_error(size, self.D)[..., 0]
        assert (np.abs(lse[ok] - want_lse[ok]) <= (err + 2.0 ** -22 * np.abs(want_lse) + (self.max_ctx / 16 + 64) * 2.0 ** -23)[ok]).all()
        # a weight: twice a score's error, 2 units of the exponential and the logarithm's rounding; their sum, rounded
        most = np.exp(0.0) * (2 * err.max(initial=0, where=np.isfinite(err)) + 2.0 ** -20 + np.abs(want_lse[ok]).max(initial=0) * 2.0 ** -22)
        for s, slot in enumerate(self.p.slots):
            w, was = by[s], self.weights[slot]
            there = np.isfinite(w)
            d = np.abs(weights[slot].astype(np.float64) - (was + w))
            rows = (self.starts[s + 1] - self.starts[s]) * (self.Hq // self.p.H)
            assert (d <= most * w + (rows + 2) * 2.0 ** -23 * (was + w) + 1e-30)[there].all()
            assert np.array_equal(np.isnan(weights[slot]), np.isnan(w))
        free = np.setdiff1d(np.arange(self.p.n_slots), self.p.slots)
        assert np.array_equal(weights[free], self.weights[free])


STEPS = [  # portions, query heads, key heads, D, page, masks: one row, few, many; odd sizes; lengths of zero and one; pages that end inside a tile
    ([(1, 1)], 4, 1, 128, 64, "chain"),
    ([(300, 1), (17, 1), (1, 1)], 8, 8, 64, 16, "chain"),
    ([(513, 1), (512, 1)], 32, 4, 128, 64, "chain"),
    ([(200, 1)], 16, 1, 256, 48, "chain"),
    ([(130, 3), (3, 3), (0, 0), (70, 5)], 6, 2, 96, 32, "tree"),
    ([(130, 3), (4, 3), (5, 0), (70, 5)], 6, 2, 80, 100, "tree"),
    ([(40, 40)], 4, 2, 128, 16, "tree"),
    ([(1000, 8)], 32, 8, 128, 64, "tree"),
    ([(600, 64), (64, 64), (333, 31)], 8, 2, 128, 64, "tree"),
    ([(600, 33), (64, 64)], 8, 2, 64, 128, "tree"),
    ([(300, 70), (200, 40)], 6, 3, 72, 8, "tree"),
    ([(700, 130)], 4, 2, 96, 24, "any"),
    ([(260, 129), (129, 129)], 2, 1, 128, 40, "any"),
    ([(30, 30), (2, 2), (1, 1)], 2, 2, 128, 64, "any"),
    ([(260, 20), (9, 9)], 4, 1, 256, 64, "any"),
    ([(100, 12)], 7, 1, 8, 5, "tree"),
    ([(64, 10), (90, 11)], 12, 3, 192, 64, "tree"),
    ([(385, 200), (700, 300)], 4, 2, 128, 64, "chain"),
    ([(50, 50), (7, 7)], 3, 3, 104, 1, "chain"),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("portions,Hq,H,D,ps,masks", STEPS, ids=str)
def test_steps(portions, Hq, H, D, ps, masks, dtype):
    s = Step(portions, Hq, H, D, ps, dtype, masks, seed=D + ps)
    s.check(s.run())


@pytest.mark.parametrize("dtype,rows", [("bfloat16", 1), ("bfloat16", 60), ("float16", 1), ("float16", 60), ("float32", 2)])
def test_long_contexts_over_many_blocks(dtype, rows):
    s = Step([(9000, rows), (4097, 1)], 4, 2, 128, 64, dtype, "tree" if rows > 1 else "chain", seed=5)
    s.check(s.run())


@pytest.mark.parametrize("dtype,portions,Hq,H,D,ps,masks", [
    ("bfloat16", [(17000, 1)], 8, 2, 128, 64, "chain"), ("float16", [(17003, 3)], 8, 2, 96, 16, "tree"), ("bfloat16", [(0, 0), (17000, 50), (5, 5), (300, 7)], 6, 1, 128, 64, "any"),
    ("float16", [(9000, 140)], 2, 1, 64, 32, "tree"), ("bfloat16", [(9001, 20)], 4, 2, 80, 100, "tree"), ("bfloat16", [(6000, 2)], 2, 1, 256, 64, "tree"),
    ("float32", [(6000, 2), (3, 3)], 4, 1, 128, 64, "any"), ("float32", [(6001, 5)], 4, 2, 64, 16, "tree"), ("float32", [(5000, 3)], 2, 1, 256, 64, "tree")])
def test_long_contexts_over_blocks_that_are_no_cluster(dtype, portions, Hq, H, D, ps, masks):
    s = Step(portions, Hq, H, D, ps, dtype, masks=masks, seed=8)
    s.check(s.run())


@pytest.mark.parametrize("dtype,rows,Hq,D", [("bfloat16", 3, 2, 128), ("float16", 70, 2, 128), ("float32", 3, 2, 64)])
def test_values_that_are_not_finite_behind_a_long_context(dtype, rows, Hq, D):
    s = Step([(17000, rows)], Hq, 1, D, 64, dtype, masks="tree", seed=4)
    x = np.full((1, D), np.nan)
    s.p.put(s.p.v, 0, [17000 - rows + 1], ref.rounded(x, dtype))
    x[:, ::2] = -np.inf
    s.p.put(s.p.v, 0, [17000 - 1], ref.rounded(x, dtype))
    s.check(s.run())


@pytest.mark.parametrize("rows", [1, 9, 40])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_masks_make_what_no_masks_make(dtype, rows):
    a = Step([(300, rows), (rows, rows)], 4, 2, 128, 64, dtype, "chain", seed=9)
    plain = a.run()
    a.masks = [row for _, n in a.portions for row in np.tril(np.ones((n, n), bool))]
    a.words = -(-rows // 32) + 2                      # more words than a step needs
    got = a.run()
    a.check(got)
    for x, y in zip(got[:2], plain[:2]):
        assert np.allclose(x, y, rtol=2 ** -6, atol=1e-3)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,D", [(4, 128), (40, 128), (40, 64), (4, 256)])
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it(rows, D, dtype):
    s = Step([(150, rows), (99, rows)], 4, 2, D, 32, dtype, "tree", seed=11)
    at = 150 - rows
    for j, x in ((at, np.nan), (at + 2, np.inf), (at + 3, -np.inf), (20, np.nan)):
        if j == 20:
            continue
        row = np.asarray(s.p.v[s.p.table[s.p.slots[0], j // 32], :, j % 32]).copy()
        row[0, 5] = ref.rounded(np.array([x]), dtype)[0]
        s.p.put(s.p.v, 0, [j], [row])
    got = s.run()
    s.check(got)
    assert np.isnan(got[0]).any()                     # the first of them is the root's: every row of the tree sees it
    # and one of the context, which every row of its sequence sees
    row = np.asarray(s.p.v[s.p.table[s.p.slots[0], 0], :, 20]).copy()
    row[1, 3] = ref.rounded(np.array([np.nan]), dtype)[0]
    s.p.put(s.p.v, 0, [20], [row])
    got = s.run()
    assert np.isnan(got[0][:rows, 2:, 3]).all() and not np.isnan(got[0][:rows, 2:, 4]).any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,D", [(9, 128), (60, 128), (60, 96), (9, 200)])
def test_infinities_among_the_drafts(rows, D, dtype):
    s = Step([(150, rows), (99, rows)], 4, 2, D, 16, dtype, "tree", seed=11)
    for t, x in ((1, np.inf), (2, -np.inf), (rows - 1, np.nan)):
        j = 99 - rows + t
        row = np.asarray(s.p.v[s.p.table[s.p.slots[1], j // 16], :, j % 16]).copy()
        row[0, 5], row[1, D - 1] = ref.rounded(np.array([x, -x]), dtype)
        s.p.put(s.p.v, 1, [j], [row])
    got = s.run()
    s.check(got)
    seen = np.array(s.masks[rows:])
    assert np.isinf(got[0][rows:][seen[:, 1] & ~seen[:, 2] & ~seen[:, rows - 1]][:, 0, 5]).all() and np.isfinite(got[0][rows:][~seen[:, 1] & ~seen[:, 2] & ~seen[:, rows - 1]]).all()
    assert np.isfinite(got[0][:rows]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows", [3, 50])
def test_a_key_that_is_nan_reaches_the_rows_that_see_it(rows, dtype):
    s = Step([(150, rows), (99, rows)], 4, 2, 128, 32, dtype, "tree", seed=12)
    j = 150 - 1
    row = np.asarray(s.p.k[s.p.table[s.p.slots[0], j // 32], :, j % 32]).copy()
    row[1] = ref.rounded(np.full(128, np.nan), dtype)
    s.p.put(s.p.k, 0, [j], [row])
    out, lse, weights = s.run()
    sees = np.array([bool(m[rows - 1]) for m in s.masks[:rows]])
    assert np.array_equal(np.isnan(lse[:rows, 2:]), np.repeat(sees[:, None], 2, 1)) and not np.isnan(lse[:rows, :2]).any() and not np.isnan(lse[rows:]).any()
    assert np.isnan(out[:rows][sees][:, 2:]).all() and not np.isnan(out[:rows][~sees]).any() and not np.isnan(out[rows:]).any()
    assert not np.isnan(weights[s.p.slots[1]]).any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows", [2, 60])
def test_large_scores_and_scales(rows, dtype):
    s = Step([(400, rows)], 4, 2, 128, 64, dtype, "tree", seed=13, std=6.0)
    s.check(s.run(scale=0.3), scale=float(np.float32(0.3)))


@pytest.mark.parametrize("dtype,rows", [("bfloat16", 1), ("float16", 40), ("bfloat16", 40), ("float32", 3)])
def test_keys_behind_max_context_are_not_seen(dtype, rows):
    s = Step([(300, rows), (64, rows)], 4, 2, 128, 16, dtype, "chain", seed=14)
    got = s.run(max_ctx=200)
    s.check(got, max_ctx=200)


@pytest.mark.parametrize("dtype,rows,ps", [("bfloat16", 1, 16), ("float16", 40, 16), ("bfloat16", 40, 8), ("float32", 3, 16), ("bfloat16", 30, 7)])
def test_pages_and_slots_that_do_not_exist(dtype, rows, ps):
    s = Step([(300, rows), (200, rows), (100, rows)], 4, 2, 128, ps, dtype, "chain", seed=15)
    s.p.table = s.p.table.copy()
    s.p.table[s.p.slots[0], 3] = -1
    s.p.table[s.p.slots[1], 5] = s.p.pages
    a = s.arrays()
    slots = s.p.slots.copy()
    slots[2] = -1
    a["slots"] = i32(slots)
    s.call(a)
    out, lse, weights = s.read(a)
    q = ref.floats(s.q, dtype)
    rep, D = s.Hq // s.p.H, s.D
    for seq, gone in ((0, 3), (1, 5)):
        ctx = s.portions[seq][0]
        there = np.arange(ctx) // ps != gone
        k, v = (np.where(there[:, None, None], 0, 1) * 0.0 for _ in range(2))
        table = np.where((s.p.table[s.p.slots[seq]] < 0) | (s.p.table[s.p.slots[seq]] >= s.p.pages), 0, s.p.table[s.p.slots[seq]])
        j = np.arange(ctx)
        k, v = (ref.floats(x[table[j // ps], :, j % ps], dtype) for x in (s.p.k, s.p.v))
        for i in range(rows):
            seen = there & (j <= ctx - rows + i)
            for h in range(s.Hq):
                x = k[seen][:, h // rep] @ q[s.starts[seq] + i, h] / np.sqrt(D)
                w = np.exp(x - x.max())
                want, spread = w @ v[seen][:, h // rep] / w.sum(), w @ np.abs(v[seen][:, h // rep]) / w.sum()
                size = (np.abs(k[seen][:, h // rep]) @ np.abs(q[s.starts[seq] + i, h])).max() / np.sqrt(D)
                tol = ref.bound(want, spread, np.asarray(size), D, ctx, dtype)
                assert (np.abs(out[s.starts[seq] + i, h] - want) <= tol).all()
    assert (out[s.starts[2]:] == 7).all() and (lse[s.starts[2]:] == 7).all()
    assert np.array_equal(weights[s.p.slots[2]], s.weights[s.p.slots[2]])


@pytest.mark.parametrize("dtype,rows", [("bfloat16", 2), ("float16", 40), ("float32", 3)])
def test_rows_that_nobody_has_are_left(dtype, rows):
    s = Step([(100, rows), (90, rows)], 4, 2, 128, 16, dtype, "chain", seed=16)
    a = s.arrays()
    a["starts"] = i32([0, rows, 2 * rows - 1])
    s.portions = [s.portions[0], (89, rows - 1)]
    a["ctx"] = i32([100, 89])
    s.call(a)
    out, lse, _ = s.read(a)
    assert (out[2 * rows - 1:] == 7).all() and (lse[2 * rows - 1:] == 7).all() and (out[:2 * rows - 1] != 7).all()
    a = s.arrays()
    a["starts"] = i32([5, 3, 10 ** 9])                # what no program means: nothing outside the arrays is touched
    s.call(a)
    synchronize()


@pytest.mark.parametrize("dtype,rows", [("bfloat16", 1), ("bfloat16", 40), ("float16", 5), ("float32", 3)])
def test_outputs_over_queries_captured_and_repeated(dtype, rows):
    s = Step([(700, rows), (130, rows)], 8, 2, 128, 64, dtype, "tree" if rows > 1 else "chain", seed=17)
    want = s.run()
    got = s.run()
    assert all(np.array_equal(x, y) for x, y in zip(got, want))
    a = s.arrays()
    a["out"] = a["q"]
    s.call(a, weigh=False)
    assert np.array_equal(s.read(a)[0], want[0])
    sets, streams, graphs = [s.arrays() for _ in range(2)], [Stream() for _ in range(2)], []
    for x, st in zip(sets, streams):
        with use_stream(st):
            s.call(x, weigh=False)
            st.synchronize()
            g = CudaGraph()
            with g.capture(st):
                s.call(x)
            graphs.append(g)
    for _ in range(3):
        for x in sets:
            x["weights"].copy_from_numpy(s.weights)
        synchronize()
        for g, st in zip(graphs, streams):
            g.replay(st)
        for st in streams:
            st.synchronize()
        for x in sets:
            assert all(np.array_equal(u, v) for u, v in zip(s.read(x), want))


def test_a_fixed_cache_is_one_page():
    s = Step([(900, 5)], 8, 2, 128, 1000, "bfloat16", "tree", seed=18)
    s.check(s.run())


def test_offsets_past_32_bits():
    """a cache of 4.8 GB: rows at its end"""
    rng = np.random.default_rng(19)
    H, D, ps = 8, 128, 64
    pages = 36900
    k = ops_zeros((pages, H, ps, D))
    v = ops_zeros((pages, H, ps, D))
    table = np.array([[pages - 1, 3, pages - 2]], np.int32)
    rows = ref.rounded(rng.standard_normal((2, 3, H, ps, D)), "bfloat16")
    for a, x in ((k, rows[0]), (v, rows[1])):
        for i, p in enumerate(table[0]):
            a._view(int(p) * H * ps * D, (H, ps, D)).copy_from_numpy(x[i])
    small = Step([(150, 1)], 16, H, D, ps, "bfloat16", seed=20)
    for a, x in ((small.p.k, rows[0]), (small.p.v, rows[1])):
        for i in range(3):
            a[small.p.table[small.p.slots[0], i]] = x[i]
    for n in (1, 40):
        s = Step([(150, n)], 16, H, D, ps, "bfloat16", seed=20)
        s.p = small.p
        arrays = s.arrays()
        arrays.update(k=k, v=v, table=from_numpy(table), slots=i32([0]))
        arrays["weights"] = from_numpy(np.zeros((1, H, 192), np.float32))
        s.call(arrays)
        big = s.read(arrays)
        ours = s.run()
        assert np.array_equal(big[0], ours[0]) and np.array_equal(big[1], ours[1])
    # and rows that move there
    ops.move_rows_paged([k, v], from_numpy(table), i32([0]), i32([[5, 100, 149]]), i32([3]))
    got = k._view((pages - 1) * H * ps * D, (H, ps, D)).to_numpy()
    assert np.array_equal(got[:, 0], rows[0][0][:, 5]) and np.array_equal(got[:, 1], rows[0][1][:, 36]) and np.array_equal(got[:, 2], rows[0][2][:, 21])


def ops_zeros(shape):
    from pygpukit_b200.core.factory import zeros
    return zeros(shape, bfloat16)
