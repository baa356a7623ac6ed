"""Positions that stay, rows of the pages that move, masks of trees and accepted drafts: exactly the oracle's."""
import numpy as np
import pytest

from pygpukit_b200 import ops
from pygpukit_b200.core.dtypes import bfloat16
from pygpukit_b200.core.factory import from_numpy
from pygpukit_b200.core.stream import CudaGraph, Stream, use_stream
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


def i32(x):
    return from_numpy(np.ascontiguousarray(np.asarray(x, np.int32)))


# ---------------------------------------------------------------------------------------------------- what stays
def weights_of(kind, rng, shape):
    if kind == "even":
        return rng.random(shape).astype(np.float32)
    if kind == "heavy":
        return (-np.log(rng.random(shape)) ** 3).astype(np.float32)
    if kind == "equal":
        return np.full(shape, 0.25, np.float32)
    if kind == "steps":
        return (np.floor(rng.random(shape) * 3) / 3).astype(np.float32)
    if kind == "close":                               # differences in the last bits
        return (1.0 + rng.integers(0, 40, shape) * 2.0 ** -23).astype(np.float32)
    x = rng.standard_normal(shape).astype(np.float32)                 # odd ones: signs, zeros of both, infinities, NaN
    x.flat[::7] = np.nan
    x.flat[1::11] = np.inf
    x.flat[2::13] = -np.inf
    x.flat[3::5] = 0.0
    x.flat[4::10] = -0.0
    return x


@pytest.mark.parametrize("kind", ["even", "heavy", "equal", "steps", "close", "odd"])
@pytest.mark.parametrize("contexts,budget,first,recent", [
    ([1, 0, 5], 3, 0, 0), ([5, 3, 4], 4, 1, 3), ([1000, 999, 40], 64, 4, 16), ([2048, 2047, 1025], 1024, 0, 0), ([3001, 70], 65, 64, 1), ([700, 33], 32, 0, 32),
    ([9000, 8191], 4000, 3, 1000), ([130], 129, 0, 5)], ids=str)
def test_select(kind, contexts, budget, first, recent):
    rng = np.random.default_rng(budget)
    S, H = len(contexts), 3
    w = weights_of(kind, rng, (S + 1, H, max(contexts) + 3))
    slots = rng.permutation(S + 1)[:S]
    kept, counts = ops.select_rows(from_numpy(w), i32(slots), i32(contexts), budget, first=first, recent=recent)
    want, n = ref.select(w, slots, contexts, budget, first, recent)
    assert np.array_equal(counts.to_numpy(), n)
    assert np.array_equal(kept.to_numpy(), want)


def test_select_of_contexts_and_slots_out_of_range():
    w = np.random.default_rng(1).random((2, 2, 50)).astype(np.float32)
    contexts, slots = [-3, 2 ** 31 - 1, 40, 10], [0, 1, 5, -1]
    kept, counts = ops.select_rows(from_numpy(w), i32(slots), i32(contexts), 8, recent=2)
    want, n = ref.select(w, slots, contexts, 8, 0, 2)
    assert np.array_equal(counts.to_numpy(), n) and np.array_equal(kept.to_numpy(), want) and n.tolist() == [0, 8, 0, 0]


# ---------------------------------------------------------------------------------------------------- rows that move
def moved(p, a, kept, counts, starts, by_head):
    """what the pages are afterwards"""
    new = a.copy()
    for s in range(len(counts)):
        for h in range(p.H):
            src = kept[s, h] if by_head else kept[s]
            for i in range(min(counts[s], len(src))):
                f, t = starts[s] + src[i], starts[s] + i
                if src[i] <= i or not 0 <= f < p.positions or not 0 <= t < p.positions:
                    continue
                pf, pt = p.table[p.slots[s], f // p.ps], p.table[p.slots[s], t // p.ps]
                if 0 <= pf < p.pages and 0 <= pt < p.pages:
                    new[pt, h, t % p.ps] = a[pf, h, f % p.ps]
    return new


MOVES = [  # contexts, heads, D, page, type, rows kept
    ([50, 3], 2, 128, 16, "bfloat16", 30), ([4000], 2, 128, 64, "bfloat16", 3000), ([700, 650, 20], 3, 8, 7, "float16", 300), ([333], 1, 256, 64, "float32", 332),
    ([2000, 1999], 4, 66, 100, "bfloat16", 900), ([100], 5, 1, 10, "bfloat16", 60), ([6000], 1, 64, 64, "float32", 5999),
]


@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("contexts,H,D,ps,dtype,m", MOVES, ids=str)
def test_rows_move_in_place(contexts, H, D, ps, dtype, m, by_head):
    rng = np.random.default_rng(D + m)
    p = ref.Pages(rng, contexts, H, D, ps, dtype)
    S = len(contexts)
    kept = np.full((S, H, m) if by_head else (S, m), -1, np.int32)
    counts = np.array([min(m, c) for c in contexts], np.int32)
    for s, c in enumerate(contexts):
        for h in range(H if by_head else 1):
            row = np.sort(rng.permutation(c)[:counts[s]])
            if by_head:
                kept[s, h, :counts[s]] = row
            else:
                kept[s, :counts[s]] = row
    extra = ref.rounded(rng.standard_normal((p.pages, H, ps, 3 * D)), dtype)          # rows of another size
    arrays = [from_numpy(p.k), from_numpy(p.v), from_numpy(extra)]
    weights = rng.random((p.n_slots, H, p.positions + 1)).astype(np.float32)
    wd = from_numpy(weights)
    ops.move_rows_paged(arrays, from_numpy(p.table), i32(p.slots), i32(kept), i32(counts), weights=wd, context_lens=i32(contexts))
    for a, x in zip(arrays, (p.k, p.v, extra)):
        assert a.to_numpy().tobytes() == moved(p, x, kept, counts, [0] * S, by_head).tobytes()
    want = weights.copy()
    for s, c in enumerate(contexts):
        for h in range(H):
            row = (kept[s, h] if by_head else kept[s])[:counts[s]]
            want[p.slots[s], h, :counts[s]] = weights[p.slots[s], h, row]
            want[p.slots[s], h, counts[s]:c] = 0.0
    assert np.array_equal(wd.to_numpy(), want)


def test_rows_that_move_behind_a_start_and_many_arrays():
    rng = np.random.default_rng(3)
    contexts, starts = [90, 200, 64], [70, 150, 64]
    p = ref.Pages(rng, contexts, 2, 64, 16, "bfloat16")
    kept = np.array([[0, 1, 5, 19, -1], [3, 4, 40, 49, 7], [0, 0, 0, 0, 0]], np.int32)           # the last entry lies behind its count
    counts = np.array([4, 4, 0], np.int32)
    base = [ref.rounded(rng.standard_normal(p.k.shape), "bfloat16") for _ in range(3)]
    arrays = [from_numpy(base[i % 3]) for i in range(150)]
    ops.move_rows_paged(arrays, from_numpy(p.table), i32(p.slots), i32(kept), i32(counts), starts=i32(starts))
    want = [moved(p, x, kept, counts, starts, False) for x in base]
    for i, a in enumerate(arrays):
        assert np.array_equal(a.to_numpy(), want[i % 3])


def test_entries_that_move_nothing():
    """in their place, before it, outside the pages, on pages that do not exist, slots without a sequence; the same source twice"""
    rng = np.random.default_rng(4)
    p = ref.Pages(rng, [60, 60, 60], 2, 32, 16, "float32")
    p.table = p.table.copy()
    p.table[p.slots[1], 2] = -1
    kept = np.array([[0, 0, 9, 9, 10 ** 6, 2 ** 31 - 1, -4, 50], [40, 41, 42, 50, 5, 6, 7, 8], [8, 9, 10, 11, 12, 13, 14, 15]], np.int32)
    counts = np.array([8, 8, 100], np.int32)
    slots = p.slots.copy()
    arrays = [from_numpy(p.k)]
    want = moved(p, p.k, kept, counts, [0, 0, 0], False)
    slots[2] = -1
    undone = p.table[p.slots[2]]
    want[undone] = p.k[undone]
    ops.move_rows_paged(arrays, from_numpy(p.table), i32(slots), i32(kept), i32(counts))
    assert arrays[0].to_numpy().tobytes() == want.tobytes()


# ---------------------------------------------------------------------------------------------------- trees
@pytest.mark.parametrize("sizes", [[1], [8, 1, 3], [64, 33, 32, 31, 0, 65], [300], [1024, 5]], ids=str)
@pytest.mark.parametrize("deep", [False, True])
def test_masks_of_trees(sizes, deep):
    rng = np.random.default_rng(sum(sizes))
    trees = [ref.tree(rng, n, deep) if n else [] for n in sizes]
    starts = np.concatenate([[0], np.cumsum(sizes)])
    parents = [x for t in trees for x in t]
    parents[0] = 10 ** 9                               # no row: a root
    masks, depths = ops.tree_masks(i32(parents), i32(starts), max(sizes))
    rows = [row for t in trees for row in ref.ancestors(t)]
    W = -(-max(sizes) // 32)
    assert np.array_equal(masks.to_numpy(), ref.words(rows, W))
    assert np.array_equal(depths.to_numpy(), [int(r.sum()) - 1 for r in rows])


def test_masks_of_parents_that_are_none_and_rows_behind():
    masks, depths = from_numpy(np.full((7, 2), 9, np.int32)), from_numpy(np.full(7, 9, np.int32))
    ops.tree_masks(i32([0, 3, 1, 2, -7, 0, 0]), i32([0, 4, 6]), 3, masks=masks, depths=depths)
    # row 0 hangs on itself and row 1 on a row behind it: roots; row 3 is past max_rows
    assert masks.to_numpy().tolist() == [[1, 0], [2, 0], [6, 0], [9, 9], [1, 0], [3, 0], [9, 9]]
    assert depths.to_numpy().tolist() == [0, 0, 1, 9, 0, 1, 9]


@pytest.mark.parametrize("dtype,V", [("bfloat16", 1000), ("float16", 4099), ("float32", 151936), ("bfloat16", 128256), ("float32", 3), ("bfloat16", 1)])
@pytest.mark.parametrize("sizes", [[1], [26], [13, 0, 64, 5], [40] * 12], ids=str)
def test_accepted_drafts(sizes, dtype, V):
    rng = np.random.default_rng(V + sum(sizes))
    starts = np.concatenate([[0], np.cumsum(sizes)])
    T = int(starts[-1])
    parents = [x for n in sizes for x in (ref.tree(rng, n) if n else [])]
    tokens = rng.integers(0, V, T)
    x = rng.standard_normal((T, V)) * 2
    for s in range(len(sizes)):
        for i in range(starts[s], starts[s + 1]):
            if parents[i] >= 0 and rng.random() < 0.8:
                x[starts[s] + parents[i], tokens[i]] = 9.0                     # of equal ones the lowest
    logits = ref.rounded(x, dtype)
    chosen = ref.floats(logits, dtype).argmax(1)
    got = ops.accept_tree(from_numpy(logits), i32(tokens), i32(parents), i32(starts), max(sizes))
    want = ref.accept(chosen, tokens, parents, starts, max(sizes))
    for a, b in zip(got, want):
        assert np.array_equal(a.to_numpy(), b)
    got = ops.accept_tree(i32(chosen), i32(tokens), i32(parents), i32(starts), max(sizes))
    for a, b in zip(got, want):
        assert np.array_equal(a.to_numpy(), b)


def test_choices_among_odd_logits():
    inf, nan = np.inf, np.nan
    x = np.array([[nan, 1, 5, 5], [nan, nan, nan, nan], [-inf, -inf, -inf, -inf], [-inf, inf, inf, nan], [-0.0, 0.0, -1, -2], [nan, -inf, -inf, -3e38]], np.float32)
    T = len(x)
    got = ops.accept_tree(from_numpy(x), i32([0] * T), i32([-1] * T), i32(np.arange(T + 1)), 1)
    assert got[2].to_numpy().tolist() == [2, 0, 0, 1, 0, 3]
    wide = np.full((T, 4096), -inf, np.float32)
    wide[:, 4000:4004] = x
    got = ops.accept_tree(from_numpy(wide), i32([0] * T), i32([-1] * T), i32(np.arange(T + 1)), 1)
    assert got[2].to_numpy().tolist() == [4002, 0, 0, 4001, 4000, 4003]


def test_twins_and_bounds():
    # two children with the chosen token: the lower one; a row that hangs on one behind it is nobody's child; starts that leave the arrays
    tokens, parents, chosen = [7, 5, 5, 6, 5], [-1, 0, 0, 2, 9], [5, 6, 6, 1, 1]
    rows, counts, nxt = ops.accept_tree(i32(chosen), i32(tokens), i32(parents), i32([0, 5]), 8)
    assert rows.to_numpy().tolist() == [[0, 1, -1, -1, -1, -1, -1, -1]] and counts.to_numpy().tolist() == [2] and nxt.to_numpy().tolist() == [6]
    rows, counts, nxt = ops.accept_tree(i32(chosen), i32(tokens), i32(parents), i32([-1, 3, 10 ** 9, 2]), 4)
    assert counts.to_numpy().tolist() == [0, 0, 0] and nxt.to_numpy().tolist() == [-1, -1, -1] and (rows.to_numpy() == -1).all()


def test_captured_side_by_side():
    rng = np.random.default_rng(8)
    n, V = 20, 50000
    parents, tokens = ref.tree(rng, n), rng.integers(0, V, n)
    streams, graphs, outs, wants = [Stream() for _ in range(2)], [], [], []
    keep = []
    for k, st in enumerate(streams):
        x = rng.standard_normal((n, V)).astype(np.float32)
        for i in range(1, n):
            if (i + k) % 2:
                x[parents[i], tokens[i]] = 20.0
        wants.append(ref.accept(x.argmax(1), tokens, parents, [0, n], n))
        with use_stream(st):
            a = [from_numpy(x), i32(tokens), i32(parents), i32([0, n])]
            out = (i32(np.zeros((1, n))), i32([0]), i32([0]))
            ops.accept_tree(*a, n, out=out)
            st.synchronize()
            g = CudaGraph()
            with g.capture(st):
                ops.accept_tree(*a, n, out=out)
        keep.append(a)
        graphs.append(g)
        outs.append(out)
    for _ in range(4):
        for g, st in zip(graphs, streams):
            g.replay(st)
    for st in streams:
        st.synchronize()
    for out, want in zip(outs, wants):
        for a, b in zip(out, want):
            assert np.array_equal(a.to_numpy(), b)


def test_a_step_from_drafts_to_the_next():
    """the operators as a program uses them: masks, attention, acceptance, rows that move -- then a plain decoded token sees what a cache without drafts holds"""
    rng = np.random.default_rng(21)
    H, Hq, D, ps, ctx0, n = 2, 8, 128, 16, 75, 12
    p = ref.Pages(rng, [ctx0 + n + 1], H, D, ps, "bfloat16")
    parents = ref.tree(rng, n)
    path = [0]
    while True:
        kids = [j for j in range(n) if parents[j] == path[-1]]
        if not kids:
            break
        path.append(kids[-1])
    tokens = np.arange(n) + 100
    chosen = np.zeros(n, np.int32)
    for a, b in zip(path, path[1:]):
        chosen[a] = tokens[b]
    chosen[path[-1]] = 3
    q = ref.rounded(rng.standard_normal((n, Hq, D)), "bfloat16")
    kd, vd, td, sd = from_numpy(p.k), from_numpy(p.v), from_numpy(p.table), i32(p.slots)
    starts, parents_d = i32([0, n]), i32(parents)
    masks, depths = ops.tree_masks(parents_d, starts, n)
    out = from_numpy(np.zeros_like(q))
    ops.sdpa_paged(from_numpy(q), kd, vd, out, td, sd, i32([ctx0 + n]), ctx0 + n, row_starts=starts, max_rows=n, masks=masks)
    rows, counts, nxt = ops.accept_tree(i32(chosen), i32(tokens), parents_d, starts, n)
    assert rows.to_numpy()[0, :len(path)].tolist() == path and counts.to_numpy().tolist() == [len(path)] and nxt.to_numpy().tolist() == [3]
    ops.move_rows_paged([kd, vd], td, sd, rows, counts, starts=i32([ctx0]))
    # the next token behind the accepted ones
    m = ctx0 + len(path)
    one = ref.rounded(rng.standard_normal((1, Hq, D)), "bfloat16")
    o2 = from_numpy(np.zeros_like(one))
    ops.sdpa_paged(from_numpy(one), kd, vd, o2, td, sd, i32([m]), m)
    k, v = (p.rows(a, 0, ctx0 + n) for a in (p.k, p.v))
    at = list(range(ctx0)) + [ctx0 + j for j in path]
    x = np.einsum("hd,jhd->hj", ref.floats(one, "bfloat16")[0], np.repeat(k[at], Hq // H, 1)) / np.sqrt(D)
    w = np.exp(x - x.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    want = np.einsum("hj,jhd->hd", w, np.repeat(v[at], Hq // H, 1))
    spread = np.einsum("hj,jhd->hd", w, np.abs(np.repeat(v[at], Hq // H, 1)))
    size = np.einsum("hd,jhd->hj", np.abs(ref.floats(one, "bfloat16")[0]), np.abs(np.repeat(k[at], Hq // H, 1))).max(1) / np.sqrt(D)
    assert (np.abs(ref.floats(o2.to_numpy(), "bfloat16")[0] - want) <= ref.bound(want, spread, size, D, m, "bfloat16")).all()
    _ = bfloat16, depths
