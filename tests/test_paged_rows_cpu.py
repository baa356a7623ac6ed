"""What the operators on 16- and 32-bit pages and on trees of drafts refuse, their C entries' checks, and the pool's bookkeeping: no GPU."""
import ctypes as C

import numpy as np
import pytest

from pygpukit_b200 import _lib, llm, ops
from pygpukit_b200.core.array import GPUArray
from pygpukit_b200.core.dtypes import bfloat16, float16, float32, int32, int64, uint8
from pygpukit_b200.llm.decode.tree import tree_size
from tests import paged_ref as ref


def arr(shape, dtype=float32):
    """an array that no call gets to read"""
    return GPUArray(shape, dtype, ptr=1 << 20)


def attend(**kw):
    a = dict(Q=arr((5, 8, 128), bfloat16), k_cache=arr((9, 2, 16, 128), bfloat16), v_cache=arr((9, 2, 16, 128), bfloat16), out=arr((5, 8, 128), bfloat16),
             page_table=arr((3, 4), int32), slots=arr((5,), int32), context_lens=arr((5,), int32), max_context=64)
    a.update(kw)
    ops.sdpa_paged(**a)


STEP = [
    dict(Q=arr((5, 1024), bfloat16)), dict(Q=arr((5, 7, 128), bfloat16)), dict(Q=arr((5, 8, 64), bfloat16)), dict(Q=arr((5, 8, 128), uint8)), dict(Q=arr((5, 8, 128), float16)),
    dict(k_cache=arr((9, 2, 16), bfloat16)), dict(k_cache=arr((0, 2, 16, 128), bfloat16)), dict(page_table=arr((12,), int32)), dict(page_table=arr((3, 4), int64)),
    dict(page_table=arr((3, 0), int32)), dict(slots=arr((4,), int32)), dict(slots=arr((5, 1), int32)), dict(slots=arr((5,), int64)), dict(context_lens=arr((4,), int32)),
    dict(max_context=-1), dict(max_context=65), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-40), dict(max_rows=2),
    dict(row_starts=arr((5,), int32)), dict(row_starts=arr((6,), int32), max_rows=0), dict(masks=arr((5,), int32)), dict(masks=arr((4, 1), int32)),
    dict(masks=arr((5, 0), int32)), dict(masks=arr((5, 1), int64)),
]


@pytest.mark.parametrize("bad", STEP + [
    dict(v_cache=arr((9, 2, 16, 64), bfloat16)), dict(v_cache=arr((9, 2, 16, 128), float16)), dict(out=arr((5, 8, 128), float32)), dict(out=arr((4, 8, 128), bfloat16)),
    dict(lse=arr((5, 7))), dict(lse=arr((5, 8), bfloat16)),
    dict(Q=arr((5, 8, 12), bfloat16), out=arr((5, 8, 12), bfloat16), k_cache=arr((9, 2, 16, 12), bfloat16), v_cache=arr((9, 2, 16, 12), bfloat16)),
    dict(Q=arr((5, 8, 264), bfloat16), out=arr((5, 8, 264), bfloat16), k_cache=arr((9, 2, 16, 264), bfloat16), v_cache=arr((9, 2, 16, 264), bfloat16)),
], ids=str)
def test_attention_refuses(bad):
    with pytest.raises(ValueError, match="sdpa_paged"):
        attend(**bad)


@pytest.mark.parametrize("bad", STEP + [dict(lse=arr((5, 7))), dict(lse=arr((5, 8), bfloat16)), dict(weights=arr((3, 2, 63))), dict(weights=arr((2, 2, 64))),
                                        dict(weights=arr((3, 4, 64))), dict(weights=arr((3, 2, 64), bfloat16)), dict(weights=arr((3, 128)))], ids=str)
def test_weights_refuse(bad):
    a = dict(Q=arr((5, 8, 128), bfloat16), k_cache=arr((9, 2, 16, 128), bfloat16), lse=arr((5, 8)), weights=arr((3, 2, 64)), page_table=arr((3, 4), int32),
             slots=arr((5,), int32), context_lens=arr((5,), int32), max_context=64)
    a.update(bad)
    with pytest.raises(ValueError, match="weigh_paged"):
        ops.weigh_paged(**a)


@pytest.mark.parametrize("bad", [dict(weights=arr((3, 2))), dict(weights=arr((3, 2, 64), bfloat16)), dict(weights=arr((3, 2, 0))), dict(slots=arr((2, 1), int32)), dict(slots=arr((2,), int64)),
                                 dict(context_lens=arr((3,), int32)), dict(budget=0), dict(budget=7, first=4, recent=4), dict(first=-1), dict(recent=-1), dict(budget=2 ** 31),
                                 dict(out=(arr((2, 2, 7), int32), arr((2,), int32))), dict(out=(arr((2, 2, 8), int64), arr((2,), int32))),
                                 dict(out=(arr((2, 2, 8), int32), arr((3,), int32)))], ids=str)
def test_selection_refuses(bad):
    a = dict(weights=arr((3, 2, 64)), slots=arr((2,), int32), context_lens=arr((2,), int32), budget=8, out=(arr((2, 2, 8), int32), arr((2,), int32)))
    a.update(bad)
    with pytest.raises(ValueError, match="select_rows"):
        ops.select_rows(**a)


def move(**kw):
    a = dict(arrays=[arr((9, 2, 16, 128), bfloat16), GPUArray((9, 2, 16, 64), float32, ptr=1 << 24)], page_table=arr((3, 4), int32), slots=arr((5,), int32), rows=arr((5, 7), int32),
             counts=arr((5,), int32))
    a.update(kw)
    ops.move_rows_paged(**a)


@pytest.mark.parametrize("bad", [
    dict(arrays=[]), dict(arrays=[arr((9, 2, 128), bfloat16)]), dict(arrays=[arr((9, 2, 16, 72), uint8)]), dict(arrays=[arr((9, 2, 16, 128), bfloat16)] * 2),
    dict(arrays=[arr((9, 2, 16, 128), bfloat16), GPUArray((9, 3, 16, 128), bfloat16, ptr=1 << 24)]), dict(arrays=[arr((9, 2, 16, 2056), bfloat16)]),
    dict(arrays=[arr((9, 501, 16, 8), bfloat16)], rows=arr((5, 501, 7), int32)), dict(page_table=arr((3,), int32)), dict(slots=arr((5, 1), int32)), dict(counts=arr((4,), int32)),
    dict(rows=arr((4, 7), int32)), dict(rows=arr((5, 3, 7), int32)), dict(rows=arr((5,), int32)), dict(rows=arr((5, 7), int64)), dict(starts=arr((4,), int32)),
    dict(weights=arr((3, 2, 64))), dict(weights=arr((3, 3, 64)), context_lens=arr((5,), int32)), dict(weights=arr((3, 2, 64)), context_lens=arr((4,), int32)),
    dict(weights=arr((3, 2, 64), bfloat16), context_lens=arr((5,), int32)),
], ids=str)
def test_moving_refuses(bad):
    with pytest.raises(ValueError, match="move_rows_paged"):
        move(**bad)


@pytest.mark.parametrize("bad", [dict(parents=arr((9, 1), int32)), dict(parents=arr((9,), int64)), dict(row_starts=arr((0,), int32)), dict(row_starts=arr((3,), int64)), dict(max_rows=0),
                                 dict(max_rows=4097), dict(masks=arr((9, 1), int32), max_rows=33), dict(masks=arr((8, 1), int32)), dict(masks=arr((9, 1), int64)), dict(depths=arr((8,), int32))], ids=str)
def test_masks_refuse(bad):
    a = dict(parents=arr((9,), int32), row_starts=arr((3,), int32), max_rows=5, masks=arr((9, 1), int32), depths=arr((9,), int32))
    a.update(bad)
    with pytest.raises(ValueError, match="tree_masks"):
        ops.tree_masks(**a)


@pytest.mark.parametrize("bad", [dict(logits=arr((9,), bfloat16)), dict(logits=arr((8, 100), bfloat16)), dict(logits=arr((9, 0), bfloat16)), dict(logits=arr((9, 100), uint8)),
                                 dict(logits=arr((8,), int32)), dict(tokens=arr((8,), int32)), dict(tokens=arr((9,), int64)), dict(max_rows=0), dict(max_rows=5000),
                                 dict(out=(arr((2, 4), int32), arr((2,), int32), arr((2,), int32))), dict(out=(arr((2, 5), int32), arr((3,), int32), arr((2,), int32))),
                                 dict(out=(arr((2, 5), int32), arr((2,), int32), arr((2,), int64)))], ids=str)
def test_acceptance_refuses(bad):
    a = dict(logits=arr((9, 100), bfloat16), tokens=arr((9,), int32), parents=arr((9,), int32), row_starts=arr((3,), int32), max_rows=5,
             out=(arr((2, 5), int32), arr((2,), int32), arr((2,), int32)))
    a.update(bad)
    with pytest.raises(ValueError, match="accept_tree"):
        ops.accept_tree(**a)


def test_c_entries_check_what_they_get():
    """each call is refused by its own check: nothing is launched"""
    lib = _lib.load()
    p = C.c_void_p(1 << 20)
    odd = C.c_void_p((1 << 20) + 8)

    def attention(q=p, q_ld=1024, k=p, v=p, out=p, o_ld=1024, pages=9, ps=16, table=p, slots=3, mp=4, seq=p, ctx=p, starts=p, seqs=5, tokens=5, rows=2, most=64, heads=8, kv=2, dim=128, scale=0.0, masks=None,
                  words=0, lse=None, dt=2):
        return lib.pgk_paged_attention(q, q_ld, k, v, out, o_ld, pages, ps, table, slots, mp, seq, ctx, starts, seqs, tokens, rows, most, heads, kv, dim, scale, masks, words, lse, dt, None)

    for bad in (dict(dt=3), dict(dim=12), dict(dim=264), dict(dim=0), dict(heads=7), dict(kv=0), dict(pages=0), dict(ps=0), dict(mp=0), dict(q_ld=1000), dict(o_ld=1000), dict(rows=0), dict(seqs=-1),
                dict(starts=None), dict(k=odd), dict(v=odd), dict(q=C.c_void_p((1 << 20) + 1)), dict(out=None), dict(q=None), dict(table=None), dict(scale=-1.0), dict(masks=p, words=0),
                dict(pages=2 ** 30, ps=16), dict(mp=2 ** 28, ps=16), dict(rows=2 ** 24), dict(most=-1), dict(seqs=70000, tokens=70000)):
        assert attention(**bad) != 0, bad
        assert "paged_attention failed" in _lib.last_error(), bad
    assert attention(seqs=0) == 0 and attention(tokens=0) == 0

    def weigh(**kw):
        a = dict(q=p, q_ld=1024, k=p, lse=p, w=p, w_ld=64, pages=9, ps=16, table=p, slots=3, mp=4, seq=p, ctx=p, starts=p, seqs=5, tokens=5, rows=2, most=64, heads=8, kv=2, dim=128, scale=0.0, masks=None,
                 words=0, dt=2)
        a.update(kw)
        return lib.pgk_paged_weigh(*a.values(), None)

    for bad in (dict(w_ld=63), dict(lse=None), dict(w=None), dict(dim=20), dict(dt=-1)):
        assert weigh(**bad) != 0 and "paged_weigh failed" in _lib.last_error(), bad
    for bad in ((p, 64, p, p, 2, 3, 2, 65, 8, 0, 0, p, p), (p, 64, p, p, 2, 3, 2, 64, 0, 0, 0, p, p), (p, 64, p, p, 2, 3, 2, 64, 8, 5, 4, p, p), (None, 64, p, p, 2, 3, 2, 64, 8, 0, 0, p, p)):
        assert lib.pgk_select_rows(*bad, None) != 0 and "select_rows failed" in _lib.last_error(), bad
    one, size = (C.c_uint64 * 1)(1 << 20), (C.c_int32 * 1)(255)
    assert lib.pgk_move_rows(one, size, 1, p, 9, 16, 3, 4, 2, p, None, p, p, 5, 7, 0, None, 0, None, None) != 0 and "move_rows failed" in _lib.last_error()
    size[0] = 4098
    assert lib.pgk_move_rows(one, size, 1, p, 9, 16, 3, 4, 2, p, None, p, p, 5, 7, 0, None, 0, None, None) != 0
    size[0] = 256
    assert lib.pgk_move_rows(one, size, 1, None, 9, 16, 3, 4, 2, p, None, p, p, 5, 7, 0, None, 0, None, None) != 0
    assert lib.pgk_move_rows(one, size, 1, p, 9, 16, 3, 4, 2, p, None, p, p, 5, 7, 0, p, 64, None, None) != 0
    assert lib.pgk_tree_masks(p, p, 2, 9, 33, 1, p, p, None) != 0 and lib.pgk_tree_masks(p, p, 2, 9, 5000, 200, p, p, None) != 0 and lib.pgk_tree_masks(None, p, 2, 9, 5, 1, p, p, None) != 0
    assert lib.pgk_accept_tree(p, 99, 2, 100, None, p, p, p, 2, 9, 5, p, p, p, None) != 0 and lib.pgk_accept_tree(p, 100, 2, 100, None, p, p, p, 2, 70000, 5, p, p, p, None) != 0
    assert lib.pgk_accept_tree(None, 100, 2, 100, None, p, p, p, 2, 9, 5, p, p, p, None) != 0 and "accept_tree failed" in _lib.last_error()


def test_trees_of_drafts_count_their_rows():
    assert [tree_size(b) for b in ((3, 2, 1), (1,), (15,), (2, 2, 2))] == [16, 2, 16, 15]
    for bad in ((), (0,), (2, -1), (1.5,)):
        with pytest.raises(ValueError, match="branches"):
            tree_size(bad)
    s = llm.DecodeTree((3, 2), draft_layers=5)
    assert s.rows == 10 and s.branches == (3, 2) and s.draft_layers == 5
    with pytest.raises(RuntimeError):
        s.step_lookahead(3)
    with pytest.raises(ValueError):
        s.step_tree(3, 4, 4)


def test_pages_of_its_own():
    pool = llm.PagePool(4, 8, 4, 8)
    pool.extend("a", 14)
    pool.assign({"b": "a", "c": "a"})
    was = pool.page_list("a")
    assert pool.page_list("b")[:3] == was[:3]
    pairs = pool.own_pages("b", 6)
    assert [old for old, _ in pairs] == was[1:3] and pool.page_list("b") == [was[0], pairs[0][1], pairs[1][1], pool.page_list("b")[3]]
    assert pool.page_list("c")[:3] == was[:3] and pool.page_list("a") == was and pool.own_pages("b", 4) == []
    assert np.array_equal(pool.table[pool.slot("b"), :4], pool.page_list("b"))
    for s in ("a", "b", "c"):
        pool.release(s)
    assert pool.free_pages == pool.pages
    with pytest.raises(KeyError):
        pool.own_pages("a", 0)


def test_the_oracle():
    parents = [-1, 0, 0, 1, 3, 2]
    m = ref.ancestors(parents)
    assert m.sum(1).tolist() == [1, 2, 2, 3, 4, 3]
    assert ref.words(m, 1)[:, 0].tolist() == [1, 3, 5, 11, 27, 37]
    rows, counts, nxt = ref.accept([4, 5, 9, 6, 7, 1], [3, 4, 4, 5, 6, 9], parents, [0, 6], 6)
    assert rows[0, :4].tolist() == [0, 1, 3, 4] and counts[0] == 4 and nxt[0] == 7
    kept, n = ref.select(np.array([[[0.5, 3, np.nan, 2, 2, 1]]]), [0], [6], 4, 1, 1)
    assert kept[0, 0].tolist() == [0, 1, 3, 5] and n[0] == 4
