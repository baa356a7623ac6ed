"""Sizes that the 32-bit counts of the operators on pages and on trees do not hold are refused, not taken for other ones.  No GPU."""
import ctypes as C

import pytest

from pygpukit_b200 import _lib, ops
from pygpukit_b200.core.dtypes import bfloat16, float16, float32, int32
from tests.test_paged_rows_cpu import arr, attend, move


@pytest.mark.parametrize("kw", [
    dict(k_cache=arr((2 ** 32 + 9, 2, 16, 128), bfloat16), v_cache=arr((2 ** 32 + 9, 2, 16, 128), bfloat16)),
    dict(page_table=arr((3, 2 ** 32 + 4), int32)), dict(page_table=arr((2 ** 32 + 3, 4), int32)), dict(page_table=arr((3, 2 ** 28), int32)),
    dict(Q=arr((2 ** 32 + 5, 8, 128), bfloat16), out=arr((2 ** 32 + 5, 8, 128), bfloat16), row_starts=arr((6,), int32), max_rows=2)], ids=str)
def test_attention(kw):
    with pytest.raises(ValueError, match="sdpa_paged"):
        attend(**kw)


@pytest.mark.parametrize("shape", [(3, 2, 2 ** 31 - 2 ** 15), (3, 2, 2 ** 32 + 64), (2 ** 32 + 3, 2, 64)], ids=str)
def test_selection(shape):
    with pytest.raises(ValueError, match="select_rows"):
        ops.select_rows(arr(shape), arr((2,), int32), arr((2,), int32), 8, out=(arr((2, 2, 8), int32), arr((2,), int32)))


@pytest.mark.parametrize("kw", [dict(rows=arr((5, 2 ** 32 + 7), int32)), dict(rows=arr((5, 2, 2 ** 31 - 2 ** 15), int32)), dict(page_table=arr((3, 2 ** 31), int32)),
                                dict(arrays=[arr((2 ** 32 + 9, 2, 16, 128), float16)])], ids=str)
def test_moving(kw):
    with pytest.raises(ValueError, match="move_rows_paged"):
        move(**kw)


def test_trees():
    with pytest.raises(ValueError, match="tree_masks"):
        ops.tree_masks(arr((9,), int32), arr((3,), int32), 5, masks=arr((9, 2 ** 18 + 1), int32), depths=arr((9,), int32))
    with pytest.raises(ValueError, match="tree_masks"):
        ops.tree_masks(arr((2 ** 32 + 9,), int32), arr((3,), int32), 5, masks=arr((2 ** 32 + 9, 1), int32), depths=arr((2 ** 32 + 9,), int32))
    for vocab in (2 ** 31 - 2 ** 15, 2 ** 32 + 100):
        with pytest.raises(ValueError, match="accept_tree"):
            ops.accept_tree(arr((9, vocab), float32), arr((9,), int32), arr((9,), int32), arr((3,), int32), 5, out=(arr((2, 5), int32), arr((2,), int32), arr((2,), int32)))


def test_the_library_refuses_them_too():
    lib, p = _lib.load(), C.c_void_p(1 << 20)
    assert lib.pgk_select_rows(p, 2 ** 31, p, p, 2, 3, 2, 2 ** 31 - 2 ** 15, 8, 0, 0, p, p, None) != 0 and "select_rows failed" in _lib.last_error()
    one, size = (C.c_uint64 * 1)(1 << 20), (C.c_int32 * 1)(256)
    assert lib.pgk_move_rows(one, size, 1, p, 9, 16, 3, 4, 2, p, None, p, p, 5, 2 ** 31 - 2 ** 15, 0, None, 0, None, None) != 0 and "move_rows failed" in _lib.last_error()
    assert lib.pgk_tree_masks(p, p, 2, 9, 5, 2 ** 18 + 1, p, p, None) != 0 and "tree_masks failed" in _lib.last_error()
    assert lib.pgk_accept_tree(p, 2 ** 31, 2, 2 ** 31 - 2 ** 15, None, p, p, p, 2, 9, 5, p, p, p, None) != 0 and "accept_tree failed" in _lib.last_error()
