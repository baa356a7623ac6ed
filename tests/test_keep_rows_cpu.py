"""`PagedKVCache.keep_rows` over shared pages: which pages are copied, and what a failure leaves.  The device is a host array behind fakes: no GPU."""
import numpy as np
import pytest

from pygpukit_b200 import llm
from pygpukit_b200.llm import paged_cache


class Array:
    """an array whose rows are integers, [pages, heads, page size, 1]; its address is its own number"""
    made: list = []

    def __init__(self, shape, dtype=None):
        self.shape, self.dtype, self.data = tuple(shape), dtype, np.zeros(shape, np.int64)
        Array.made.append(self)
        self.device_ptr = len(Array.made)

    @property
    def size(self):
        return self.data.size

    @property
    def nbytes(self):
        return self.data.nbytes

    def view(self, shape):
        return self

    def _view(self, at, shape):
        n = int(np.prod(shape))
        return self.data.reshape(-1)[at:at + n].reshape(shape)


class Api:
    room = 10 ** 9

    def upload(self, to, host, nbytes, stream):
        pass

    def memcpy_d2d(self, to, src, nbytes, stream):
        a, b = Array.made[to - 1].data, Array.made[src - 1].data
        a.reshape(-1)[:b.size] = b.reshape(-1)

    def device_sync(self):
        pass


@pytest.fixture
def cache(monkeypatch):
    Array.made.clear()
    fake = Api()

    def zeros(shape, dtype):
        if int(np.prod(shape)) > fake.room:
            raise RuntimeError("out of memory")
        return Array(shape, dtype)
    copied = []

    def copy(self, arrays, pairs):
        copied.extend(pairs)
        for a in arrays:
            for src, dst in pairs:
                a.data[dst] = a.data[src]

    def move(arrays, table, slots, rows, counts, starts=None):
        """in place, row by row, as the sequences' tables say"""
        for seq, start, kept in c._moving:
            pages, ps = c.pool.page_list(seq), c.page_size
            assert list(c.pool.table[c.pool.slot(seq), :len(pages)]) == pages
            for i, r in enumerate(kept):
                for a in arrays:
                    a.data[pages[(start + i) // ps], :, (start + i) % ps] = a.data[pages[(start + r) // ps], :, (start + r) % ps]
    monkeypatch.setattr(paged_cache, "api", fake)
    monkeypatch.setattr(paged_cache, "zeros", zeros)
    monkeypatch.setattr(paged_cache, "GPUArray", Array)
    monkeypatch.setattr(paged_cache, "move_rows_paged", move)
    monkeypatch.setattr(paged_cache.PagedKVCache, "_copy", copy)
    c = llm.PagedKVCache([(2, 1, 1)], "bfloat16", page_size=4, tokens_hint=64, slots=4)
    c.copied, c.fake = copied, fake
    return c


def fill(c, seq, n):
    c.extend(seq, n)
    for j, page in ((j, c.pool.page_list(seq)[j // 4]) for j in range(n)):
        for a in c._page_arrays():
            a.data[page, :, j % 4] = 1000 * (ord(seq) - ord("a") + 1) + j


def rows(c, seq):
    pages = c.pool.page_list(seq)
    return [int(c.k[0].data[pages[j // 4], 0, j % 4, 0]) for j in range(c.pool.length(seq))]


def keep(c, keeps):
    c._moving = [(s, a, r) for s, (a, r) in keeps.items()]
    c.copied.clear()
    c.keep_rows(keeps)


def test_pages_that_no_row_moves_into_stay_shared(cache):
    fill(cache, "a", 40)
    cache.assign({"b": "a"})
    was, free = cache.pool.page_list("a"), cache.pool.free_pages
    kept = [0, 1, 2, 3, 4, 6, 9, 30, 31]               # the first that moves goes to position 5, the last to 8
    keep(cache, {"a": (0, kept)})
    assert cache.copied == [(was[1], cache.pool.page_list("a")[1]), (was[2], cache.pool.page_list("a")[2])]
    assert cache.pool.page_list("a")[0] == was[0] and cache.pool.free_pages == free - 2
    assert rows(cache, "a") == [1000 + j for j in kept] and rows(cache, "b") == [1000 + j for j in range(40)]
    keep(cache, {"b": (2, list(range(30)))})           # nothing moves: nothing is copied
    assert cache.copied == [] and cache.pool.length("b") == 32 and rows(cache, "b") == [1000 + j for j in range(32)]


def test_sequences_that_share_pages_and_move_together(cache):
    fill(cache, "a", 32)
    cache.assign({"b": "a", "c": "a"})
    keep(cache, {"a": (4, [1, 2, 3, 20, 27]), "b": (8, [2, 5]), "c": (0, [0, 1, 2, 3, 4, 31])})
    assert rows(cache, "a") == [1000 + j for j in (0, 1, 2, 3, 5, 6, 7, 24, 31)]
    assert rows(cache, "b") == [1000 + j for j in (0, 1, 2, 3, 4, 5, 6, 7, 10, 13)]
    assert rows(cache, "c") == [1000 + j for j in (0, 1, 2, 3, 4, 31)]
    for s in ("a", "b", "c"):
        cache.release(s)
    assert cache.pool.free_pages == cache.pool.pages and not cache.pool._shared


def test_the_last_holder_of_a_page_keeps_it(cache):
    fill(cache, "a", 8)
    cache.assign({"b": "a"})
    keep(cache, {"a": (0, [1]), "b": (0, [2])})
    assert len(cache.copied) == 1 and rows(cache, "a") == [1001] and rows(cache, "b") == [1002]


def test_growth_that_fails_leaves_the_sequences(cache):
    fill(cache, "a", 60)
    fill(cache, "b", 8)
    cache.assign({"c": "a"})
    for i, n in enumerate((4, 4)):
        cache.extend(("x", i), n)
    while cache.pool.free_pages:
        cache.extend(("y", cache.pool.free_pages), 4)
    before = {s: (cache.pool.page_list(s), rows(cache, s)) for s in ("a", "b", "c")}
    table, shared = cache.pool.table.copy(), dict(cache.pool._shared)
    cache.fake.room = cache.k[0].size
    with pytest.raises(RuntimeError, match="out of memory"):
        keep(cache, {"b": (0, [0, 3]), "a": (0, [1, 2, 30])})
    assert {s: (cache.pool.page_list(s), rows(cache, s)) for s in ("a", "b", "c")} == before
    assert np.array_equal(cache.pool.table, table) and cache.pool._shared == shared and cache.copied == []
    cache.fake.room = 10 ** 9                          # and with room again it works
    keep(cache, {"b": (0, [0, 3]), "a": (0, [1, 2, 30])})
    assert rows(cache, "a") == [1001, 1002, 1030] and rows(cache, "b") == [2000, 2003] and rows(cache, "c") == before["c"][1]


def test_plans_are_taken_at_once():
    pool = llm.PagePool(4, 8, 4, 8)
    pool.extend("a", 8)
    pool.assign({"b": "a"})
    plan = pool.plan_pages([("a", 0, 8)])
    assert len(plan) == 2 and len(pool.pairs_of(plan)) == 2 and pool.page_list("a") == pool.page_list("b")
    pool.extend("c", 1)
    with pytest.raises(RuntimeError, match="planned"):
        pool.take_pages(plan)
