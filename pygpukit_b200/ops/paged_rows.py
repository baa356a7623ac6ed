"""Operators on a paged key / value cache of 16 or 32 bits (net-new: the reference's paged attention kernels, native/ops/nn/attention/paged_attention.cuh:46-283,
serve one decoded token a sequence): attention of steps whose rows see each other by masks, the attention weights summed by cached position, the
positions that stay when a cache is cut, and the rows of its pages that move together.

A cache is two arrays, keys and values, `[pages, kv_heads, page_size, dim]` of the queries' type -- `llm.PagedKVCache` makes them, and a fixed cache
`[kv_heads, length, dim]` is one page -- and an int32 page table `[slots, pages of a slot]`.  dim is a multiple of 8 up to 256, pages have any size.

A step: sequence s has the rows row_starts[s] ... row_starts[s + 1] - 1 of the queries (int32 [sequences + 1]; row s without row_starts), the last of its
context_lens[s] positions, whose keys and values are in the pages.  Row i sees every position before the step's and, of the step's rows, those whose bits its
mask has (`tree_masks` makes them; bit j % 32 of word j // 32 for row j), without masks itself and the rows before it.  Rows from max_rows on of a sequence, rows
behind the last sequence and those of a sequence with a negative slot are not computed.

Which rows and positions a call names is data on the device.  Whatever a slot, a position or a page number says, nothing outside the arrays is touched: positions whose
page does not exist, or from max_context on, are not seen.
"""
from __future__ import annotations

from array import array

from .._lib import api
from ..core.array import GPUArray
from ..core.dtypes import float32, float_code, int32, uint8
from ._common import _st
from .paged import _index, _is


MOST_POSITIONS = 2 ** 31 - 2 ** 16          # of a slot's weights or of a list of rows: the kernels count in 32 bits


def _pages(name: str, cache: GPUArray, page_table: GPUArray) -> tuple[int, int, int, int, int, int]:
    """(pages, kv_heads, page size, dim, slots, pages of a slot)"""
    if len(cache._shape) != 4:
        raise ValueError(f"{name}: a cache is [pages, kv_heads, page_size, dim], got {cache.shape}")
    if len(page_table._shape) != 2 or not _is(page_table, int32):
        raise ValueError(f"{name}: page_table must be int32 [slots, max_pages], got {page_table.dtype} {page_table.shape}")
    pages, H, ps, D = cache._shape
    slots, max_pages = page_table._shape
    if min(pages, H, ps, D, slots, max_pages) < 1:
        raise ValueError(f"{name}: a cache without rows, {cache.shape}, or slots, {page_table.shape}")
    if max(pages * H * ps, max_pages * ps, slots) >= 2 ** 31:
        raise ValueError(f"{name}: a cache {cache.shape} behind {page_table.shape} pages (2^31 - 1 rows, and positions of a slot, at most)")
    return pages, H, ps, D, slots, max_pages


def _step(name: str, Q: GPUArray, k_cache: GPUArray, page_table: GPUArray, slots: GPUArray, context_lens: GPUArray, max_context: int, scale: float,
          row_starts: "GPUArray | None", max_rows: int, masks: "GPUArray | None"):
    """what attention and its weights take of a step: (type, heads, arguments)"""
    code = float_code(Q._dtype, name)
    if len(Q._shape) != 3:
        raise ValueError(f"{name} expects Q [tokens, heads, dim], got {Q.shape}")
    T, Hq, D = Q._shape
    pages, H, ps, dim, n_slots, max_pages = _pages(name, k_cache, page_table)
    if T >= 2 ** 31:
        raise ValueError(f"{name}: {T} rows")
    if dim != D or not _is(k_cache, Q._dtype):
        raise ValueError(f"{name}: a cache of {k_cache.dtype} {k_cache.shape} for queries of {Q.dtype} {Q.shape}")
    if D % 8 or D > 256:
        raise ValueError(f"{name}: heads of {D} elements (multiples of 8 up to 256)")
    if Hq < 1 or Hq % H:
        raise ValueError(f"{name}: n_heads {Hq} must be a multiple of KV heads {H}")
    if len(slots._shape) != 1:
        raise ValueError(f"{name}: slots must be int32 [sequences], got {slots.dtype} {slots.shape}")
    S = slots._shape[0]
    _index(name, "slots", slots, S)
    _index(name, "context_lens", context_lens, S)
    if S > 65535:
        raise ValueError(f"{name}: {S} sequences (65535 at most)")
    if row_starts is not None:
        _index(name, "row_starts", row_starts, S + 1)
    elif S != T or max_rows != 1:
        raise ValueError(f"{name}: {S} sequences and {T} rows need row_starts")
    if max_rows < 1 or not 0 <= max_context <= max_pages * ps:
        raise ValueError(f"{name}: max_rows {max_rows}, max_context {max_context} out of range ({max_pages} pages of {ps})")
    if not scale >= 0.0 or (scale and not 1e-37 < scale < 1e38):
        raise ValueError(f"{name}: scale {scale} is not 0 or a number that float32 keeps (1e-37 ... 1e38)")
    words = 0
    if masks is not None:
        if len(masks._shape) != 2 or masks._shape[0] != T or masks._shape[1] < 1 or not _is(masks, int32):
            raise ValueError(f"{name}: masks must be int32 [{T}, words], got {masks.dtype} {masks.shape}")
        words = masks._shape[1]
    args = (pages, ps, page_table._ptr, n_slots, max_pages, slots._ptr, context_lens._ptr, None if row_starts is None else row_starts._ptr, S, T,
            min(max_rows, max(T, 1)), max_context, Hq, H, D, scale, None if masks is None else masks._ptr, words)
    return code, T, Hq, args


def sdpa_paged(Q: GPUArray, k_cache: GPUArray, v_cache: GPUArray, out: GPUArray, page_table: GPUArray, slots: GPUArray, context_lens: GPUArray,
               max_context: int, scale: float = 0.0, *, row_starts: "GPUArray | None" = None, max_rows: int = 1, masks: "GPUArray | None" = None,
               lse: "GPUArray | None" = None) -> None:
    """Attention of many sequences' steps over the cache: decoded tokens, trees of drafted tokens (masks), portions of prompts.  Q, out [tokens, heads, dim].

    scale 0: 1 / sqrt(dim).  lse float32 [tokens, heads]: the natural logarithm of the sum of the scores' exponentials, -infinity for a row that sees nothing,
    whose outputs are zeros.  out may be Q.  Scores, maxima and sums are float32.  An infinite value is the output of the rows that see it, whatever its weight.

    16-bit types: from 33 rows a sequence and key head on (a token's heads of one key head are rows; the longest step of a call decides for all of it), heads of 64 to 128 elements on
    pages of a multiple of 8 positions take tiles whose weights are rounded once, to the cache's type (half a unit of it: in the end 1.4 times the error of the output's own rounding).  Up to 32 rows, and
    for other heads and pages, a weight is two terms of the type, and what is left is the output's rounding."""
    name = "sdpa_paged"
    code, T, Hq, args = _step(name, Q, k_cache, page_table, slots, context_lens, max_context, scale, row_starts, max_rows, masks)
    if v_cache._shape != k_cache._shape or not _is(v_cache, k_cache._dtype):
        raise ValueError(f"{name}: the caches differ: {k_cache.dtype} {k_cache.shape} and {v_cache.dtype} {v_cache.shape}")
    if out._shape != Q._shape or not _is(out, Q._dtype):
        raise ValueError(f"{name}: out must be {Q.dtype} {Q.shape}, got {out.dtype} {out.shape}")
    if lse is not None and (lse._shape != (T, Hq) or not _is(lse, float32)):
        raise ValueError(f"{name}: lse must be float32 [{T}, {Hq}], got {lse.dtype} {lse.shape}")
    ld = Hq * Q._shape[2]
    api.paged_attention(Q._ptr, ld, k_cache._ptr, v_cache._ptr, out._ptr, ld, *args, None if lse is None else lse._ptr, code, _st())


def weigh_paged(Q: GPUArray, k_cache: GPUArray, lse: GPUArray, weights: GPUArray, page_table: GPUArray, slots: GPUArray, context_lens: GPUArray,
                max_context: int, scale: float = 0.0, *, row_starts: "GPUArray | None" = None, max_rows: int = 1, masks: "GPUArray | None" = None) -> None:
    """Add the attention weights of a step to what the positions have: weights float32 [slots, kv_heads, positions] gains, at the sequence's slot, the sum over its
    rows and the query heads of the key head of exp(scale q . k - lse).  lse float32 [tokens, heads] is what `sdpa_paged` leaves with the same arguments
    (rows at -infinity have no weights; lse is float32, and weights are off by a factor of e^(|lse| 2^-24) for its rounding: 6 % where scores are a million).  The same
    call gives the same bits unless two of its sequences have one slot."""
    name = "weigh_paged"
    code, T, Hq, args = _step(name, Q, k_cache, page_table, slots, context_lens, max_context, scale, row_starts, max_rows, masks)
    if lse._shape != (T, Hq) or not _is(lse, float32):
        raise ValueError(f"{name}: lse must be float32 [{T}, {Hq}], got {lse.dtype} {lse.shape}")
    n_slots, H = page_table._shape[0], k_cache._shape[1]
    if len(weights._shape) != 3 or weights._shape[:2] != (n_slots, H) or not _is(weights, float32) or weights._shape[2] < max_context:
        raise ValueError(f"{name}: weights must be float32 [{n_slots}, {H}, positions >= {max_context}], got {weights.dtype} {weights.shape}")
    api.paged_weigh(Q._ptr, Hq * Q._shape[2], k_cache._ptr, lse._ptr, weights._ptr, weights._shape[2], *args, code, _st())


def select_rows(weights: GPUArray, slots: GPUArray, context_lens: GPUArray, budget: int, *, first: int = 0, recent: int = 0,
                out: "tuple[GPUArray, GPUArray] | None" = None) -> tuple[GPUArray, GPUArray]:
    """The positions that stay when sequences are cut to `budget`: the `first` and the `recent` ones, and of the others those of the largest weights, ties to
    the lower position; all of a sequence that has no more.  weights float32 [slots, kv_heads, positions]; contexts are taken up to `positions`.  Returns (kept
    int32 [sequences, kv_heads, budget], ascending, -1 behind the last; counts int32 [sequences]).  NaN is the smallest weight."""
    name = "select_rows"
    if len(weights._shape) != 3 or not _is(weights, float32) or min(weights._shape) < 1:
        raise ValueError(f"{name}: weights must be float32 [slots, kv_heads, positions], got {weights.dtype} {weights.shape}")
    n_slots, H, P = weights._shape
    if P > MOST_POSITIONS or n_slots >= 2 ** 31:
        raise ValueError(f"{name}: weights {weights.shape} ({MOST_POSITIONS} positions at most)")
    if len(slots._shape) != 1:
        raise ValueError(f"{name}: slots must be int32 [sequences], got {slots.dtype} {slots.shape}")
    S = slots._shape[0]
    _index(name, "slots", slots, S)
    _index(name, "context_lens", context_lens, S)
    if S > 65535:
        raise ValueError(f"{name}: {S} sequences (65535 at most)")
    if budget < 1 or first < 0 or recent < 0 or first + recent > budget or budget >= 2 ** 31:
        raise ValueError(f"{name}: a budget of {budget} with {first} first and {recent} recent positions")
    if out is None:
        out = GPUArray((S, H, budget), int32), GPUArray((S,), int32)
    kept, counts = out
    if kept._shape != (S, H, budget) or not _is(kept, int32):
        raise ValueError(f"{name}: out's positions must be int32 {(S, H, budget)}, got {kept.dtype} {kept.shape}")
    _index(name, "out's counts", counts, S)
    api.select_rows(weights._ptr, P, slots._ptr, context_lens._ptr, S, n_slots, H, P, budget, first, recent, kept._ptr, counts._ptr, _st())
    return out


def move_rows_paged(arrays: "list[GPUArray]", page_table: GPUArray, slots: GPUArray, rows: GPUArray, counts: GPUArray, *,
                    starts: "GPUArray | None" = None, weights: "GPUArray | None" = None, context_lens: "GPUArray | None" = None) -> None:
    """Rows of the pages move together, in place: position starts[s] + i (starts None: i) of sequence s becomes what position starts[s] + rows[s, i] was, in every
    array [pages, kv_heads, page_size, elements] (keys and values of any number of layers), for i < counts[s].  rows int32 [sequences, n], or
    [sequences, kv_heads, n] as `select_rows` returns them; rows[s, i] >= i, entries below and rows outside the pages are skipped.

    weights float32 [slots, kv_heads, positions] moves along, and what lies behind the last row up to context_lens[s], the context before the move, becomes zero.
    The arrays do not overlap, and no two of the call's sequences share the pages that are written."""
    name = "move_rows_paged"
    if not arrays:
        raise ValueError(f"{name}: no arrays")
    pages, H, ps, _, n_slots, max_pages = _pages(name, arrays[0], page_table)
    shape, dtype = arrays[0]._shape, arrays[0]._dtype
    sizes = array("i", [shape[3] * dtype.itemsize]) * len(arrays)
    unlike = [i for i, a in enumerate(arrays) if a._shape != shape or a._dtype is not dtype]      # most calls have none
    for i in (0, *unlike):
        a = arrays[i]
        if len(a._shape) != 4 or a._shape[:3] != shape[:3] or a._shape[3] < 1:
            raise ValueError(f"{name}: arrays [{pages}, {H}, {ps}, elements], got {a.shape}")
        if a._dtype == uint8:
            raise ValueError(f"{name}: pages of bytes keep a position's row in two places")
        sizes[i] = a._shape[3] * a._dtype.itemsize
        if sizes[i] % 2 or sizes[i] > 4096:
            raise ValueError(f"{name}: rows of an even number of bytes up to 4096, got {a._dtype} {a.shape}")
    ptrs = array("Q", [a._ptr for a in arrays])
    if len(set(ptrs)) < len(ptrs):
        raise ValueError(f"{name}: an array is there twice")
    if len(slots._shape) != 1:
        raise ValueError(f"{name}: slots must be int32 [sequences], got {slots.dtype} {slots.shape}")
    S = slots._shape[0]
    _index(name, "slots", slots, S)
    _index(name, "counts", counts, S)
    if S > 65535 or H > 500:
        raise ValueError(f"{name}: {S} sequences of {H} heads (65535 and 500 at most)")
    by_head = len(rows._shape) == 3
    if not _is(rows, int32) or rows._shape[:-1] != ((S, H) if by_head else (S,)):
        raise ValueError(f"{name}: rows must be int32 [{S}, n] or [{S}, {H}, n], got {rows.dtype} {rows.shape}")
    if rows._shape[-1] > MOST_POSITIONS:
        raise ValueError(f"{name}: {rows._shape[-1]} rows of a sequence ({MOST_POSITIONS} at most)")
    if starts is not None:
        _index(name, "starts", starts, S)
    ld = 0
    if weights is not None:
        if len(weights._shape) != 3 or weights._shape[:2] != (n_slots, H) or not _is(weights, float32):
            raise ValueError(f"{name}: weights must be float32 [{n_slots}, {H}, positions], got {weights.dtype} {weights.shape}")
        if context_lens is None:
            raise ValueError(f"{name}: weights move with context_lens")
        _index(name, "context_lens", context_lens, S)
        ld = weights._shape[2]
    api.move_rows(ptrs.buffer_info()[0], sizes.buffer_info()[0], len(ptrs), page_table._ptr, pages, ps, n_slots, max_pages, H, slots._ptr,
                  None if starts is None else starts._ptr, rows._ptr, counts._ptr, S, rows._shape[-1], 1 if by_head else 0, None if weights is None else weights._ptr, ld,
                  None if weights is None else context_lens._ptr, _st())


__all__ = ["sdpa_paged", "weigh_paged", "select_rows", "move_rows_paged"]
