"""Operators on the paged key / value cache in four bits (net-new: the reference's paged attention kernels,
native/ops/attention/paged_attention.cuh:46-283, read 16-bit pages).

A cache is two uint8 arrays, keys and values, `[pages, kv_heads, page_size, int4_row_bytes(head_dim)]` -- `llm.PagedKVCache` with dtype "int4"
makes them -- and an int32 page table `[slots, max_pages]`.  A group of 32 elements of a row is held as codes of four bits, a scale of four
significant bits and a zero point: 4.5 bits an element, and what they stand for is a bfloat16 number exactly.  Scales run from 2^-40 (smaller
groups are zeros) to 2^53; a group with a NaN, an infinity or a magnitude of 2^56 comes back as NaN.

Which rows and positions a call names is data on the device.  Whatever a slot, a position or a page number says, nothing outside the arrays is
touched: a row whose slot is negative (padding), or whose page does not exist, is skipped.
"""
from __future__ import annotations

from .._lib import api
from ..core.array import GPUArray
from ..core.dtypes import bfloat16, float32, float_code, int32, uint8
from ._common import _st

INT4_DIMS = (64, 96, 128, 192, 256)


def int4_row_bytes(head_dim: int) -> int:
    """Bytes of one head's row: codes of four bits and a 16-bit word per 32 elements."""
    if head_dim not in INT4_DIMS:
        raise ValueError(f"a cache in four bits serves heads of {', '.join(map(str, INT4_DIMS))} elements, got {head_dim}")
    return head_dim // 2 + head_dim // 16


def _is(a: GPUArray, dtype) -> bool:
    return a._dtype is dtype or a._dtype == dtype


def _cache_check(name: str, caches, page_table: GPUArray, kv_heads: int, dim: int) -> tuple[int, int, int, int]:
    """(pages, page size, slots, pages of a slot)"""
    row = int4_row_bytes(dim)
    shape = caches[0]._shape
    for c in caches:
        if len(c._shape) != 4 or not _is(c, uint8):
            raise ValueError(f"{name}: a cache is uint8 [pages, kv_heads, page_size, {row}], got {c.dtype} {c.shape}")
        if c._shape != shape:
            raise ValueError(f"{name}: the caches' shapes differ: {shape} and {c.shape}")
    pages, heads, page_size, held = shape
    if heads != kv_heads or held != row:
        raise ValueError(f"{name}: cache {shape} does not hold {kv_heads} heads of {dim} elements (rows of {row} bytes)")
    if len(page_table._shape) != 2 or not _is(page_table, int32):
        raise ValueError(f"{name}: page_table must be int32 [slots, max_pages], got {page_table.dtype} {page_table.shape}")
    if page_size < 16 or page_size % 16:
        raise ValueError(f"{name}: pages of {page_size} positions (multiples of 16)")
    slots, max_pages = page_table._shape
    return pages, page_size, slots, max_pages


def _index(name: str, what: str, a: GPUArray, n: int) -> None:
    if a._shape != (n,) or not _is(a, int32):
        raise ValueError(f"{name}: {what} must be int32 [{n}], got {a.dtype} {a.shape}")


def rope_append_paged_int4(q: "GPUArray | None", k: GPUArray, v: GPUArray, cos: "GPUArray | None", sin: "GPUArray | None", k_cache: GPUArray,
                           v_cache: GPUArray, page_table: GPUArray, slots: GPUArray, positions: GPUArray, *, interleaved: bool = False) -> None:
    """Rotate q [tokens, heads, dim] in place and k [tokens, kv_heads, dim], and write k and v into the cache at (slots[t], positions[t]).

    cos, sin: float32 [max positions, R], row p the angles of position p, R a multiple of 16 up to dim: the first R elements turn, in halves
    (i, i + R / 2) as `rope_inplace` turns them, or in neighbours (2 i, 2 i + 1) with `interleaved`; the first R / 2 columns are read.
    cos = sin = None: nothing turns.  q None: only keys and values.  The keys are rounded to four bits from their float32 values.  Rows of a
    call name different positions.  A row whose slot is negative, or whose position the tables do not have, is skipped, its q included."""
    name = "rope_append_paged_int4"
    code = float_code(k._dtype, name)
    shape = k._shape
    if len(shape) != 3 or v._shape != shape or not _is(v, k._dtype):
        raise ValueError(f"{name} expects k, v [tokens, kv_heads, dim] of one type, got {k.dtype} {k.shape} and {v.dtype} {v.shape}")
    T, H, D = shape
    Hq, q_ptr = 0, None
    if q is not None:
        if len(q._shape) != 3 or q._shape[0] != T or q._shape[2] != D or not _is(q, k._dtype):
            raise ValueError(f"{name} expects q [{T}, heads, {D}] of type {k.dtype}, got {q.dtype} {q.shape}")
        Hq, q_ptr = q._shape[1], q._ptr
    pages, ps, n_slots, max_pages = _cache_check(name, (k_cache, v_cache), page_table, H, D)
    _index(name, "slots", slots, T)
    _index(name, "positions", positions, T)
    rot, rows, cos_ptr, sin_ptr = 0, 0, None, None
    if (cos is None) != (sin is None):
        raise ValueError(f"{name}: cos and sin come together")
    if cos is not None:
        if len(cos._shape) != 2 or sin._shape != cos._shape or not _is(cos, float32) or not _is(sin, float32):
            raise ValueError(f"{name}: cos, sin must be float32 [max positions, R], got {cos.dtype} {cos.shape} and {sin.dtype} {sin.shape}")
        rows, rot = cos._shape
        if rows < 1 or rot < 16 or rot % 16 or rot > D:
            raise ValueError(f"{name}: a rotation of {rot} elements by tables of {rows} positions (R is a multiple of 16 up to {D})")
        cos_ptr, sin_ptr = cos._ptr, sin._ptr
    api.kv4_append(q_ptr, k._ptr, v._ptr, Hq * D, H * D, H * D, cos_ptr, sin_ptr, rows, rot, 1 if interleaved else 0, k_cache._ptr, v_cache._ptr, pages, ps,
                   page_table._ptr, n_slots, max_pages, slots._ptr, positions._ptr, T, Hq, H, D, code, _st())


def kv_read_paged_int4(cache: GPUArray, page_table: GPUArray, slots: GPUArray, positions: GPUArray, *, out: GPUArray | None = None) -> GPUArray:
    """What the cache holds at (slots[t], positions[t]) as rows [tokens, kv_heads, dim] (of `out`'s type; bfloat16, which is exact, without
    one).  Skipped rows come back as zeros."""
    name = "kv_read_paged_int4"
    shape = cache._shape
    if len(shape) != 4 or shape[3] % 9 or shape[3] // 9 * 16 not in INT4_DIMS:
        raise ValueError(f"{name}: a cache is uint8 [pages, kv_heads, page_size, row bytes], got {cache.dtype} {cache.shape}")
    H, D = shape[1], shape[3] // 9 * 16
    pages, ps, n_slots, max_pages = _cache_check(name, (cache,), page_table, H, D)
    if len(slots._shape) != 1:
        raise ValueError(f"{name}: slots must be int32 [tokens], got {slots.dtype} {slots.shape}")
    T = slots._shape[0]
    _index(name, "slots", slots, T)
    _index(name, "positions", positions, T)
    if out is None:
        out = GPUArray((T, H, D), bfloat16)
    elif out._shape != (T, H, D):
        raise ValueError(f"{name}: out shape {out.shape} does not match expected {(T, H, D)}")
    code = float_code(out._dtype, name)
    api.kv4_read(cache._ptr, pages, ps, page_table._ptr, n_slots, max_pages, slots._ptr, positions._ptr, out._ptr, T, H, D, code, _st())
    return out


def sdpa_paged_int4(Q: GPUArray, k_cache: GPUArray, v_cache: GPUArray, out: GPUArray, page_table: GPUArray, slots: GPUArray,
                    context_lens: GPUArray, max_context: int, scale: float = 0.0, *, row_starts: GPUArray | None = None, max_rows: int = 1,
                    window: int = 0, softcap: float = 0.0, sinks: GPUArray | None = None) -> None:
    """Causal attention of many sequences over the cache in four bits.  Q, out [tokens, heads, dim]; sequence s has the rows
    row_starts[s] ... row_starts[s + 1] - 1 (int32 [sequences + 1]), the last positions of its context_lens[s] cached ones -- one row each, row s,
    without row_starts.  max_context and max_rows bound what the two arrays hold: keys from max_context on are not seen, rows from
    max_rows on of a sequence and rows behind the last sequence keep their outputs, as do those of a sequence with a negative slot.

    scale 0: 1 / sqrt(dim).  window > 0: a row sees itself and the window - 1 positions before it.  softcap > 0: scores become softcap
    tanh(score / softcap).  Both are finite numbers, 1e-37 to 1e38 where they are not 0.  sinks float32 [heads]: a logit of each head that
    joins the softmax and carries no value.  A row that sees no key is zeros.  out may be Q.

    Sums are float32; values are weighed by weights rounded to 8 bits for bfloat16 rows, 16 for float16 and 24 for float32 ones (the attention
    on 16-bit pages keeps 24 for bfloat16 rows too), and float32 queries keep 22 bits of their row's largest element.  Heads of up to 128
    elements run on the tensor cores' large tiles from 17 rows (33 at 64 elements) a sequence and key head on, bfloat16 and float16, without a
    softcap above 177; the longest sequence of a call decides for all of it, so that a prompt and many decoded tokens are two calls rather than one."""
    name = "sdpa_paged_int4"
    code = float_code(Q._dtype, name)
    shape = Q._shape
    if len(shape) != 3 or out._shape != shape or not _is(out, Q._dtype):
        raise ValueError(f"{name} expects Q and out [tokens, heads, dim] of one type, got {Q.dtype} {Q.shape} and {out.dtype} {out.shape}")
    T, Hq, D = shape
    H = k_cache._shape[1] if len(k_cache._shape) == 4 else 0
    pages, ps, n_slots, max_pages = _cache_check(name, (k_cache, v_cache), page_table, H, D)
    if H < 1 or Hq < 1 or Hq % H:
        raise ValueError(f"{name}: n_heads {Hq} must be a multiple of KV heads {H}")
    if len(slots._shape) != 1:
        raise ValueError(f"{name}: slots must be int32 [sequences], got {slots.dtype} {slots.shape}")
    S = slots._shape[0]
    _index(name, "slots", slots, S)
    _index(name, "context_lens", context_lens, S)
    if row_starts is not None:
        _index(name, "row_starts", row_starts, S + 1)
    elif S != T or max_rows != 1:
        raise ValueError(f"{name}: {S} sequences and {T} rows need row_starts")
    if max_rows < 1 or not 0 <= max_context <= max_pages * ps:
        raise ValueError(f"{name}: max_rows {max_rows}, max_context {max_context} out of range ({max_pages} pages of {ps})")
    if window < 0 or not softcap >= 0.0 or not scale >= 0.0:
        raise ValueError(f"{name}: window {window}, softcap {softcap} and scale {scale} must not be negative")
    for what, x in (("softcap", softcap), ("scale", scale)):
        if x and not 1e-37 < x < 1e38:
            raise ValueError(f"{name}: {what} {x} is not 0 or a number that float32 keeps (1e-37 ... 1e38)")
    window, max_rows = min(window, 2**31 - 1), min(max_rows, max(T, 1))        # no position and no row lies behind
    if sinks is not None and (sinks._shape != (Hq,) or not _is(sinks, float32)):
        raise ValueError(f"{name}: sinks must be float32 [{Hq}], got {sinks.dtype} {sinks.shape}")
    api.kv4_attention(Q._ptr, Hq * D, k_cache._ptr, v_cache._ptr, out._ptr, Hq * D, pages, ps, page_table._ptr, n_slots, max_pages, slots._ptr,
                      context_lens._ptr, None if row_starts is None else row_starts._ptr, S, T, max_rows, max_context, Hq, H, D, scale, window, softcap,
                      None if sinks is None else sinks._ptr, code, _st())


__all__ = ["int4_row_bytes", "rope_append_paged_int4", "kv_read_paged_int4", "sdpa_paged_int4"]
