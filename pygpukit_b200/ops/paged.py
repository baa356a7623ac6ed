"""Operators on the paged key / value cache in four bits (net-new: the reference's paged attention kernels,
native/ops/nn/attention/paged_attention.cuh:46-283, read 16-bit pages).

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
from ._common import _out, _st, _validate_float_dtype

INT4_DIMS = (64, 96, 128, 192, 256)


def int4_row_bytes(head_dim: int) -> int:
    """Bytes of one head's row: codes of four bits and a 16-bit word per 32 elements."""
    if head_dim not in INT4_DIMS:
        raise ValueError(f"a cache in four bits serves heads of {', '.join(map(str, INT4_DIMS))} elements, got {head_dim}")
    return head_dim // 2 + head_dim // 16


def _cache_check(name: str, caches, page_table: GPUArray, kv_heads: int, dim: int) -> tuple[int, int, int, int]:
    """(pages, page size, slots, pages of a slot)"""
    row = int4_row_bytes(dim)
    for c in caches:
        if c.dtype != uint8 or c.ndim != 4:
            raise ValueError(f"{name}: a cache is uint8 [pages, kv_heads, page_size, {row}], got {c.dtype} {c.shape}")
        if c.shape != caches[0].shape:
            raise ValueError(f"{name}: the caches' shapes differ: {caches[0].shape} and {c.shape}")
        if c.shape[1] != kv_heads or c.shape[3] != row:
            raise ValueError(f"{name}: cache {c.shape} does not hold {kv_heads} heads of {dim} elements (rows of {row} bytes)")
    if page_table.dtype != int32 or page_table.ndim != 2:
        raise ValueError(f"{name}: page_table must be int32 [slots, max_pages], got {page_table.dtype} {page_table.shape}")
    pages, _, page_size, _ = caches[0].shape
    if page_size < 16 or page_size % 16:
        raise ValueError(f"{name}: pages of {page_size} positions (multiples of 16)")
    return pages, page_size, page_table.shape[0], page_table.shape[1]


def _index(name: str, what: str, a: GPUArray, n: int) -> None:
    if a.dtype != int32 or a.ndim != 1 or a.shape[0] != n:
        raise ValueError(f"{name}: {what} must be int32 [{n}], got {a.dtype} {a.shape}")


def rope_append_paged_int4(q: "GPUArray | None", k: GPUArray, v: GPUArray, cos: "GPUArray | None", sin: "GPUArray | None", k_cache: GPUArray,
                           v_cache: GPUArray, page_table: GPUArray, slots: GPUArray, positions: GPUArray, *, interleaved: bool = False) -> None:
    """Rotate q [tokens, heads, dim] in place and k [tokens, kv_heads, dim], and write k and v into the cache at (slots[t], positions[t]).

    cos, sin: float32 [max positions, R], row p the angles of position p, R a multiple of 16 up to dim: the first R elements turn, in halves
    (i, i + R / 2) as `rope_inplace` turns them, or in neighbours (2 i, 2 i + 1) with `interleaved`; the first R / 2 columns are read.
    cos = sin = None: nothing turns.  q None: only keys and values.  The keys are rounded to four bits from their float32 values.  Rows of a
    call name different positions.  A row whose slot is negative, or whose position the tables do not have, is skipped, its q included."""
    name = "rope_append_paged_int4"
    _validate_float_dtype(k, name)
    if k.ndim != 3 or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{name} expects k, v [tokens, kv_heads, dim] of one type, got {k.dtype} {k.shape} and {v.dtype} {v.shape}")
    T, H, D = k.shape
    if q is not None and (q.ndim != 3 or q.dtype != k.dtype or q.shape[0] != T or q.shape[2] != D):
        raise ValueError(f"{name} expects q [{T}, heads, {D}] of type {k.dtype}, got {q.dtype} {q.shape}")
    pages, ps, n_slots, max_pages = _cache_check(name, (k_cache, v_cache), page_table, H, D)
    _index(name, "slots", slots, T)
    _index(name, "positions", positions, T)
    rot = rows = 0
    if (cos is None) != (sin is None):
        raise ValueError(f"{name}: cos and sin come together")
    if cos is not None:
        if cos.dtype != float32 or sin.dtype != float32 or cos.ndim != 2 or cos.shape != sin.shape:
            raise ValueError(f"{name}: cos, sin must be float32 [max positions, R], got {cos.dtype} {cos.shape} and {sin.dtype} {sin.shape}")
        rows, rot = cos.shape
        if rows < 1 or rot < 16 or rot % 16 or rot > D:
            raise ValueError(f"{name}: a rotation of {rot} elements by tables of {rows} positions (R is a multiple of 16 up to {D})")
    Hq = q.shape[1] if q is not None else 0
    api.kv4_append(q.device_ptr if q is not None else None, k.device_ptr, v.device_ptr, Hq * D, H * D, H * D, cos.device_ptr if rot else None,
                   sin.device_ptr if rot else None, rows, rot, 1 if interleaved else 0, k_cache.device_ptr, v_cache.device_ptr, pages, ps,
                   page_table.device_ptr, n_slots, max_pages, slots.device_ptr, positions.device_ptr, T, Hq, H, D, float_code(k.dtype), _st())


def kv_read_paged_int4(cache: GPUArray, page_table: GPUArray, slots: GPUArray, positions: GPUArray, *, out: GPUArray | None = None) -> GPUArray:
    """What the cache holds at (slots[t], positions[t]) as rows [tokens, kv_heads, dim] (of `out`'s type; bfloat16, which is exact, without
    one).  Skipped rows come back as zeros."""
    name = "kv_read_paged_int4"
    if cache.ndim != 4 or cache.shape[3] % 9 or cache.shape[3] // 9 * 16 not in INT4_DIMS:
        raise ValueError(f"{name}: a cache is uint8 [pages, kv_heads, page_size, row bytes], got {cache.dtype} {cache.shape}")
    H, D = cache.shape[1], cache.shape[3] // 9 * 16
    pages, ps, n_slots, max_pages = _cache_check(name, (cache,), page_table, H, D)
    if slots.ndim != 1:
        raise ValueError(f"{name}: slots must be int32 [tokens], got {slots.dtype} {slots.shape}")
    T = slots.shape[0]
    _index(name, "slots", slots, T)
    _index(name, "positions", positions, T)
    if out is not None:
        _validate_float_dtype(out, name)
    out = _out(out, (T, H, D), bfloat16 if out is None else out.dtype)
    api.kv4_read(cache.device_ptr, pages, ps, page_table.device_ptr, n_slots, max_pages, slots.device_ptr, positions.device_ptr, out.device_ptr, T, H, D,
                 float_code(out.dtype), _st())
    return out


def sdpa_paged_int4(Q: GPUArray, k_cache: GPUArray, v_cache: GPUArray, out: GPUArray, page_table: GPUArray, slots: GPUArray,
                    context_lens: GPUArray, max_context: int, scale: float = 0.0, *, row_starts: GPUArray | None = None, max_rows: int = 1,
                    window: int = 0, softcap: float = 0.0, sinks: GPUArray | None = None) -> None:
    """Causal attention of many sequences over the cache in four bits.  Q, out [tokens, heads, dim]; sequence s has the rows
    row_starts[s] ... row_starts[s + 1] - 1 (int32 [sequences + 1]), the last positions of its context_lens[s] cached ones -- one row each, row s,
    without row_starts.  max_context and max_rows bound what the two arrays hold: keys from max_context on are not seen, rows from
    max_rows on of a sequence and rows behind the last sequence keep their outputs, as do those of a sequence with a negative slot.

    scale 0: 1 / sqrt(dim).  window > 0: a row sees itself and the window - 1 positions before it.  softcap > 0: scores become
    softcap tanh(score / softcap).  sinks float32 [heads]: a logit of each head that joins the softmax and carries no value.  A row that sees no key is
    zeros.  Sums are float32; bfloat16 and float16 rows weigh values by weights of eight bits' rounding, float32 rows by full ones."""
    name = "sdpa_paged_int4"
    _validate_float_dtype(Q, name)
    if Q.ndim != 3 or out.shape != Q.shape or out.dtype != Q.dtype:
        raise ValueError(f"{name} expects Q and out [tokens, heads, dim] of one type, got {Q.dtype} {Q.shape} and {out.dtype} {out.shape}")
    T, Hq, D = Q.shape
    H = k_cache.shape[1] if k_cache.ndim == 4 else 0
    pages, ps, n_slots, max_pages = _cache_check(name, (k_cache, v_cache), page_table, H, D)
    if H < 1 or Hq % H:
        raise ValueError(f"{name}: n_heads {Hq} must be a multiple of KV heads {H}")
    if slots.ndim != 1:
        raise ValueError(f"{name}: slots must be int32 [sequences], got {slots.dtype} {slots.shape}")
    S = slots.shape[0]
    _index(name, "slots", slots, S)
    _index(name, "context_lens", context_lens, S)
    if row_starts is not None:
        _index(name, "row_starts", row_starts, S + 1)
    elif S != T or max_rows != 1:
        raise ValueError(f"{name}: {S} sequences and {T} rows need row_starts")
    if max_rows < 1 or max_context < 0 or max_context > max_pages * ps:
        raise ValueError(f"{name}: max_rows {max_rows}, max_context {max_context} out of range ({max_pages} pages of {ps})")
    if window < 0 or not softcap >= 0.0 or not scale >= 0.0:
        raise ValueError(f"{name}: window {window}, softcap {softcap} and scale {scale} must not be negative")
    if sinks is not None and (sinks.dtype != float32 or sinks.shape != (Hq,)):
        raise ValueError(f"{name}: sinks must be float32 [{Hq}], got {sinks.dtype} {sinks.shape}")
    api.kv4_attention(Q.device_ptr, Hq * D, k_cache.device_ptr, v_cache.device_ptr, out.device_ptr, Hq * D, pages, ps, page_table.device_ptr, n_slots,
                      max_pages, slots.device_ptr, context_lens.device_ptr, row_starts.device_ptr if row_starts is not None else None, S, T, int(max_rows),
                      int(max_context), Hq, H, D, float(scale), int(window), float(softcap), sinks.device_ptr if sinks is not None else None,
                      float_code(Q.dtype), _st())


__all__ = ["int4_row_bytes", "rope_append_paged_int4", "kv_read_paged_int4", "sdpa_paged_int4"]
