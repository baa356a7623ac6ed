"""Beam search on the device (net-new): the selection over beams and vocabulary, and the rows of memory that follow their beams."""
from __future__ import annotations

import ctypes as C

from .._lib import api
from ..core.array import GPUArray
from ..core.dtypes import float32, float_code, int32
from ._common import _out, _st, _validate_float_dtype

MAX_BEAMS = 64


def beam_select(logits: GPUArray, scores: GPUArray, n: int | None = None, *, finished: GPUArray | None = None, pad_token: int = 0,
                out: "tuple[GPUArray, GPUArray, GPUArray] | None" = None) -> tuple[GPUArray, GPUArray, GPUArray]:
    """The n best continuations of every group of beams.  logits [groups * beams, vocab]; scores float32 [groups, beams], the beams' sums of log
    probabilities.  A candidate (beam k, token v) scores scores[k] + log_softmax(logits[k])[v]; returns (scores float32, beams int32, tokens int32), each
    [groups, n], best first, ties to the lower beam and then the lower token.  n (default: the number of beams) and beams are 64 at most.

    finished int32 [groups, beams]: a beam with a nonzero entry keeps its score and has one candidate, pad_token.  Other candidates at
    -infinity (logits of -infinity, beams whose score is NaN or below -1e30, rows that hold a NaN or +infinity) come last, in order."""
    name = "beam_select"
    _validate_float_dtype(logits, name)
    if scores.dtype != float32 or scores.ndim != 2:
        raise ValueError(f"{name}: scores must be float32 [groups, beams], got {scores.dtype} {scores.shape}")
    B, K = scores.shape
    if logits.ndim != 2 or logits.shape[0] != B * K or logits.shape[1] < 1:
        raise ValueError(f"{name}: logits must be [{B} * {K}, vocab], got {logits.shape}")
    V = logits.shape[1]
    n = K if n is None else int(n)
    if not 1 <= K <= MAX_BEAMS or not 1 <= n <= min(MAX_BEAMS, K * V):
        raise ValueError(f"{name}: {n} of {K} beams x {V} tokens (beams and candidates are 1 ... {MAX_BEAMS})")
    if finished is not None:
        if finished.dtype != int32 or finished.shape != scores.shape:
            raise ValueError(f"{name}: finished must be int32 {scores.shape}, got {finished.dtype} {finished.shape}")
        if not 0 <= pad_token < V:
            raise ValueError(f"{name}: pad_token {pad_token} is outside the vocabulary of {V}")
    given = out if out is not None else (None, None, None)
    got = tuple(_out(o, (B, n), dt, f"{name}: {what}") for o, dt, what in zip(given, (float32, int32, int32), ("scores", "beams", "tokens")))
    api.beam_select(logits.device_ptr, V, float_code(logits.dtype), scores.device_ptr, finished.device_ptr if finished is not None else None,
                    int(pad_token), B, K, V, n, got[0].device_ptr, got[1].device_ptr, got[2].device_ptr, _st())
    return got


def _rows_of(name: str, arrays) -> tuple[int, "C.Array", "C.Array"]:
    """(rows, device pointers, bytes of a row) of arrays that share their first dimension"""
    arrays = list(arrays)
    rows = arrays[0].shape[0] if arrays and arrays[0].ndim else 0
    for a in arrays:
        if a.ndim < 1 or a.shape[0] != rows:
            raise ValueError(f"{name}: arrays of {rows} rows, got {a.shape}")
    n = len(arrays)
    return rows, (C.c_void_p * n)(*[a.device_ptr for a in arrays]), (C.c_int64 * n)(*[a.nbytes // max(1, rows) for a in arrays])


def reorder_rows(arrays: "list[GPUArray]", parents: GPUArray) -> None:
    """Row (g, k) of every array [groups * beams, ...] becomes, in place, what row (g, parents[g, k]) was.  parents int32 [groups, beams], 64
    beams at most, as `beam_select` returns them.  A row whose parent is not one of its group's beams stays as it is.  The arrays do not overlap."""
    name = "reorder_rows"
    if parents.dtype != int32 or parents.ndim != 2 or not 1 <= parents.shape[1] <= MAX_BEAMS:
        raise ValueError(f"{name}: parents must be int32 [groups, beams] with 1 ... {MAX_BEAMS} beams, got {parents.dtype} {parents.shape}")
    if not arrays:
        return
    rows, ptrs, sizes = _rows_of(name, arrays)
    if rows != parents.size:
        raise ValueError(f"{name}: arrays of {rows} rows and parents {parents.shape}")
    api.copy_rows(ptrs, sizes, len(ptrs), rows, parents.device_ptr, None, parents.size, parents.shape[1], _st())


def copy_rows(arrays: "list[GPUArray]", src: GPUArray, dst: GPUArray) -> None:
    """Row dst[i] of every array [rows, ...] becomes row src[i] (int32 [pairs] on the device): pages of a cache, rows of states.  Destinations
    differ from one another and from every source; pairs that name a row outside the arrays are skipped.  The arrays do not overlap."""
    name = "copy_rows"
    for what, a in (("src", src), ("dst", dst)):
        if a.dtype != int32 or a.ndim != 1 or a.shape != src.shape:
            raise ValueError(f"{name}: {what} must be int32 [pairs], got {a.dtype} {a.shape}")
    if not arrays or not src.size:
        return
    rows, ptrs, sizes = _rows_of(name, arrays)
    api.copy_rows(ptrs, sizes, len(ptrs), rows, src.device_ptr, dst.device_ptr, src.size, 16, _st())


__all__ = ["beam_select", "reorder_rows", "copy_rows"]
