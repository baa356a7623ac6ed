"""Beam search on the device (net-new): the selection over beams and vocabulary, and the rows of memory that follow their beams."""
from __future__ import annotations

from array import array

from .._lib import api
from ..core.array import GPUArray
from ..core.dtypes import float32, float_code, int32
from ._common import _st
from .paged import _is

MAX_BEAMS = 64
MAX_ROWS = 65535             # groups x beams of a selection
MAX_VOCAB = 2048000


def beam_select(logits: GPUArray, scores: GPUArray, n: int | None = None, *, finished: GPUArray | None = None, pad_token: int = 0,
                out: "tuple[GPUArray, GPUArray, GPUArray] | None" = None) -> tuple[GPUArray, GPUArray, GPUArray]:
    """The n best continuations of every group of beams.  logits [groups * beams, vocab]; scores float32 [groups, beams], the beams' sums of log
    probabilities.  A candidate (beam k, token v) scores scores[k] + log_softmax(logits[k])[v]; returns (scores float32, beams int32, tokens int32), each
    [groups, n], best first, ties to the lower beam and then the lower token (of one beam the larger logit comes first, also where the scores round to one number).
    n (default: the number of beams) and beams are 64 at most, groups * beams 65535.

    finished int32 [groups, beams]: a beam with a nonzero entry keeps its score and has one candidate, pad_token.  Other candidates at
    -infinity (logits of -infinity, beams whose score is NaN or below -1e30, rows that hold a NaN or +infinity) come last, in order."""
    name = "beam_select"
    code = float_code(logits._dtype, name)
    if len(scores._shape) != 2 or not _is(scores, float32):
        raise ValueError(f"{name}: scores must be float32 [groups, beams], got {scores.dtype} {scores.shape}")
    B, K = scores._shape
    if len(logits._shape) != 2 or logits._shape[0] != B * K or not 1 <= logits._shape[1] <= MAX_VOCAB:
        raise ValueError(f"{name}: logits must be [{B} * {K}, vocab], got {logits.shape}")
    V = logits._shape[1]
    n = K if n is None else int(n)
    if B * K > MAX_ROWS:
        raise ValueError(f"{name}: {B} groups of {K} beams ({MAX_ROWS} rows at most)")
    if not 1 <= K <= MAX_BEAMS or not 1 <= n <= min(MAX_BEAMS, K * V):
        raise ValueError(f"{name}: {n} of {K} beams x {V} tokens (beams and candidates are 1 ... {MAX_BEAMS})")
    if finished is not None:
        if finished._shape != (B, K) or not _is(finished, int32):
            raise ValueError(f"{name}: finished must be int32 {scores.shape}, got {finished.dtype} {finished.shape}")
        if not 0 <= pad_token < V:
            raise ValueError(f"{name}: pad_token {pad_token} is outside the vocabulary of {V}")
    if out is None:
        out = tuple(GPUArray((B, n), dt) for dt in (float32, int32, int32))
    else:
        for o, dt, what in zip(out, (float32, int32, int32), ("scores", "beams", "tokens"), strict=True):
            if o._shape != (B, n) or not _is(o, dt):
                raise ValueError(f"{name}: out's {what} must be {dt} {(B, n)}, got {o.dtype} {o.shape}")
    got = out
    api.beam_select(logits._ptr, V, code, scores._ptr, None if finished is None else finished._ptr, pad_token, B, K, V, n, got[0]._ptr, got[1]._ptr,
                    got[2]._ptr, _st())
    return got


def _rows_of(name: str, arrays) -> tuple[int, array, array]:
    """(rows, device pointers, bytes of a row) of arrays that share their first dimension"""
    first = arrays[0]
    shape, dtype = first._shape, first._dtype
    rows = shape[0] if shape else 0
    if all([a._shape == shape and a._dtype is dtype for a in arrays]):
        if not shape:
            raise ValueError(f"{name}: an array without rows, {shape}")
        sizes = array("q", [first.nbytes // max(1, rows)]) * len(arrays)
    else:
        for a in arrays:
            if not a._shape or a._shape[0] != rows:
                raise ValueError(f"{name}: arrays of {rows} rows, got {a.shape}")
        sizes = array("q", [a.nbytes // max(1, rows) for a in arrays])
    ptrs = [a._ptr for a in arrays]
    if len(set(ptrs)) < len(ptrs):
        held = [p for p, n in zip(ptrs, sizes) if n]               # arrays without bytes may share an address
        if len(set(held)) < len(held):
            raise ValueError(f"{name}: an array is there twice")
    return rows, array("Q", ptrs), sizes


def reorder_rows(arrays: "list[GPUArray]", parents: GPUArray) -> None:
    """Row (g, k) of every array [groups * beams, ...] becomes, in place, what row (g, parents[g, k]) was.  parents int32 [groups, beams], 64
    beams at most, as `beam_select` returns them.  A row whose parent is not one of its group's beams stays as it is.  The arrays do not overlap."""
    name = "reorder_rows"
    if len(parents._shape) != 2 or not _is(parents, int32) or not 1 <= parents._shape[1] <= MAX_BEAMS:
        raise ValueError(f"{name}: parents must be int32 [groups, beams] with 1 ... {MAX_BEAMS} beams, got {parents.dtype} {parents.shape}")
    if not arrays:
        return
    rows, ptrs, sizes = _rows_of(name, arrays)
    if rows != parents.size:
        raise ValueError(f"{name}: arrays of {rows} rows and parents {parents.shape}")
    api.copy_rows(ptrs.buffer_info()[0], sizes.buffer_info()[0], len(ptrs), rows, parents._ptr, None, rows, parents._shape[1], _st())


def copy_rows(arrays: "list[GPUArray]", src: GPUArray, dst: GPUArray) -> None:
    """Row dst[i] of every array [rows, ...] becomes row src[i] (int32 [pairs] on the device): pages of a cache, rows of states.  Destinations
    differ from one another and from every source; pairs that name a row outside the arrays are skipped.  The arrays do not overlap."""
    name = "copy_rows"
    for what, a in (("src", src), ("dst", dst)):
        if len(a._shape) != 1 or a._shape != src._shape or not _is(a, int32):
            raise ValueError(f"{name}: {what} must be int32 [pairs], got {a.dtype} {a.shape}")
    if not arrays or not src.size:
        return
    rows, ptrs, sizes = _rows_of(name, arrays)
    api.copy_rows(ptrs.buffer_info()[0], sizes.buffer_info()[0], len(ptrs), rows, src._ptr, dst._ptr, src.size, 16, _st())


__all__ = ["beam_select", "reorder_rows", "copy_rows"]
