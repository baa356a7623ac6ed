"""Trees of drafted tokens on the device (net-new: the reference's speculative steps draft chains): which rows of a step see each other, and which drafts
the model accepts.  A tree is given by its parents, int32 [tokens]: the number, within its sequence's rows, of the row that a row hangs on, smaller than its own;
anything else makes a row a root.  Sequence s has the rows row_starts[s] ... row_starts[s + 1] - 1 (int32 [sequences + 1])."""
from __future__ import annotations

from .._lib import api
from ..core.array import GPUArray
from ..core.dtypes import float_code, int32
from ._common import _st
from .paged import _index, _is

MAX_TREE_ROWS = 4096
MAX_MASK_WORDS = 1 << 18
MOST_VOCABULARY = 2 ** 31 - 2 ** 16


def _trees(name: str, parents: GPUArray, row_starts: GPUArray, max_rows: int) -> tuple[int, int]:
    """(tokens, sequences)"""
    if len(parents._shape) != 1 or not _is(parents, int32):
        raise ValueError(f"{name}: parents must be int32 [tokens], got {parents.dtype} {parents.shape}")
    if len(row_starts._shape) != 1 or row_starts._shape[0] < 1 or not _is(row_starts, int32):
        raise ValueError(f"{name}: row_starts must be int32 [sequences + 1], got {row_starts.dtype} {row_starts.shape}")
    if not 1 <= max_rows <= MAX_TREE_ROWS:
        raise ValueError(f"{name}: max_rows {max_rows} (1 ... {MAX_TREE_ROWS})")
    if parents._shape[0] >= 2 ** 31:
        raise ValueError(f"{name}: {parents._shape[0]} rows")
    return parents._shape[0], row_starts._shape[0] - 1


def tree_masks(parents: GPUArray, row_starts: GPUArray, max_rows: int, *, masks: "GPUArray | None" = None,
               depths: "GPUArray | None" = None) -> tuple[GPUArray, GPUArray]:
    """What `sdpa_paged` takes as masks: (masks int32 [tokens, words], depths int32 [tokens]), words = ceil(max_rows / 32) without `masks`.  A row's mask has its own
    bit and its ancestors', its depth is how many ancestors it has: its position behind the step's first one.  Rows from max_rows on of a sequence, and rows
    behind the last one, are left as they are."""
    name = "tree_masks"
    T, S = _trees(name, parents, row_starts, max_rows)
    words = -(-max_rows // 32)
    if masks is None:
        masks = GPUArray((T, words), int32)
    elif len(masks._shape) != 2 or masks._shape[0] != T or masks._shape[1] < words or not _is(masks, int32):
        raise ValueError(f"{name}: masks must be int32 [{T}, {words} words], got {masks.dtype} {masks.shape}")
    elif masks._shape[1] > MAX_MASK_WORDS:
        raise ValueError(f"{name}: masks of {masks._shape[1]} words ({MAX_MASK_WORDS} at most)")
    if depths is None:
        depths = GPUArray((T,), int32)
    else:
        _index(name, "depths", depths, T)
    api.tree_masks(parents._ptr, row_starts._ptr, S, T, max_rows, masks._shape[1], masks._ptr, depths._ptr, _st())
    return masks, depths


def accept_tree(logits: GPUArray, tokens: GPUArray, parents: GPUArray, row_starts: GPUArray, max_rows: int, *,
                out: "tuple[GPUArray, GPUArray, GPUArray] | None" = None) -> tuple[GPUArray, GPUArray, GPUArray]:
    """The drafts that the model accepts.  logits [tokens, vocab] of any float type: the model's choice behind a row is the largest, the lowest index of equal ones
    (NaN is never chosen; a row without anything above -infinity chooses 0); or int32 [tokens], the choices themselves, which a sampler made.  tokens int32 [tokens]: the
    rows' own.  Row 0 of a sequence, the last token that was accepted before the step, is accepted; then of a row's children the lowest whose token is the
    choice behind it.  Returns (rows int32 [sequences, max_rows], the accepted ones in order, -1 behind them; counts int32 [sequences]; next tokens int32 [sequences], the
    choice behind the last accepted row).  A sequence without rows has a count of 0 and the next token -1.  rows are what `move_rows_paged` takes."""
    name = "accept_tree"
    T, S = _trees(name, parents, row_starts, max_rows)
    _index(name, "tokens", tokens, T)
    V = code = 0
    if _is(logits, int32):
        _index(name, "choices", logits, T)
    else:
        code = float_code(logits._dtype, name)
        if len(logits._shape) != 2 or logits._shape[0] != T or logits._shape[1] < 1:
            raise ValueError(f"{name}: logits must be [{T}, vocab], got {logits.shape}")
        V = logits._shape[1]
        if V > MOST_VOCABULARY:
            raise ValueError(f"{name}: a vocabulary of {V} ({MOST_VOCABULARY} at most)")
    if T > 65535:
        raise ValueError(f"{name}: {T} rows (65535 at most)")
    if out is None:
        out = GPUArray((S, max_rows), int32), GPUArray((S,), int32), GPUArray((S,), int32)
    rows, counts, nxt = out
    if rows._shape != (S, max_rows) or not _is(rows, int32):
        raise ValueError(f"{name}: out's rows must be int32 {(S, max_rows)}, got {rows.dtype} {rows.shape}")
    _index(name, "out's counts", counts, S)
    _index(name, "out's next tokens", nxt, S)
    ptrs = (logits._ptr, V, code, V, None) if V else (None, 0, 0, 0, logits._ptr)
    api.accept_tree(*ptrs, tokens._ptr, parents._ptr, row_starts._ptr, S, T, max_rows, rows._ptr, counts._ptr, nxt._ptr, _st())
    return rows, counts, nxt


__all__ = ["tree_masks", "accept_tree"]
