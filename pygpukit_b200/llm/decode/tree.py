"""Decode strategy with trees of drafted tokens (net-new; the reference's `DecodeSpeculative` drafts a chain): the model's first layers draft several tokens
behind every row of a level, the full model verifies the tree in one batched pass (`CausalTransformerModel.decode_step_tree_lookahead`)."""
from __future__ import annotations

import numpy as np

from ..._lib import api
from ...core.array import GPUArray
from ...core.dtypes import int32
from ...core.factory import zeros
from ...core.stream import current_stream_handle as _st
from ...ops.tree import tree_masks
from .base import DecodeStrategy


def tree_size(branches) -> int:
    """rows of a tree: the last accepted token, and branches[i] drafts behind each row of level i"""
    if not branches or any(int(w) != w or w < 1 for w in branches):
        raise ValueError(f"branches must be positive numbers of drafts, level by level, got {branches!r}")
    n = level = 1
    for w in branches:
        level *= int(w)
        n += level
    return n


class TreeStep:
    """what the layers and the acceptance take of a tree of n rows: views of the holder's arrays"""

    def __init__(self, rows: "TreeRows", n: int):
        words = -(-n // 32)
        self.masks, self.depths = rows.masks._view(0, (n, words)), rows.depths._view(0, (n,))
        self.zero, self.context, self.base, self.starts = (rows.ints._view(i, (k,)) for i, k in ((0, 1), (1, 1), (2, 1), (3, 2)))
        self.tokens, self.parents = rows.ints._view(5, (n,)), rows.ints._view(5 + n, (n,))


class TreeRows:
    """device arrays of the trees that a model steps through, one upload a step"""

    def __init__(self, most: int):
        self.most = most
        self.ints = GPUArray((5 + 2 * most,), int32)           # 0 | context | committed positions | first row, end | tokens | parents
        self.masks, self.depths = GPUArray((most * -(-most // 32),), int32), GPUArray((most,), int32)
        self._scores = zeros((most,))

    def scores(self, n: int) -> GPUArray:
        return self._scores._view(0, (n, 1))

    def step(self, tokens, parents, base: int) -> TreeStep:
        n = len(tokens)
        host = np.array([0, base + n, base, 0, n, *tokens, *parents], np.int32)
        api.upload(self.ints.device_ptr, host.ctypes.data, host.nbytes, _st())
        step = TreeStep(self, n)
        tree_masks(step.parents, step.starts, n, masks=step.masks, depths=step.depths)
        return step


class DecodeTree(DecodeStrategy):
    def __init__(self, branches: tuple = (3, 2, 1), draft_layers: int = 8) -> None:
        super().__init__()
        self._branches, self._draft_layers = tuple(int(w) for w in branches), draft_layers
        self._rows = tree_size(branches)

    def step(self, token_id: int, position: int, context_len: int, buffers):
        """Plain decode step: hidden [1, H] of one token."""
        return self.model._decode_step_fixed_cache(token_id, position, context_len)

    def step_tree(self, token_id: int, position: int, context_len: int) -> tuple[list[int], int, dict]:
        """(accepted tokens, new position, stats) for one step starting at `position`; `context_len` must be position + 1."""
        if context_len != position + 1:
            raise ValueError("step_tree expects context_len == position + 1")
        self.model.set_lookahead_confirmed_pos(position)
        accepted, stats = self.step_lookahead(token_id)
        return accepted, position + len(accepted), stats

    def step_lookahead(self, token_id: int) -> tuple[list[int], dict]:
        """the model tracks the committed position itself"""
        return self.model.decode_step_tree_lookahead(token_id, branches=self._branches, draft_layers=self._draft_layers)

    @property
    def branches(self) -> tuple:
        return self._branches

    @property
    def rows(self) -> int:
        """rows of the verifying pass: the buffers have as many (`init_decode(max_batch_size=...)`)"""
        return self._rows

    @property
    def draft_layers(self) -> int:
        return self._draft_layers


__all__ = ["DecodeTree", "TreeRows", "TreeStep", "tree_size"]
