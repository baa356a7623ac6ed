"""Paged key/value cache for many sequences (net-new: the reference's Python layers keep one fixed cache per
sequence; its paged-attention kernels, native/ops/nn/attention/paged_attention.cuh:46-283, are not wired to them).

`PagePool` is the host-side bookkeeping, pure Python so that it is tested without a GPU: a pool of pages of
`page_size` positions, a free list, and per sequence a slot (row of the device page table), its page list and its
length.  `PagedKVCache` adds the device side: per layer one K and one V array of `[pages, kv_heads, page_size, dim]`
(bfloat16 or float32) and the int32 page table `[slots, max_pages]` that the kernels read.  Sequences are named by
any hashable id; `release(id)` gives the slot and the pages back, and both are handed out again (lowest first).

Per-sequence STATE: a layer may keep, beside or instead of pages, float32 arrays with one row per slot (the state of a
recurrent mixer, the last inputs of a short convolution): `state[i][j]` is `[slots, n]`.  A state row needs no clearing
when its slot is handed out again -- the kernels that read it take a sequence whose first position is 0 as starting from
zero -- and cannot be truncated.

Pooled rows: a layer whose attention sees means of blocks of `pool` positions keeps them beside its pages, in two arrays
`[pages, kv_heads, rows, dim]` with rows = ceil(page_size / pool): the mean of block b lives with the page that holds the
block's last position, row b - floor(page_index page_size / pool), so that pages carry their blocks when they change hands.

Shared pages: `assign` makes sequences into what others hold (the beams of a search after a step: a beam goes on from itself, several
from one, some end).  Whole pages are shared and counted; a partly filled one goes to one of the takers and is copied for the others, as
state rows are, by `ops.copy_rows`.  A sequence that was cut back into a shared page gets a copy of its own before it grows again.

Rows that move: `keep_rows` cuts sequences to some of their positions, which move together in place (drafts of a tree that were accepted, evicted positions).

Four bits: dtype "int4" keeps uint8 arrays `[pages, kv_heads, page_size, ops.int4_row_bytes(dim)]` for the operators of `ops/paged.py` (keys and
values of one size, pages of a multiple of 16 positions, no pooled rows).  The models' layers do not read them: `LayeredCausalModel` refuses such a cache.

Growth: when the free list runs dry the pool doubles (device arrays are reallocated and the old pages copied, page
numbers stay valid); a page table row grows the same way.  Sizing the pool for the expected number of live tokens up
front (`tokens_hint`) avoids both.
"""
from __future__ import annotations

import heapq
import itertools

import numpy as np

from .._lib import api
from ..core.array import GPUArray
from ..core.dtypes import bfloat16, float32, int32, uint8
from ..core.factory import zeros
from ..core.stream import current_stream_handle as _st
from ..ops.beam import copy_rows
from ..ops.paged import int4_row_bytes
from ..ops.paged_rows import move_rows_paged


_versions = itertools.count(1)


class PagePool:
    def __init__(self, page_size: int, pages: int, slots: int, max_pages_per_seq: int):
        if page_size < 1 or pages < 1 or slots < 1 or max_pages_per_seq < 1:
            raise ValueError("PagePool: sizes must be positive")
        self.page_size, self.pages, self.slots, self.max_pages = page_size, pages, slots, max_pages_per_seq
        self._free_pages = list(range(pages))
        self._free_slots = list(range(slots))
        heapq.heapify(self._free_pages)
        heapq.heapify(self._free_slots)
        self._seq: dict = {}            # id -> [slot, [pages], length, steps that extended it]
        self.table = np.zeros((slots, max_pages_per_seq), np.int32)
        self.dirty = True               # the device copy of `table` is stale
        self._shared: dict = {}         # page -> sequences that hold it, where it is more than one

    # ---- queries
    def __contains__(self, seq_id) -> bool:
        return seq_id in self._seq

    def length(self, seq_id) -> int:
        return self._seq[seq_id][2]

    def slot(self, seq_id) -> int:
        return self._seq[seq_id][0]

    def steps(self, seq_id) -> int:
        """How many times the sequence has been extended (double-buffered per-sequence state flips on it)."""
        return self._seq[seq_id][3]

    def page_list(self, seq_id) -> list[int]:
        return list(self._seq[seq_id][1])

    @property
    def free_pages(self) -> int:
        return len(self._free_pages)

    @property
    def live_sequences(self) -> int:
        return len(self._seq)

    # ---- growth hooks (PagedKVCache reallocates the device arrays)
    def _grow_pages(self, need: int) -> None:
        new = max(self.pages * 2, self.pages + need)
        for p in range(self.pages, new):
            heapq.heappush(self._free_pages, p)
        self.pages = new

    def _grow_slots(self) -> None:
        new = self.slots * 2
        for s in range(self.slots, new):
            heapq.heappush(self._free_slots, s)
        self.table = np.concatenate([self.table, np.zeros((new - self.slots, self.max_pages), np.int32)])
        self.slots = new
        self.dirty = True

    def _grow_table(self, need: int) -> None:
        new = max(self.max_pages * 2, need)
        self.table = np.concatenate([self.table, np.zeros((self.slots, new - self.max_pages), np.int32)], axis=1)
        self.max_pages = new
        self.dirty = True

    # ---- allocation
    def extend(self, seq_id, n_tokens: int) -> tuple[int, int]:
        """Make room for `n_tokens` more positions of `seq_id` (a new id starts a sequence at position 0).
        Returns (slot, first new position)."""
        if n_tokens < 1:
            raise ValueError("extend: at least one token")
        ent = self._seq.get(seq_id)
        if ent is None:
            if not self._free_slots:
                self._grow_slots()
            ent = self._seq[seq_id] = [heapq.heappop(self._free_slots), [], 0, 0]
        slot, pages, length, _ = ent
        if length % self.page_size and pages[-1] in self._shared:
            raise RuntimeError("extend: the last page is shared (`own_last_page` first)")
        need = -(-(length + n_tokens) // self.page_size) - len(pages)
        if need > 0:
            if len(pages) + need > self.max_pages:
                self._grow_table(len(pages) + need)
            if need > len(self._free_pages):
                self._grow_pages(need - len(self._free_pages))
            for _ in range(need):
                p = heapq.heappop(self._free_pages)
                self.table[slot, len(pages)] = p
                pages.append(p)
            self.dirty = True
        ent[2] = length + n_tokens
        ent[3] += 1
        return slot, length

    def truncate(self, seq_id, length: int) -> None:
        """Forget the positions from `length` on (rejected speculative tokens); whole pages past it are freed."""
        ent = self._seq[seq_id]
        if not 0 <= length <= ent[2]:
            raise ValueError(f"truncate: length {length} outside 0..{ent[2]}")
        keep = -(-length // self.page_size)
        for p in ent[1][keep:]:
            self._drop(p)
        del ent[1][keep:]
        ent[2] = length

    def own_pages(self, seq_id, start: int) -> list:
        """Pages of its own in the place of those from position `start` on that others hold too: (that one, the new one) each, to be copied."""
        length = self._seq[seq_id][2]
        if not 0 <= start <= length:
            raise ValueError(f"own_pages: position {start} outside 0..{length}")
        plan = self.plan_pages([(seq_id, start, length)])
        pairs = self.pairs_of(plan)
        self.take_pages(plan)
        return pairs

    def plan_pages(self, ranges: list) -> list:
        """Pages of their own for the (id, start, end) of `ranges`, the first sequence first, in the place of those of the positions start ... end - 1 that others hold
        too: (id, number of the page in the sequence, new page) each, for `take_pages`.  No sequence changes; there are enough free pages then."""
        held, plan = dict(self._shared), []
        for seq_id, start, end in ranges:
            pages = self._seq[seq_id][1]
            for i in range(start // self.page_size, -(-end // self.page_size)):
                n = held.get(pages[i], 1)
                if n > 1:                              # the last of those that hold it keeps it
                    held[pages[i]] = n - 1
                    plan.append((seq_id, i))
        if len(plan) > len(self._free_pages):
            self._grow_pages(len(plan) - len(self._free_pages))
        return [(*at, new) for at, new in zip(plan, heapq.nsmallest(len(plan), self._free_pages))]

    def pairs_of(self, plan: list) -> list:
        """(page, new page) of a plan, to be copied before it is taken"""
        return [(self._seq[seq_id][1][i], new) for seq_id, i, new in plan]

    def take_pages(self, plan: list) -> None:
        """What `plan_pages` has planned, with nothing in between."""
        for seq_id, i, new in plan:
            slot, pages, _, _ = self._seq[seq_id]
            if heapq.heappop(self._free_pages) != new:
                raise RuntimeError("take_pages: pages were taken since they were planned")
            self._drop(pages[i])
            pages[i] = new
            self.table[slot, i] = new
            self.dirty = True

    def release(self, seq_id) -> None:
        slot, pages, _, _ = self._seq.pop(seq_id)
        for p in pages:
            self._drop(p)
        heapq.heappush(self._free_slots, slot)

    # ---- shared pages
    def _drop(self, page: int) -> None:
        n = self._shared.get(page, 1)
        if n == 1:
            heapq.heappush(self._free_pages, page)
        elif n == 2:
            del self._shared[page]
        else:
            self._shared[page] = n - 1

    def _new_page(self) -> int:
        if not self._free_pages:
            self._grow_pages(1)
        return heapq.heappop(self._free_pages)

    def own_last_page(self, seq_id) -> "tuple[int, int] | None":
        """A page of its own in the place of a partly filled last one that others hold too: (that one, the new one), to be copied."""
        slot, pages, length, _ = self._seq[seq_id]
        if not length % self.page_size or pages[-1] not in self._shared:
            return None
        old, new = pages[-1], self._new_page()
        self._drop(old)
        pages[-1] = new
        self.table[slot, len(pages) - 1] = new
        self.dirty = True
        return old, new

    def assign(self, takes: dict) -> tuple[list, list]:
        """Every sequence of `takes` (new ones among them) becomes what the one that it names was, all at once.  Returns the pairs of pages and the
        pairs of slots that have to be copied, (from, to) each: nothing that is copied to is copied from."""
        for src in takes.values():
            if src not in self._seq:
                raise KeyError(src)
        heirs: dict = {}                               # a sequence that is named, and those that hold its content in the end
        for dst, src in takes.items():
            heirs.setdefault(src, []).append(dst)
        for src, who in heirs.items():
            if src not in takes:                       # it stays what it is
                who.insert(0, src)
            elif src in who:                           # its own slot and last page stay with it
                who.remove(src)
                who.insert(0, src)
        old = {s: (e[0], list(e[1]), e[2], e[3]) for s, e in self._seq.items() if s in heirs or s in takes}
        free = [old[s][0] for s in takes if s in old and s not in heirs]       # slots whose content nobody takes
        lost = [p for s in takes if s in old and s not in heirs for p in old[s][1]]
        page_pairs, slot_pairs, given = [], [], {}
        for src, who in heirs.items():
            slot, pages, length, steps = old[src]
            part = length % self.page_size != 0
            if len(who) > 1:
                for p in pages[:-1] if part else pages:
                    self._shared[p] = self._shared.get(p, 1) + len(who) - 1
            for i, dst in enumerate(who):
                mine, at = list(pages), slot
                if i > 0:
                    if part:
                        mine[-1] = self._new_page()
                        page_pairs.append((pages[-1], mine[-1]))
                    if not free and not self._free_slots:
                        self._grow_slots()
                    at = free.pop() if free else heapq.heappop(self._free_slots)
                    slot_pairs.append((slot, at))
                given[dst] = [at, mine, length, steps]
        for p in lost:                                 # after the new pages were chosen: none of them is a source
            self._drop(p)
        for s in free:
            heapq.heappush(self._free_slots, s)
        for dst, ent in given.items():
            self._seq[dst] = ent
            self.table[ent[0], :len(ent[1])] = ent[1]
        self.dirty = True
        return page_pairs, slot_pairs


class PagedKVCache:
    """Device arrays of every layer + the page pool.  `layer_shapes` = [(kv_heads, dim, vdim), ...], one entry per cache
    (a layer that runs several times in a loop has one per run); vdim 0: the layer keeps one array whose rows serve as
    keys and, by a prefix, as values (latent attention) -- `v[i]` is then None; kv_heads 0: the layer has no pages at all.
    `state_shapes` = per cache the float32 elements per slot of each of its state arrays; `pools` = per cache the block size of
    its pooled rows (0: none; `pk[i]`, `pv[i]` are then None).
    `version` names the device arrays that are in use: another number, never given before in this process, whenever any of them is
    replaced.  (Their addresses name them no longer: freed memory comes back, for one array of a set and not for the next.)"""

    def __init__(self, layer_shapes: list[tuple[int, int, int]], dtype: str = "bfloat16", page_size: int = 64,
                 tokens_hint: int = 4096, slots: int = 8, state_shapes: "list[tuple] | None" = None,
                 pools: "list[int] | None" = None):
        if dtype not in ("bfloat16", "float32", "int4"):
            raise ValueError("PagedKVCache: dtype is 'bfloat16', 'float32' or 'int4'")
        self.dtype = {"bfloat16": bfloat16, "float32": float32, "int4": uint8}[dtype]
        self.dtype_code = {"bfloat16": 2, "float32": 0, "int4": None}[dtype]       # of the kernels that read float pages
        self.int4 = dtype == "int4"
        self.layer_shapes = list(layer_shapes)
        if self.int4:
            if page_size < 16 or page_size % 16:
                raise ValueError(f"PagedKVCache: four-bit pages of {page_size} positions (multiples of 16)")
            if pools and any(pools):
                raise ValueError("PagedKVCache: pooled rows are kept in 'bfloat16' or 'float32'")
            for g, d, dv in self.layer_shapes:
                if g > 0 and d != dv:
                    raise ValueError(f"PagedKVCache: four-bit keys of {d} elements with values of {dv} (one size)")
                if g > 0:
                    int4_row_bytes(d)
        pages = -(-max(1, tokens_hint) // page_size) + slots          # every live sequence may hold one partial page
        self.pool = PagePool(page_size, pages, slots, max(4, -(-max(1, tokens_hint) // page_size) + 1))
        self.k: list[GPUArray | None] = []
        self.v: list[GPUArray | None] = []
        self.pk: list[GPUArray | None] = []
        self.pv: list[GPUArray | None] = []
        self.pools = [int(p) for p in (pools or [0] * len(self.layer_shapes))]
        if len(self.pools) != len(self.layer_shapes) or any(p < 0 for p in self.pools):
            raise ValueError("PagedKVCache: one block size per cache")
        self._alloc(pages, copy_from=None)
        self.state_shapes = [tuple(int(n) for n in sh) for sh in (state_shapes or [()] * len(self.layer_shapes))]
        if len(self.state_shapes) != len(self.layer_shapes):
            raise ValueError("PagedKVCache: one tuple of state sizes per cache")
        self.state: list[list[GPUArray]] = []
        self._alloc_state(self.pool.slots, copy_from=None)
        self.table_dev = zeros((self.pool.slots * self.pool.max_pages,), int32)
        self._pairs: GPUArray | None = None            # rows that are copied, and the stream of the last copy
        self._pairs_stream = None

    @property
    def page_size(self) -> int:
        return self.pool.page_size

    def pool_rows(self, i: int) -> int:
        """rows per page of cache i's pooled arrays"""
        return -(-self.page_size // self.pools[i]) if self.pools[i] > 0 else 0

    def _alloc(self, pages: int, copy_from) -> None:
        ps = self.pool.page_size
        new: list[list] = [[], [], [], []]
        for i, (g, d, dv) in enumerate(self.layer_shapes):
            pr = self.pool_rows(i) if g > 0 and dv > 0 else 0
            if self.int4 and g > 0:
                d = dv = int4_row_bytes(d)
            shapes = ((g, ps, d) if g > 0 else None, (g, ps, dv) if dv > 0 and g > 0 else None, (g, pr, d) if pr else None,
                      (g, pr, dv) if pr else None)
            for arrays, old, sh in zip(new, (self.k, self.v, self.pk, self.pv), shapes):
                a = zeros((pages, *sh), self.dtype) if sh is not None else None
                if copy_from is not None and a is not None:
                    api.memcpy_d2d(a.device_ptr, old[i].device_ptr, old[i].nbytes, _st())
                arrays.append(a)
        if copy_from is not None:
            api.device_sync()
        self.k, self.v, self.pk, self.pv = new
        self.version = next(_versions)
        self._pages_dev = pages

    def _alloc_state(self, slots: int, copy_from) -> None:
        new = []
        for i, sizes in enumerate(self.state_shapes):
            arrs = []
            for j, n in enumerate(sizes):
                a = zeros((slots, n), float32)
                if copy_from is not None:
                    api.memcpy_d2d(a.device_ptr, self.state[i][j].device_ptr, self.state[i][j].nbytes, _st())
                arrs.append(a)
            new.append(arrs)
        if copy_from is not None:
            api.device_sync()
        self.state = new
        self.version = next(_versions)
        self._slots_dev = slots

    @property
    def has_state(self) -> bool:
        return any(self.state_shapes)

    def _grown(self) -> None:
        if self.pool.pages > self._pages_dev:
            self._alloc(self.pool.pages, copy_from=True)
        if self.pool.slots > self._slots_dev:
            self._alloc_state(self.pool.slots, copy_from=True)

    def _copy(self, arrays, pairs) -> None:
        """rows of the arrays, (from, to) each, in the order of the current stream"""
        if not pairs or not arrays:
            return
        n = len(pairs)
        host = np.asarray(pairs, np.int32).T.copy()
        if self._pairs is None or self._pairs.size < 2 * n:
            self._pairs = GPUArray((max(128, 4 * n),), int32)
        if self._pairs_stream is not _st():            # the copy before, on another stream, may still read its pairs
            api.device_sync()
            self._pairs_stream = _st()
        api.upload(self._pairs.device_ptr, host.ctypes.data, host.nbytes, _st())
        copy_rows(arrays, self._pairs._view(0, (n,)), self._pairs._view(n, (n,)))

    def _page_arrays(self) -> list:
        return [a for arrs in (self.k, self.v, self.pk, self.pv) for a in arrs if a is not None]

    def extend(self, seq_id, n_tokens: int) -> tuple[int, int]:
        if seq_id in self.pool and n_tokens > 0:
            own = self.pool.own_last_page(seq_id)
            if own is not None:
                self._grown()
                self._copy(self._page_arrays(), [own])
        out = self.pool.extend(seq_id, n_tokens)
        self._grown()
        return out

    def assign(self, takes: dict) -> None:
        """Every sequence of `takes` (new ones among them) becomes what the one that it names was, all at once: {new or old id: id}.  What is
        shared stays where it is; partly filled pages and state rows of the others are copied in the order of the current stream."""
        pages, slots = self.pool.assign(takes)
        self._grown()
        self._copy(self._page_arrays(), pages)
        self._copy([a for arrs in self.state for a in arrs], slots)

    def page_table(self) -> GPUArray:
        """The device's page table, up to date, as int32 [slots, pages of a slot]."""
        self.sync_table()
        return self.table_dev.view((self.pool.slots, self.pool.max_pages))

    def release(self, seq_id) -> None:
        self.pool.release(seq_id)

    def truncate(self, seq_id, length: int) -> None:
        if self.has_state and length != self.pool.length(seq_id):
            raise ValueError("PagedKVCache: a sequence with recurrent state cannot be cut back")
        self.pool.truncate(seq_id, length)

    def keep_rows(self, keeps: dict) -> None:
        """Cut sequences to some of their positions: {id: (start, rows)} leaves the positions before `start`, and behind them those at start + rows[0],
        start + rows[1], ... (ascending numbers), in every layer; the sequence ends there.  Accepted drafts of a tree, say, or what is left when
        positions are evicted, the same ones of all key heads.  Rows move in the order of the current stream (`ops.move_rows_paged`).  Pages that rows move into and that others
        hold too are copied first; a call that fails for want of memory leaves every sequence as it was.  Keys stay turned by the positions that they had, while what is appended later is
        numbered from the sequence's new length on: a program that evicts turned keys numbers its queries itself."""
        if self.int4 or self.has_state or any(self.pools):
            raise ValueError("PagedKVCache: rows of four-bit pages, pooled rows and recurrent states do not move")
        # everything is looked at before anything changes
        for seq, (start, rows) in keeps.items():
            length = self.pool.length(seq)
            if not 0 <= start <= length or any(not 0 <= r < length - start for r in rows) or any(a >= b for a, b in zip(rows, rows[1:])):
                raise ValueError(f"keep_rows: rows {list(rows)!r} behind position {start} of a sequence of {length} (ascending)")
        moving = [(seq, start, rows) for seq, (start, rows) in keeps.items() if any(r != i for i, r in enumerate(rows))]
        if moving:
            # pages that a row moves into: from the first row that is another one to the last
            plan = self.pool.plan_pages([(seq, start + next(i for i, r in enumerate(rows) if r != i), start + len(rows)) for seq, start, rows in moving])
            self._grown()
            self._copy(self._page_arrays(), self.pool.pairs_of(plan))
            self.pool.take_pages(plan)
            table, arrays = self.page_table(), self._page_arrays()
            S, width = len(moving), max(len(rows) for _, _, rows in moving)
            host = np.full(S * (3 + width), -1, np.int32)
            host[:S] = [self.pool.slot(seq) for seq, _, _ in moving]
            host[S:2 * S] = [start for _, start, _ in moving]
            host[2 * S:3 * S] = [len(rows) for _, _, rows in moving]
            for i, (_, _, rows) in enumerate(moving):
                host[3 * S + i * width:3 * S + i * width + len(rows)] = rows
            dev = GPUArray((host.size,), int32)
            api.upload(dev.device_ptr, host.ctypes.data, host.nbytes, _st())
            slots, starts, counts = (dev._view(i * S, (S,)) for i in range(3))
            at = dev._view(3 * S, (S, width))
            for heads in sorted({a.shape[1] for a in arrays}):        # a call's arrays have one number of heads
                move_rows_paged([a for a in arrays if a.shape[1] == heads], table, slots, at, counts, starts=starts)
        for seq, (start, rows) in keeps.items():
            self.pool.truncate(seq, start + len(rows))

    def sync_table(self) -> None:
        """Upload the page table when it changed since the last upload."""
        if not self.pool.dirty:
            return
        t = self.pool.table
        if self.table_dev.size != t.size:
            self.table_dev = GPUArray((t.size,), int32)
            self.version = next(_versions)
        api.upload(self.table_dev.device_ptr, t.ctypes.data, t.nbytes, _st())       # a copy is taken: `t` may change at once
        self.pool.dirty = False

    @property
    def nbytes(self) -> int:
        return (sum(a.nbytes for arrs in (self.k, self.v, self.pk, self.pv) for a in arrs if a is not None)
                + sum(a.nbytes for arrs in self.state for a in arrs))


__all__ = ["PagePool", "PagedKVCache"]
