"""Beam search on the token-major models (net-new; the reference samples one continuation a prompt).

A prompt's beams are sequences of the model's cache: the prompt runs once, its sequence is taken by all of them, and every step is one ragged
batch of one token per beam.  Selection is on the device (`ops.beam_select`: 12 bytes a candidate come back), and `PagedKVCache.assign` lets
the chosen beams go on: whole pages are shared, partly filled pages and recurrent states are copied.

The search keeps 2 K candidates of K beams a step, best first: one that ends with `eos_token_id` among the first K is a finished hypothesis, the
first K others are the next beams.  A hypothesis counts score / length ** length_penalty, length being its generated tokens; a prompt is done
with K hypotheses that no beam can beat any more (by what its score counts at its present length), or at max_new_tokens.
"""
from __future__ import annotations

import heapq
import itertools
from dataclasses import dataclass, field

import numpy as np

from ...core.array import GPUArray
from ...core.dtypes import float32, int32
from ...ops.beam import MAX_BEAMS, MAX_ROWS, beam_select


class _Sequence:
    """the name of a beam's sequence in the cache, which no other search has"""


@dataclass
class _Search:
    id: object
    prompt: list[int]
    max_new_tokens: int
    eos: int | None
    beams: list = field(default_factory=list)          # (score, generated tokens, sequence)
    done: list = field(default_factory=list)           # heap of (what it counts, order, tokens): the worst first
    generated: int = 0


class BeamSearch:
    """`add_request`, then `run`: {request id: [(what it counts, prompt + generated tokens), ...] best first}.  Where a step raises, the cache gets
    the search's sequences back, and the requests that had not come to their end wait again: another `run` searches them from their prompts."""

    def __init__(self, model, num_beams: int, length_penalty: float = 1.0):
        if not 1 <= num_beams <= MAX_BEAMS // 2:
            raise ValueError(f"num_beams must be 1 ... {MAX_BEAMS // 2}, got {num_beams}")
        if 2 * num_beams > num_beams * model.config.vocab_size:
            raise ValueError("a vocabulary of one token has no second candidate")
        self.model, self.K, self.penalty = model, int(num_beams), float(length_penalty)
        self.waiting: list[_Search] = []
        self.finished: dict = {}
        self._held: dict = {}                          # sequences that the cache may have
        self._order = itertools.count()
        self._scores: GPUArray | None = None
        self._out = None

    def add_request(self, req_id, prompt: list[int], max_new_tokens: int = 20, eos_token_id: int | None = None) -> None:
        if req_id in self.finished or any(s.id == req_id for s in self.waiting):
            raise ValueError(f"request {req_id!r} already exists")
        if not prompt:
            raise ValueError("empty prompt")
        s = _Search(req_id, [int(t) for t in prompt], int(max_new_tokens), eos_token_id)
        if s.max_new_tokens <= 0:
            self.finished[req_id] = [(0.0, s.prompt)]
        else:
            self.waiting.append(s)

    # ------------------------------------------------------------------ one selection
    def _select(self, logits: GPUArray, scores: np.ndarray, n: int):
        B, K = scores.shape
        V = self.model.config.vocab_size
        if self._scores is None or self._scores.size < B * K:
            self._scores = GPUArray((B * K,), float32)
        if self._out is None or self._out[0].size < B * n:
            self._out = tuple(GPUArray((B * n,), t) for t in (float32, int32, int32))
        view = self._scores._view(0, (B, K))
        view.copy_from_numpy(scores)
        out = tuple(o._view(0, (B, n)) for o in self._out)
        beam_select(logits._view(0, (B * K, V)), view, n, out=out)
        return [o.to_numpy() for o in out]

    def _counts(self, score: float, length: int) -> float:
        return score / max(1, length) ** self.penalty

    def _finish(self, s: _Search, score: float, tokens: list[int]) -> None:
        heapq.heappush(s.done, (self._counts(score, len(tokens)), -next(self._order), tokens))
        if len(s.done) > self.K:
            heapq.heappop(s.done)

    def _release(self, seq) -> None:
        self.model.release(seq)
        del self._held[seq]

    def _advance(self, s: _Search, cand) -> dict:
        """The next beams from a step's candidates (scores, beams, tokens of one group); what the cache is asked for."""
        old = s.beams
        s.beams, s.generated = [], s.generated + 1
        for rank, (score, beam, tok) in enumerate(zip(*cand)):
            score, beam, tok = float(score), int(beam), int(tok)
            if score == -np.inf:                       # fewer candidates than beams
                break
            tokens = old[beam][1] + [tok]
            if s.eos is not None and tok == s.eos:
                if rank < self.K:
                    self._finish(s, score, tokens)
                continue
            if len(s.beams) < self.K:
                s.beams.append((score, tokens, beam))
        over = s.generated >= s.max_new_tokens or not s.beams
        if not over and len(s.done) == self.K:
            over = max(self._counts(b[0], s.generated) for b in s.beams) <= s.done[0][0]
        if over:
            for score, tokens, _ in s.beams or (() if s.done else old):        # no candidate at all: the beams as they were
                self._finish(s, score, tokens)
            for b in old:
                self._release(b[2])
            best = sorted(s.done, reverse=True)
            self.finished[s.id] = [(c, s.prompt + t) for c, _, t in best]
            s.beams = []
            return {}
        # beams keep their parents' sequences where they can; the others are taken from them
        used, takes, beams = set(), {}, []
        for score, tokens, beam in s.beams:
            src = old[beam][2]
            if src not in used:
                used.add(src)
                beams.append((score, tokens, src))
            else:
                new = _Sequence()
                takes[new] = src
                beams.append((score, tokens, new))
        s.beams = beams
        for b in old:
            if b[2] not in used:
                self._release(b[2])
        return takes

    # ------------------------------------------------------------------ the search
    def run(self) -> dict:
        """Search every waiting request to its end, side by side: as many at a time as a selection has rows for."""
        most = max(1, MAX_ROWS // self.K)
        while self.waiting:
            live, self.waiting = self.waiting[:most], self.waiting[most:]
            self._run_or_wait(live)
        return self.finished

    def _run_or_wait(self, live: list) -> None:
        try:
            self._run(live)
        except BaseException:
            cache = getattr(self.model, "cache", None)
            for seq in [q for q in self._held if cache is not None and q in cache.pool]:
                self.model.release(seq)
            self._held.clear()
            self.waiting = [_Search(s.id, s.prompt, s.max_new_tokens, s.eos) for s in live if s.id not in self.finished] + self.waiting
            raise

    def _run(self, live: list) -> None:
        for s in live:
            s.beams = [(0.0, [], _Sequence())]
            self._held[s.beams[0][2]] = None
        n0 = min(2 * self.K, self.model.config.vocab_size)
        entries = [(s.beams[0][2], s.prompt, [len(s.prompt) - 1]) for s in live]
        logits, _ = self.model.step_device(entries)
        cands = self._select(logits, np.zeros((len(live), 1), np.float32), n0)
        while True:
            takes = {}
            for i, s in enumerate(live):
                takes.update(self._advance(s, [c[i] for c in cands]))
            live = [s for s in live if s.beams]
            if not live:
                return
            if takes:
                self._held.update(dict.fromkeys(takes))
                self.model.cache.assign(takes)
            # beams that are missing (fewer candidates than K) have a row all the same: the first beam's, at -infinity
            entries, rows, scores = [], [], np.full((len(live), self.K), -np.inf, np.float32)
            for i, s in enumerate(live):
                for k, (score, tokens, seq) in enumerate(s.beams):
                    scores[i, k] = score
                    entries.append((seq, [tokens[-1]], [0]))
                rows.append(len(s.beams))
            logits, _ = self.model.step_device(entries)
            if any(r < self.K for r in rows):
                logits = self._padded(logits, rows)
            cands = self._select(logits, scores, 2 * self.K)

    def _padded(self, logits: GPUArray, rows: list[int]) -> GPUArray:
        """K rows for every request, where some have fewer beams"""
        from ..._lib import api
        from ...core.stream import current_stream_handle as _st
        V = self.model.config.vocab_size
        out, at = GPUArray((len(rows) * self.K, V), float32), 0
        for i, n in enumerate(rows):
            for k in range(self.K):
                api.memcpy_d2d(out.device_ptr + 4 * V * (i * self.K + k), logits.device_ptr + 4 * V * (at + min(k, n - 1)), 4 * V, _st())
            at += n
        return out


__all__ = ["BeamSearch"]
