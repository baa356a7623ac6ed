"""A beam search that does not come to its end: nothing of it stays behind, and it can be run again; what it refuses.  No GPU."""
from types import SimpleNamespace

import numpy as np
import pytest

from pygpukit_b200 import ops
from pygpukit_b200.llm.decode import beam as beam_mod
from pygpukit_b200.llm.models.layered import LayeredCausalModel
from pygpukit_b200.llm.paged_cache import PagePool
from tests.test_int4_cache_cpu import arr

V = 7


class Model:
    """A function of a sequence's tokens, over a real pool of pages; the call number `fails` of what it names raises"""

    def __init__(self):
        self.pool = PagePool(page_size=4, pages=8, slots=2, max_pages_per_seq=4)
        self.held, self.config = {}, SimpleNamespace(vocab_size=V)
        self.cache = SimpleNamespace(pool=self.pool, assign=self.assign)
        self.calls, self.fails = 0, None

    def due(self, what):
        self.calls += 1
        if self.fails == (what, self.calls):
            raise RuntimeError("out of memory")

    def step_device(self, entries):
        rows = []
        for i, (seq, toks, _) in enumerate(entries):
            if i == len(entries) // 2:
                self.due("step")                                    # some sequences have their new positions, others not
            if seq in self.pool:
                self.pool.own_last_page(seq)
            _, first = self.pool.extend(seq, len(toks))
            assert first == len(self.held.setdefault(seq, []))
            self.held[seq] += toks
            x = np.random.default_rng([13, *self.held[seq]]).standard_normal(V)
            rows.append(x)
        return np.array(rows), len(rows)

    def assign(self, takes):
        self.due("assign early")
        self.pool.assign(takes)
        self.held.update({d: list(self.held[s]) for d, s in takes.items()})
        self.due("assign")

    def release(self, seq):
        self.pool.release(seq)
        self.held.pop(seq, None)


def make(model, monkeypatch, K=3):
    s = beam_mod.BeamSearch(model, K)

    def select(logits, scores, n):
        model.due("select")
        B, k = scores.shape
        x = logits.reshape(B, k, V)
        c = (scores[..., None] + x - np.log(np.exp(x).sum(-1, keepdims=True))).reshape(B, -1)
        o = np.argsort(-c, 1, kind="stable")[:, :n]
        return [np.take_along_axis(c, o, 1), o // V, o % V]

    monkeypatch.setattr(s, "_select", select)
    return s


def search(model, monkeypatch, prompts=([1, 2, 3], [4])):
    s = make(model, monkeypatch)
    for i, p in enumerate(prompts):
        s.add_request(i, p, 5)
    return s


@pytest.mark.parametrize("what", ["step", "select", "assign early", "assign"])
def test_a_search_that_fails_leaves_nothing_and_can_be_run_again(monkeypatch, what):
    want = search(Model(), monkeypatch).run()
    failed = 0
    for call in range(1, 25):
        model = Model()
        s = search(model, monkeypatch)
        model.fails = (what, call)
        try:
            s.run()
            continue
        except RuntimeError as e:
            assert "out of memory" in str(e)
        failed += 1
        assert model.pool.live_sequences == 0 and not model.pool._shared and model.pool.free_pages == model.pool.pages
        model.fails = None
        # another search on the same model, with requests of the same names, and the one that failed once more
        assert search(model, monkeypatch).run() == want
        assert s.run() == want
        assert model.pool.live_sequences == 0 and model.pool.free_pages == model.pool.pages
    assert failed >= 4


def test_searches_name_their_sequences_apart(monkeypatch):
    """what another search has in the cache, under the same names of requests, is not gone on from"""
    model = Model()
    want = search(Model(), monkeypatch).run()
    model.pool.extend((0, "beam", 0), 3)
    model.held[(0, "beam", 0)] = [9, 9, 9]
    assert search(model, monkeypatch).run() == want
    assert model.pool.live_sequences == 1 and model.pool.length((0, "beam", 0)) == 3


def test_more_requests_than_a_selection_has_rows_for(monkeypatch):
    prompts = [[1, 2, 3], [4], [0, 6], [5, 5], [2]]
    want = search(Model(), monkeypatch, prompts).run()
    monkeypatch.setattr(beam_mod, "MAX_ROWS", 7)                    # two requests of three beams
    model = Model()
    s = search(model, monkeypatch, prompts)
    inner, seen = s._select, []
    monkeypatch.setattr(s, "_select", lambda logits, scores, n: (seen.append(scores.size), inner(logits, scores, n))[1])
    assert s.run() == want and max(seen) == 6 and model.pool.live_sequences == 0
    failed = 0
    for call in range(1, 60):                                       # whichever step fails: requests are done, or wait
        model = Model()
        model.fails = ("step", call)
        s = search(model, monkeypatch, prompts)
        try:
            s.run()
            continue
        except RuntimeError:
            failed += 1
        assert len(s.finished) + len(s.waiting) == 5 and model.pool.live_sequences == 0
        model.fails = None
        assert s.run() == want
    assert failed >= 10


def test_a_selection_of_too_many_rows_is_refused():
    with pytest.raises(ValueError, match="beam_select"):
        ops.beam_select(arr((65536, 10)), arr((16384, 4)))


@pytest.mark.parametrize("bad", [dict(temperature=0.7), dict(top_k=5), dict(top_p=0.9), dict(prefill_chunk=16)], ids=str)
def test_generate_refuses_what_a_search_does_not_do(bad):
    with pytest.raises(ValueError, match="beam search takes no"):
        LayeredCausalModel.generate(Model(), [[1, 2]], 3, num_beams=2, **bad)
