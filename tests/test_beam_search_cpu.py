"""Pages that several sequences hold (PagePool.assign), and the bookkeeping of a beam search, without a GPU."""
import random
from types import SimpleNamespace

import numpy as np
import pytest

from pygpukit_b200.llm.decode import beam as beam_mod
from pygpukit_b200.llm.paged_cache import PagedKVCache, PagePool


class Memory:
    """What the device would hold: pages and slots, written as the pool says, and copied as it asks"""

    def __init__(self, **kw):
        self.pool = PagePool(**kw)
        self.pages, self.slots, self.want, self.n = {}, {}, {}, 0

    def extend(self, s, n):
        if s in self.pool:
            own = self.pool.own_last_page(s)
            if own:
                self.copy(self.pages, [own])
        slot, first = self.pool.extend(s, n)
        assert first == len(self.want.setdefault(s, []))
        for i in range(first, first + n):
            self.n += 1
            self.want[s].append(self.n)
            page = self.pool.table[slot, i // self.pool.page_size]
            self.pages.setdefault(page, {})[i % self.pool.page_size] = self.n
        self.slots[slot] = list(self.want[s])

    def copy(self, what, pairs):
        src, dst = [a for a, _ in pairs], [b for _, b in pairs]
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for a, b in pairs:
            what[b] = type(what[a])(what[a])

    def assign(self, takes):
        p, s = self.pool.assign(takes)
        self.copy(self.pages, p)
        self.copy(self.slots, s)
        self.want.update({d: list(w) for d, w in [(d, self.want[src]) for d, src in takes.items()]})

    def release(self, s):
        self.pool.release(s)
        del self.want[s]

    def truncate(self, s, n):
        self.pool.truncate(s, n)
        del self.want[s][n:]
        self.slots[self.pool.slot(s)] = list(self.want[s])

    def check(self):
        held = {}
        for s, want in self.want.items():
            assert self.pool.length(s) == len(want)
            slot, pages = self.pool.slot(s), self.pool.page_list(s)
            assert len(pages) == -(-len(want) // self.pool.page_size)
            got = [self.pages[self.pool.table[slot, i // self.pool.page_size]][i % self.pool.page_size] for i in range(len(want))]
            assert got == want and self.slots[slot] == want
            assert [self.pool.table[slot, i] for i in range(len(pages))] == pages
            for p in pages:
                held[p] = held.get(p, 0) + 1
        assert self.pool._shared == {p: n for p, n in held.items() if n > 1}
        free = sorted(self.pool._free_pages)
        assert sorted(free + list(held)) == list(range(self.pool.pages))
        slots = sorted(self.pool._free_slots + [self.pool.slot(s) for s in self.want])
        assert slots == list(range(self.pool.slots))


@pytest.mark.parametrize("seed", range(20))
def test_sequences_keep_what_they_hold(seed):
    r = random.Random(seed)
    m = Memory(page_size=r.choice([1, 3, 4]), pages=5, slots=2, max_pages_per_seq=2)
    for _ in range(300):
        names, op = list(m.want), r.random()
        if op < 0.45 or not names:
            m.extend(r.choice(names + ["n%d" % r.randrange(100)]), r.choice([1, 1, 2, 7]))
        elif op < 0.6 and len(names) > 3:
            m.release(r.choice(names))
        elif op < 0.7:
            s = r.choice(names)
            m.truncate(s, r.randrange(len(m.want[s]) + 1))
        else:
            dst = r.sample(names, r.randrange(1, len(names) + 1)) + ["n%d" % r.randrange(100) for _ in range(r.randrange(3))]
            m.assign({d: r.choice(names) for d in dst})
        m.check()


def test_a_step_of_beams_moves_whole_pages_by_count():
    m = Memory(page_size=4, pages=64, slots=8, max_pages_per_seq=16)
    m.extend("a", 11)
    m.assign({("a", k): "a" for k in range(3)})
    m.check()
    assert m.pool.free_pages == 64 - 2 - 4                          # two shared pages, four partly filled ones
    for k in range(3):
        m.extend(("a", k), 1)
    m.assign({("a", 0): ("a", 2), ("a", 1): ("a", 0), ("a", 2): ("a", 1)})      # nothing is copied: they change names
    assert m.pool.assign({("a", 0): ("a", 0)}) == ([], [])
    m.check()
    with pytest.raises(KeyError):
        m.pool.assign({"x": "nobody"})
    for s in list(m.want):
        m.release(s)
    assert m.pool.free_pages == 64 and not m.pool._shared


def test_a_page_that_others_hold_is_not_written():
    m = Memory(page_size=4, pages=16, slots=4, max_pages_per_seq=4)
    m.extend("a", 8)
    m.assign({"b": "a"})
    m.truncate("b", 6)
    with pytest.raises(RuntimeError, match="shared"):
        m.pool.extend("b", 1)
    m.extend("b", 3)
    m.check()


@pytest.mark.parametrize("bad", [dict(dtype="int8"), dict(dtype="int4", page_size=24), dict(dtype="int4", layer_shapes=[(2, 80, 80)]),
                                 dict(dtype="int4", layer_shapes=[(2, 128, 64)]), dict(dtype="int4", layer_shapes=[(1, 128, 0)]),
                                 dict(dtype="int4", pools=[8])], ids=str)
def test_four_bit_caches_refuse(bad):
    a = dict(layer_shapes=[(2, 128, 128)], dtype="int4", page_size=64)
    a.update(bad)
    with pytest.raises(ValueError):
        PagedKVCache(**a)


# ---------------------------------------------------------------------------------------------------- the search
def search(K, V, table, prompts, n, eos=None, penalty=1.0, monkeypatch=None):
    """BeamSearch over a model that is a function of a sequence's tokens"""
    held = {}

    class Array(np.ndarray):
        pass

    def step_device(entries):
        rows = []
        for seq, toks, want in entries:
            held.setdefault(seq, []).extend(toks)
            rows.append(table(tuple(held[seq])))
        return np.array(rows), len(rows)

    model = SimpleNamespace(config=SimpleNamespace(vocab_size=V), step_device=step_device, release=lambda s: held.pop(s),
                            cache=SimpleNamespace(assign=lambda takes: held.update({d: list(held[s]) for d, s in takes.items()})))
    s = beam_mod.BeamSearch(model, K, penalty)

    def select(logits, scores, n):
        B, k = scores.shape
        x = logits.reshape(B, k, V)
        with np.errstate(divide="ignore", invalid="ignore"):
            c = scores[..., None] + x - np.log(np.exp(x).sum(-1, keepdims=True))
        c[np.isnan(c)] = -np.inf
        flat = c.reshape(B, -1)
        o = np.argsort(-flat, 1, kind="stable")[:, :n]
        return [np.take_along_axis(flat, o, 1), o // V, o % V]

    def padded(logits, rows):
        out, at = [], 0
        for r in rows:
            out += [logits[at + min(i, r - 1)] for i in range(K)]
            at += r
        return np.array(out)

    monkeypatch.setattr(s, "_select", select)
    monkeypatch.setattr(s, "_padded", padded)
    for i, p in enumerate(prompts):
        s.add_request(i, p, n, eos)
    out = s.run()
    assert not held                                                 # every sequence was given back
    return out


def every(table, V, prompt, n, eos, penalty):
    """all continuations and what they count, best first"""
    out = []

    def walk(seq, score):
        g = len(seq) - len(prompt)
        if g and (seq[-1] == eos or g == n):
            out.append((score / g ** penalty, list(seq)))
            return
        x = table(tuple(seq))
        lp = x - np.log(np.exp(x).sum())
        for t in range(V):
            walk(seq + [t], score + lp[t])

    walk(list(prompt), 0.0)
    return sorted(out, reverse=True)


def random_table(V, seed):
    known = {}

    def table(seq):
        if seq not in known:
            known[seq] = np.random.default_rng(abs(hash((seed, seq))) % 2 ** 32).standard_normal(V) * 1.5
        return known[seq]
    return table


@pytest.mark.parametrize("eos", [None, 2])
@pytest.mark.parametrize("penalty", [0.0, 1.0])
def test_wide_beams_find_the_best_of_all(monkeypatch, eos, penalty):
    """as many beams as there are prefixes: nothing is lost"""
    for seed in range(5):
        V, n = 3, 3
        table = random_table(V, seed)
        prompts = [[1], [0, 2, 1]]
        got = search(27, V, table, prompts, n, eos, penalty, monkeypatch)
        for i, p in enumerate(prompts):
            want = every(table, V, p, n, eos, penalty)
            # scores are float32 sums, rounded once a step
            assert got[i][0][1] == want[0][1] and abs(got[i][0][0] - want[0][0]) <= n * 2.0 ** -24 * 16


def test_one_beam_is_greedy(monkeypatch):
    table = random_table(6, 3)
    got = search(1, 6, table, [[1, 2], [3]], 5, None, 1.0, monkeypatch)
    for i, p in enumerate(([1, 2], [3])):
        seq = list(p)
        for _ in range(5):
            seq.append(int(np.argmax(table(tuple(seq)))))
        assert got[i][0][1] == seq


@pytest.mark.parametrize("dead", [0, 2])
def test_a_model_without_continuations_ends_where_it_is(monkeypatch, dead):
    """logits that leave no candidate (masked, or not numbers): the beams as far as they came"""
    table = random_table(5, 1)
    got = search(5, 5, lambda seq: np.full(5, -np.inf) if len(seq) >= 1 + dead else table(seq), [[2]], 6, None, 1.0, monkeypatch)
    assert len(got[0]) == (5 if dead else 1) and all(len(t) == 1 + dead for _, t in got[0])
    want = every(table, 5, [2], dead, None, 1.0) if dead else [(0.0, [2])]
    assert got[0][0][1] == want[0][1]


def test_requests_and_refusals(monkeypatch):
    model = SimpleNamespace(config=SimpleNamespace(vocab_size=10))
    for k in (0, 33, -1):
        with pytest.raises(ValueError):
            beam_mod.BeamSearch(model, k)
    with pytest.raises(ValueError):
        beam_mod.BeamSearch(SimpleNamespace(config=SimpleNamespace(vocab_size=1)), 2)
    s = beam_mod.BeamSearch(model, 4)
    with pytest.raises(ValueError):
        s.add_request(0, [])
    s.add_request(0, [1], 0)
    s.add_request(1, [1], 3)
    for i in (0, 1):
        with pytest.raises(ValueError):
            s.add_request(i, [1])
    assert s.finished[0] == [(0.0, [1])]
    assert beam_mod.BeamSearch(model, 2).run() == {}
