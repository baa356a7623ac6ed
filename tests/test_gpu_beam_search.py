"""Beam search through a model's steps, its cache and the operators, against a search over the float64 oracles; and a run of the operators on the
four-bit cache as a decoder's layer uses them."""
import math

import numpy as np
import pytest

from pygpukit_b200 import llm, ops
from pygpukit_b200.core.dtypes import bfloat16
from pygpukit_b200.core.factory import empty, from_numpy
from tests import kv4_ref as ref
from tests import test_gpu_goluzen, test_gpu_layered, test_gpu_rezulorn, test_gpu_sumitar, test_gpu_vosolorn

pytestmark = pytest.mark.gpu

MODELS = [  # pages alone; states beside pages, double-buffered ones and pooled rows among them
    (test_gpu_layered, None), (test_gpu_rezulorn, "base"), (test_gpu_vosolorn, None), (test_gpu_goluzen, None), (test_gpu_sumitar, None)]


def oracle_search(logits_of, prompt, K, n, eos, penalty):
    """(hypotheses best first, whether every choice had a margin): 2 K candidates a step as the search defines it"""
    beams, done, clear = [(0.0, [])], [], True
    for step in range(n):
        cand = []
        for k, (score, toks) in enumerate(beams):
            x = logits_of(prompt + toks)
            lp = x - (x.max() + math.log(np.exp(x - x.max()).sum()))
            cand += [(score + lp[t], k, t) for t in range(len(x))]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        gaps = [a[0] - b[0] for a, b in zip(cand[:2 * K], cand[1:2 * K + 1])]
        clear = clear and min(gaps) > 1e-4
        new = []
        for rank, (score, k, t) in enumerate(cand[:2 * K]):
            toks = beams[k][1] + [t]
            if t == eos:
                if rank < K:
                    done.append((score / len(toks) ** penalty, toks))
            elif len(new) < K:
                new.append((score, toks))
        done = sorted(done, reverse=True)[:K]
        beams = new
        if len(done) == K and max(b[0] / (step + 1) ** penalty for b in beams) <= done[-1][0]:
            break
    done += [(s / len(t) ** penalty, t) for s, t in beams]
    return sorted(done, reverse=True)[:K], clear


@pytest.mark.parametrize("which", range(len(MODELS)))
@pytest.mark.parametrize("K", [2, 4])
def test_a_search_against_the_oracle(which, K):
    mod, name = MODELS[which]
    cfg, P, m = mod.make(name or next(iter(mod.VARIANTS)), tokens_hint=64)
    prompts = [mod.tokens(cfg, k, seed=60 + k) for k in (3, 14, 8)]
    known = {}

    def logits_of(seq):
        if tuple(seq) not in known:
            known[tuple(seq)] = np.asarray(mod.R.forward(cfg, P, seq)[-1], np.float64)
        return known[tuple(seq)]

    eos = int(np.argsort(logits_of(prompts[0]))[-2])                 # a token that comes up
    for penalty, end in ((1.0, None), (0.6, eos)):
        outs = [oracle_search(logits_of, p, K, 7, end, penalty) for p in prompts]
        search = llm.BeamSearch(m, K, penalty)
        for i, p in enumerate(prompts):
            search.add_request(i, p, 7, end)
        got = search.run()
        compared = 0
        for i, (p, (want, clear)) in enumerate(zip(prompts, outs)):
            assert len(got[i]) == K and all(t[:len(p)] == p for _, t in got[i])
            if clear:
                compared += 1
                assert [t for _, t in got[i]] == [p + t for _, t in want]
                assert np.abs(np.array([c for c, _ in got[i]]) - np.array([c for c, _ in want])).max() < 1e-3      # seven steps of logits off by 2e-4 at most
        assert compared > 0
        assert m.cache.pool.live_sequences == 0 and not m.cache.pool._shared and m.cache.pool.free_pages == m.cache.pool.pages
        assert m.generate(prompts, 7, eos_token_id=end, num_beams=K, length_penalty=penalty) == [got[i][0][1] for i in range(3)]
    with pytest.raises(ValueError):
        m.generate(prompts, 3, temperature=1.0, num_beams=2)


def test_sequences_that_share_pages_on_the_device():
    """assign, cut back, grow: every position of every sequence holds what was written there"""
    rng = np.random.default_rng(1)
    H, D, PS = 2, 64, 16
    cache = llm.PagedKVCache([(H, D, D)] * 2, "int4", PS, tokens_hint=64, slots=2, state_shapes=[(5,), ()])
    want = {}

    def write(seq, n):
        slot, first = cache.extend(seq, n)
        x = rng.standard_normal((n, H, D)).astype(np.float32)
        table = cache.page_table()
        i32 = lambda a: from_numpy(np.asarray(a, np.int32))                                  # noqa: E731
        for layer in range(2):
            ops.rope_append_paged_int4(None, from_numpy(x + layer), from_numpy(x - layer), None, None, cache.k[layer], cache.v[layer], table, i32([slot] * n),
                                       i32(range(first, first + n)))
        want.setdefault(seq, []).extend(x)

    def check():
        table = cache.page_table()
        for seq, rows in want.items():
            n = len(rows)
            i32 = lambda a: from_numpy(np.asarray(a, np.int32))                              # noqa: E731
            for layer in range(2):
                got = ops.kv_read_paged_int4(cache.v[layer], table, i32([cache.pool.slot(seq)] * n), i32(range(n))).to_numpy()
                held = ref.decode(*ref.encode((np.array(rows) - layer).astype(np.float32)))
                assert np.array_equal(ref.floats(got, "bfloat16"), held.astype(np.float32))

    write("a", 21)
    write("b", 5)
    cache.state[0][0].copy_from_numpy(np.arange(cache.state[0][0].size, dtype=np.float32).reshape(cache.state[0][0].shape))
    state_of = cache.state[0][0].to_numpy()[cache.pool.slot("a")].copy()
    cache.assign({("a", k): "a" for k in range(5)} | {"b": "a"})
    want.update({s: list(want["a"]) for s in [("a", k) for k in range(5)] + ["b"]})
    assert all(np.array_equal(cache.state[0][0].to_numpy()[cache.pool.slot(s)], state_of) for s in want)
    check()
    for k in range(5):
        write(("a", k), 1 + 7 * k)
    cache.assign({("a", 0): ("a", 3), ("a", 1): ("a", 3), ("a", 3): ("a", 0), "c": ("a", 4)})
    old = dict(want)
    want.update({("a", 0): list(old[("a", 3)]), ("a", 1): list(old[("a", 3)]), ("a", 3): list(old[("a", 0)]), "c": list(old[("a", 4)])})
    check()
    bare = llm.PagedKVCache([(H, D, D)], "int4", PS, tokens_hint=64, slots=2)
    assert bare.k[0].shape[1:] == (H, PS, 36) and bare.dtype_code is None
    with pytest.raises(ValueError):
        cache.truncate("c", 3)                                       # it has states
    cache.release("b")
    del want["b"]
    check()


def test_a_layers_run_prompt_drafts_and_decoding():
    """A decoder layer's attention over the four-bit cache as it is used: two prompts of unequal length, decoded tokens, a draft that is taken back, a
    sequence that ends while another takes its place; each step against float64 over what was appended."""
    rng = np.random.default_rng(2)
    Hq, H, D, PS = 8, 2, 128, 16
    cache = llm.PagedKVCache([(H, D, D)], "int4", PS, tokens_hint=128, slots=2)
    a = np.arange(512)[:, None] * 1e4 ** (-np.arange(0, D, 2) / D)
    cos, sin = (np.concatenate([f(a), f(a)], 1).astype(np.float32) for f in (np.cos, np.sin))
    cosd, sind = from_numpy(cos), from_numpy(sin)
    held = {}

    def step(entries):
        """entries: (sequence, new rows)"""
        slots, pos, starts, ctx, seq_slots = [], [], [0], [], []
        for seq, n in entries:
            slot, first = cache.extend(seq, n)
            slots += [slot] * n
            pos += range(first, first + n)
            starts.append(starts[-1] + n)
            ctx.append(first + n)
            seq_slots.append(slot)
        T = starts[-1]
        q, k, v = (ref.rounded(rng.standard_normal((T, n, D)), "bfloat16") for n in (Hq, H, H))
        i32 = lambda x: from_numpy(np.asarray(x, np.int32))                                  # noqa: E731
        qd, table, out = from_numpy(q), cache.page_table(), empty((T, Hq, D), bfloat16)
        args = [from_numpy(k), from_numpy(v), i32(slots), i32(pos), i32(seq_slots), i32(ctx), i32(starts)]
        ops.rope_append_paged_int4(qd, args[0], args[1], cosd, sind, cache.k[0], cache.v[0], table, args[2], args[3])
        ops.sdpa_paged_int4(qd, cache.k[0], cache.v[0], out, table, args[4], args[5], max(ctx), row_starts=args[6], max_rows=max(n for _, n in entries))
        got, p = ref.floats(out.to_numpy(), "bfloat16").astype(np.float64), np.array(pos)
        kr = ref.encode(ref.rotate(ref.floats(k, "bfloat16"), cos[p], sin[p], False))
        vr = ref.encode(ref.floats(v, "bfloat16"))
        qr = ref.floats(ref.rounded(ref.rotate(ref.floats(q, "bfloat16"), cos[p], sin[p], False), "bfloat16"), "bfloat16").astype(np.float64)
        kx, vx = ref.decode(*kr), ref.decode(*vr)
        sx = np.repeat(((vr[1].astype(np.uint32) & 0x7FF0) << 16).astype(np.uint32).view(np.float32).astype(np.float64), 32, -1)
        for i, (seq, n) in enumerate(entries):
            rows = slice(starts[i], starts[i + 1])
            old = held.setdefault(seq, [np.zeros((0, H, D))] * 3)
            held[seq] = [np.concatenate([o, x[rows]]) for o, x in zip(old, (kx, vx, sx))]
            want, spread, size = ref.attention(qr[rows], *held[seq], ctx[i], 0, 0.0, None, 1.0 / math.sqrt(D))
            assert (np.abs(got[rows] - want) <= ref.bound(want, spread, size, D, "bfloat16", 0.0)).all()

    step([("a", 45), ("b", 130)])
    for _ in range(3):
        step([("b", 1), ("a", 1)])
    step([("a", 5), ("b", 1)])
    cache.truncate("a", 50)
    held["a"] = [x[:50] for x in held["a"]]
    step([("a", 1), ("b", 1)])
    cache.release("b")
    del held["b"]
    step([("c", 20), ("a", 1)])
    step([("c", 1), ("a", 1)])
