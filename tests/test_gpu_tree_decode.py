"""Trees of drafts on a model: whatever the early layers draft, the emitted tokens are the full model's greedy tokens, and the cache behind a step holds what
plain steps leave; rows that move in a paged cache."""
import numpy as np
import pytest

from pygpukit_b200 import llm
from pygpukit_b200.core.dtypes import bf16_bits_to_f32
from pygpukit_b200.llm.decode.tree import tree_size
from tests.test_gpu_model import MAX_SEQ, _build, _check_tokens, _oracle_tokens

pytestmark = pytest.mark.gpu
N_NEW = 48


def _first(model, prompt):
    hidden = model.prefill(prompt)
    last = hidden.row(hidden.shape[0] - 1).view((1, hidden.shape[1]))
    model.set_lookahead_confirmed_pos(len(prompt))
    return int(np.argmax(bf16_bits_to_f32(model.get_logits(last).to_numpy()[0])))


def _run(model, prompt, n_new, branches, draft_layers, via_strategy=False):
    tok = _first(model, prompt)
    out, drafted, agreed, steps = [tok], 0, 0, 0
    strat = llm.DecodeTree(branches, draft_layers)
    strat.bind(model)
    assert strat.rows == tree_size(branches)
    while len(out) < n_new:
        pos = len(prompt) + len(out) - 1
        assert model.get_lookahead_confirmed_pos() == pos
        if via_strategy:
            accepted, new_pos, stats = strat.step_tree(tok, pos, pos + 1)
            assert new_pos == pos + len(accepted)
        else:
            accepted, stats = model.decode_step_tree_lookahead(tok, branches, draft_layers)
        assert 1 <= len(accepted) <= len(branches) + 1 and stats["draft_count"] == tree_size(branches) - 1
        assert stats["accepted_count"] == len(accepted) - 1
        out.extend(accepted)
        drafted, agreed, steps, tok = drafted + len(branches), agreed + stats["accepted_count"], steps + 1, accepted[-1]
    return out[:n_new], drafted, agreed, steps


@pytest.mark.parametrize("name,fmt", [("small-qwen3", "fp8"), ("small-llama", "nvf4"), ("tiny-qwen3", "bf16"), ("tiny-moe", "fp8")])
@pytest.mark.parametrize("branches,via_strategy", [((3, 2, 1), True), ((2, 2), False), ((1, 1, 1, 1), False), ((15,), True)])
def test_tokens_are_the_full_models_greedy_tokens(name, fmt, branches, via_strategy):
    model = _build(name, fmt)
    rng = np.random.default_rng(3)
    prompt = [int(t) for t in rng.integers(0, model.config.vocab_size, 12)]
    exp, margins, tops = _oracle_tokens((name, fmt), model, prompt, 128)
    got, _, _, steps = _run(model, prompt, N_NEW, branches, max(1, len(model.blocks) // 2), via_strategy)
    ok = _check_tokens(list(prompt) + got, exp[:len(prompt) + N_NEW], margins, len(prompt), tops)
    assert ok >= N_NEW // 4, f"only {ok} tokens before a tie"
    assert steps <= N_NEW


def test_a_draft_of_full_depth_is_accepted_and_wider_trees_accept_no_less():
    model = _build("small-qwen3", "fp8")
    prompt = [5, 99, 1023, 77, 300, 12, 640, 8]
    _, drafted, agreed, steps = _run(model, prompt, 40, (2, 2, 1), len(model.blocks))
    assert agreed >= 0.9 * drafted and steps <= 14
    with pytest.raises(ValueError, match="max_batch_size"):
        model.decode_step_tree_lookahead(5, (16, 1), 1)
    with pytest.raises(ValueError, match="fixed cache"):
        model.set_lookahead_confirmed_pos(MAX_SEQ - 4)
        model.decode_step_tree_lookahead(5, (2, 2), 1)


def test_the_cache_behind_a_step_is_that_of_plain_steps():
    model = _build("small-llama", "bf16")
    prompt = [9, 8, 7, 6, 5, 4]
    tok = _first(model, prompt)
    out = [tok]
    while len(out) < 30:
        accepted, _ = model.decode_step_tree_lookahead(out[-1], (3, 2), len(model.blocks) - 1)
        out.extend(accepted)
    n = model.get_lookahead_confirmed_pos()
    assert n == len(prompt) + len(out) - 1
    caches = [(k.copy(), v.copy()) for k, v in model.snapshot_kv_cache()]
    model.prefill(prompt + out[:-1])
    for (k, v), (k1, v1) in zip(caches, model.snapshot_kv_cache()):
        for a, b in ((k, k1), (v, v1)):
            x, y = bf16_bits_to_f32(a[:, :n]), bf16_bits_to_f32(b[:, :n])
            # layers' inputs went through attention in another order of sums: bfloat16 roundings of hidden states may fall on either side, a few of 2^-8
            assert np.abs(x - y).max() <= 2.0 ** -4 * np.abs(y).max()
            assert np.sqrt(np.mean((x - y) ** 2)) <= 2.0 ** -7 * np.sqrt(np.mean(y ** 2))


# ---------------------------------------------------------------------------------------------------- a paged cache
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_of_a_paged_cache_move_and_shared_pages_stay(dtype):
    cache = llm.PagedKVCache([(2, 16, 16), (2, 8, 0), (3, 16, 24)], dtype, page_size=4, tokens_hint=64, slots=4)
    rng = np.random.default_rng(5)
    cache.extend("a", 22)
    cache.extend("b", 9)
    host = []
    for arr in cache._page_arrays():
        x = rng.integers(0, 2 ** 14, arr.shape).astype(np.uint16) if dtype == "bfloat16" else rng.standard_normal(arr.shape).astype(np.float32)
        arr.copy_from_numpy(x)
        host.append(x)

    def rows(seq, arrays):
        pages, n = cache.pool.page_list(seq), cache.pool.length(seq)
        return [np.stack([a[pages[j // 4], :, j % 4] for j in range(n)]) for a in arrays]
    a, b = rows("a", host), rows("b", host)
    cache.assign({"c": "a"})                                       # shares a's whole pages
    cache.keep_rows({"a": (6, [0, 2, 3, 9, 15]), "b": (0, [0, 1, 2])})
    now = [x.to_numpy() for x in cache._page_arrays()]
    assert cache.pool.length("a") == 11 and cache.pool.length("b") == 3 and cache.pool.length("c") == 22
    keep = list(range(6)) + [6, 8, 9, 15, 21]
    for got, was in zip(rows("a", now), a):
        assert np.array_equal(got, was[keep])
    for got, was in zip(rows("b", now), b):
        assert np.array_equal(got, was[:3])
    for got, was in zip(rows("c", now), a):
        assert np.array_equal(got, was)
    cache.keep_rows({"c": (22, [])})
    cache.keep_rows({"c": (4, [1])})
    assert cache.pool.length("c") == 5
    for got, was in zip(rows("c", [x.to_numpy() for x in cache._page_arrays()]), a):
        assert np.array_equal(got, was[[0, 1, 2, 3, 5]])
    for bad in ((4, [1, 0]), (4, [0, 0]), (3, [2]), (6, []), (-1, []), (4, [-1])):
        with pytest.raises(ValueError, match="keep_rows"):
            cache.keep_rows({"c": bad})
    assert cache.pool.length("c") == 5
