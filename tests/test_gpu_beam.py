"""Beam search's selection and the rows that follow, against NumPy in float64."""
import numpy as np
import pytest

from pygpukit_b200 import ops
from pygpukit_b200._lib import api
from pygpukit_b200.core.dtypes import float32, int32
from pygpukit_b200.core.factory import empty, from_numpy
from pygpukit_b200.core.stream import CudaGraph, Stream, synchronize, use_stream
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu


def i32(x):
    return from_numpy(np.ascontiguousarray(np.asarray(x, np.int32)))


def run(logits, scores, n, dtype, finished=None, pad=0):
    got = ops.beam_select(from_numpy(logits), from_numpy(scores.astype(np.float32)), n, finished=None if finished is None else i32(finished), pad_token=pad)
    return [a.to_numpy() for a in got]


def check(logits, scores, n, dtype="float32", finished=None, pad=0):
    with np.errstate(invalid="ignore", over="ignore"):
        want = ref.select(ref.floats(logits, dtype), scores.astype(np.float32), n, finished, pad)
    got = run(logits, scores, n, dtype, finished, pad)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    fin = np.isfinite(want[0])
    assert np.array_equal(np.isfinite(got[0]), fin) and (got[0][~fin] == want[0][~fin]).all()
    # a sum of exponentials of two units each in any order (2^-22 relative is 2^-22 of its logarithm), the sum's rounding
    assert (np.abs(got[0][fin] - want[0][fin]) <= 2.0 ** -22 * (4 + np.abs(want[0][fin]))).all()
    return got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 1, 3), (1, 4, 32768, 8), (3, 5, 8191, 10), (2, 8, 8193, 16), (2, 2, 1000, 64),
                                     (1, 64, 70, 64), (5, 4, 257, 8), (1, 3, 151936, 6), (16, 1, 33, 33)])
def test_selection(B, K, V, n, dtype):
    rng = np.random.default_rng(B * 100 + K + V)
    logits = ref.rounded(rng.standard_normal((B * K, V)) * 3, dtype)
    check(logits, -np.cumsum(rng.uniform(0, 2, (B, K)), 1), n, dtype)


@pytest.mark.parametrize("n", [4, 8, 64])
def test_ties_go_to_the_lowest_beam_and_token(n):
    rng = np.random.default_rng(n)
    logits = rng.integers(0, 3, (8, 20000)).astype(np.float32)      # three values only
    logits[1], logits[5] = logits[0], logits[4]                      # beams with the same rows
    scores = np.array([[-1, -1, -2, -2], [-3, -3, -3, -3]], np.float32)
    check(logits, scores, n)
    check(np.zeros((4, 9000), np.float32), np.zeros((1, 4), np.float32), n)
    signed = np.zeros((2, 300), np.float32)
    signed[:, ::2] = -0.0
    check(signed, np.zeros((1, 2), np.float32), n)


@pytest.mark.parametrize("order", [1, -1])
def test_sorted_rows(order):
    """all the best elements in one place"""
    logits = np.stack([np.linspace(-9, 9, 30000, dtype=np.float32)[::order] + k * 0.01 for k in range(4)]).astype(np.float32)
    check(logits, np.linspace(-1, -3, 4)[None], 64)
    logits = np.full((1, 20000), -5.0, np.float32)
    logits[0, 3::256] = np.arange(79)[:: order]                     # all in one thread's column
    check(logits, np.zeros((1, 1)), 64)


def test_first_step_and_masks():
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((8, 5000)).astype(np.float32)
    scores = np.full((2, 4), -np.inf, np.float32)
    scores[:, 0] = 0.0
    got = check(logits, scores, 8)
    assert (got[1] == 0).all()
    scores[:, 1:] = np.finfo(np.float32).min                         # masked by the type's lowest value
    got = run(logits, scores, 8, "float32")
    assert (got[1] == 0).all()
    logits[:, 7:] = -np.inf                                          # a constrained vocabulary: 7 tokens
    check(logits, np.array([[0, -1, -2, -3]] * 2, np.float32), 40)
    logits[:, :] = -np.inf
    check(logits, np.array([[0, -1, -2, -3]] * 2, np.float32), 10)
    check(logits, np.full((2, 4), -np.inf, np.float32), 10)


def test_what_is_not_a_number_stays_in_its_beam():
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((4, 9000)).astype(np.float32)
    scores = np.array([[0.0, -0.5, -1.0, np.nan]], np.float32)
    logits[0, 8500] = np.nan
    logits[1, 3] = np.inf
    got = check(logits, scores, 8)
    assert (got[1] == 2).all()
    check(logits, np.array([[0.0, -0.5, np.nan, np.nan]], np.float32), 8)


@pytest.mark.parametrize("pad", [0, 5, 6999])
def test_finished_beams_keep_their_score(pad):
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((12, 7000)).astype(np.float32) * 3
    logits[2] = np.nan                                               # what a finished beam's row holds is not read
    scores = -np.cumsum(rng.uniform(0.5, 1, (3, 4)), 1)
    finished = np.array([[0, 0, 1, 0], [1, 1, 1, 1], [0, 0, 0, 5]], np.int32)
    got = check(logits, scores, 12, "float32", finished, pad)
    assert got[2][1, :4].tolist() == [pad] * 4 and got[1][1, :4].tolist() == [0, 1, 2, 3]


def test_rows_apart_and_repeated_calls():
    """rows of a wider array, off 16-byte boundaries; the same bits every time"""
    rng = np.random.default_rng(4)
    wide = ref.rounded(rng.standard_normal((6, 10007)) * 3, "bfloat16")
    scores = from_numpy((-rng.uniform(0, 2, (2, 3))).astype(np.float32))
    x = from_numpy(wide)
    out = [empty((2, 6), t) for t in (float32, int32, int32)]
    first = None
    for _ in range(5):
        api.beam_select(x.device_ptr + 2 * 5, 10007, 2, scores.device_ptr, None, 0, 2, 3, 10000, 6, *[o.device_ptr for o in out], None)
        got = [o.to_numpy() for o in out]
        first = first or got
        assert all(np.array_equal(a, b) for a, b in zip(got, first))
    want = ref.select(ref.floats(wide[:, 5:10005], "bfloat16"), scores.to_numpy(), 6)
    assert np.array_equal(first[1], want[1]) and np.array_equal(first[2], want[2])


# ---------------------------------------------------------------------------------------------------- rows
@pytest.mark.parametrize("K", [1, 2, 5, 16, 17, 64])
@pytest.mark.parametrize("dtype,cols", [("float32", 4), ("float32", 1023), ("uint8", 7), ("uint8", 5000), ("bfloat16", 9), ("float32", 70001)])
def test_rows_follow_their_parents(K, dtype, cols):
    rng = np.random.default_rng(K + cols)
    B = 3
    shape = (B * K, cols)
    arrays = [rng.integers(0, 256, shape).astype(np.uint8) if dtype == "uint8" else
              (rng.integers(0, 60000, shape).astype(np.uint16) if dtype == "bfloat16" else rng.standard_normal(shape).astype(np.float32)) for _ in range(3)]
    arrays.append(rng.standard_normal((B * K, 3, 2)).astype(np.float32))
    dev = [from_numpy(a) for a in arrays]
    parents = rng.integers(0, K, (B, K)).astype(np.int32)
    parents[1] = np.roll(np.arange(K), 1)                            # a cycle
    parents[2, 0] = -1 if K % 2 else K                               # no beam of the group: stays
    ops.reorder_rows(dev, i32(parents))
    at = (parents + np.arange(B)[:, None] * K)
    at[2, 0] = 2 * K
    for a, d in zip(arrays, dev):
        assert np.array_equal(d.to_numpy(), a[at.reshape(-1)])


def test_more_arrays_than_a_launch_takes_and_rows_without_bytes():
    rng = np.random.default_rng(5)
    arrays = [rng.standard_normal((4, 1 + i % 9)).astype(np.float32) for i in range(150)]
    dev = [from_numpy(a) for a in arrays] + [empty((4, 0), float32)]
    ops.reorder_rows(dev, i32([[3, 2, 1, 0]]))
    assert all(np.array_equal(d.to_numpy(), a[::-1]) for a, d in zip(arrays, dev))
    ops.reorder_rows([], i32([[0]]))


@pytest.mark.parametrize("pairs", [1, 3, 16, 17, 100])
def test_pairs_of_rows(pairs):
    rng = np.random.default_rng(pairs)
    rows = rng.permutation(256)
    src, dst = rng.choice(rows[:100], pairs), rows[100:100 + pairs]        # a source may have several copies
    arrays = [rng.integers(0, 256, (256, 4608)).astype(np.uint8), rng.standard_normal((256, 3)).astype(np.float32)]
    dev = [from_numpy(a) for a in arrays]
    ops.copy_rows(dev, i32(np.r_[src, -1, 256, 5, 5]), i32(np.r_[dst, 201, 202, 256, -7]))
    for a, d in zip(arrays, dev):
        a[dst] = a[src]
        assert np.array_equal(d.to_numpy(), a)


def test_a_step_of_beam_search_captured():
    """select and reorder, captured once and replayed on new logits"""
    rng = np.random.default_rng(6)
    B, K, V = 2, 4, 3000
    s, g = Stream(), CudaGraph()
    logits, scores, state = empty((B * K, V), float32), empty((B, K), float32), empty((B * K, 100), float32)
    out = tuple(empty((B, K), t) for t in (float32, int32, int32))
    synchronize()
    with g.capture(s):
        ops.beam_select(logits, scores, K, out=out)
        ops.reorder_rows([state], out[1])
    with use_stream(s):
        for _ in range(3):
            x, y, z = rng.standard_normal((B * K, V)).astype(np.float32), -rng.uniform(0, 2, (B, K)).astype(np.float32), rng.standard_normal((B * K, 100)).astype(np.float32)
            for a, b in ((logits, x), (scores, y), (state, z)):
                a.copy_from_numpy(b)
            g.replay(s)
            want = ref.select(x, y, K)
            assert np.array_equal(out[1].to_numpy(), want[1]) and np.array_equal(out[2].to_numpy(), want[2])
            assert np.array_equal(state.to_numpy(), z[(want[1] + np.arange(B)[:, None] * K).reshape(-1)])
