"""Infinities in the keys and values of a paged cache, before the step and among its rows: attention and the weights by position against float64."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.test_gpu_paged import Step

pytestmark = pytest.mark.gpu


def put(s, a, seq, j, head, elements, x):
    """elements of position j of a sequence's key head"""
    row = np.asarray(a[s.p.table[s.p.slots[seq], j // s.p.ps], :, j % s.p.ps]).copy()
    row[head, elements] = ref.rounded(np.array([x]), s.dtype)[0]
    s.p.put(a, seq, [j], [row])


def checked(s):
    got = s.run()
    with np.errstate(invalid="ignore"):               # infinities that agree, subtracted
        s.check(got)
    return got


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,D", [(1, 128), (9, 128), (40, 128), (40, 64), (3, 200), (1, 256)])
@pytest.mark.parametrize("context", [150, 17000])
def test_values_before_the_step(context, rows, D, dtype):
    """an infinity is what every row of its key head has there, whatever its weight; two of unlike signs, or a NaN, are NaN; a finite value beside them stays one"""
    s = Step([(context, rows), (99, rows)], 4, 2, D, 32, dtype, "tree" if rows > 1 else "chain", seed=21)
    for j, e, x in ((3, 0, np.inf), (70, 5, -np.inf), (4, 9, np.inf), (60, 9, -np.inf), (31, 11, np.nan), (context - rows - 1, D - 1, -np.inf)):
        put(s, s.p.v, 0, j, 1, e, x)
    out = checked(s)[0]
    assert (out[:rows, 2:, 0] == np.inf).all() and (out[:rows, 2:, [5, D - 1]] == -np.inf).all() and np.isnan(out[:rows, 2:, [9, 11]]).all()
    assert np.isfinite(np.delete(out[:rows, 2:], [0, 5, 9, 11, D - 1], axis=2)).all() and np.isfinite(out[:rows, :2]).all() and np.isfinite(out[rows:]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows", [2, 9, 60])
def test_values_before_the_step_and_among_its_rows(rows, dtype):
    s = Step([(300, rows)], 4, 2, 128, 16, dtype, "tree", seed=22)
    put(s, s.p.v, 0, 17, 0, 3, np.inf)
    put(s, s.p.v, 0, 300 - rows + 1, 0, 3, -np.inf)    # the step's row 1: where it is seen both are, NaN
    put(s, s.p.v, 0, 300 - 1, 0, 64, np.inf)
    out = checked(s)[0]
    sees = np.array([bool(m[1]) for m in s.masks])
    assert np.isnan(out[sees][:, :2, 3]).all() and (out[~sees][:, :2, 3] == np.inf).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_values_of_weights_that_are_zero(dtype):
    """an infinite value whose weight is too small for 32 bits is seen all the same; where a row's scores are NaN it is NaN throughout"""
    s = Step([(200, 2)], 4, 2, 128, 16, dtype, "chain", seed=23)
    s.q[:] = ref.rounded(np.full(s.q.shape, 1.0), dtype)
    for j in range(200):
        put(s, s.p.k, 0, j, slice(None), slice(None), -12.0 if j == 30 else 12.0)      # scores -136 and 136: weights of e^-272
    put(s, s.p.v, 0, 30, 1, 7, np.inf)
    out = s.run()[0]
    assert (out[:, 2:, 7] == np.inf).all() and np.isfinite(np.delete(out[:, 2:], 7, axis=2)).all() and np.isfinite(out[:, :2]).all()
    put(s, s.p.k, 0, 31, 1, 0, np.nan)
    out = s.run()[0]
    assert np.isnan(out[:, 2:]).all() and np.isfinite(out[:, :2]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,Hq", [(1, 8), (1, 32), (3, 2), (5, 14), (9, 16), (40, 6), (33, 2)])
def test_keys_whose_scores_are_minus_infinity(rows, Hq, dtype):
    """a key that is infinite where the queries are positive weighs nothing or all; rows that fill up a product have no part in it"""
    s = Step([(300, rows), (70, rows)], Hq, 2, 128, 32, dtype, "tree" if rows > 1 else "chain", seed=24)
    q = ref.floats(s.q, dtype)
    q[..., 17] = 1.0
    s.q = ref.rounded(q, dtype)
    minus = (0, 5), (0, 200), (1, 1), (0, 300 - 1)
    for seq, j in minus:
        put(s, s.p.k, seq, j, slice(None), 17, -30000.0)
    far = checked(s)                                   # scores that weigh nothing, either
    for seq, j in minus:
        put(s, s.p.k, seq, j, slice(None), 17, -np.inf)
    out, lse, weights = got = s.run()
    assert all(np.array_equal(x, y) for x, y in zip(got, far))
    assert np.isfinite(out).all() and np.isfinite(lse).all() and np.isfinite(weights).all()
    for seq, j in ((0, 5), (0, 200), (1, 1)):
        assert np.array_equal(weights[s.p.slots[seq], :, j], s.weights[s.p.slots[seq], :, j])
    put(s, s.p.k, 0, 9, 1, 17, np.inf)                 # a score of +infinity: the rows of its key head are NaN, and what they weigh
    out, lse, weights = s.run()
    assert np.isnan(out[:rows, Hq // 2:]).all() and np.isnan(lse[:rows, Hq // 2:]).all() and np.isfinite(out[:rows, :Hq // 2]).all() and np.isfinite(out[rows:]).all()
    assert np.isnan(weights[s.p.slots[0], 1, :300 - rows]).all() and np.isfinite(weights[s.p.slots[0], 0]).all() and np.isfinite(weights[s.p.slots[1]]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_a_key_that_only_the_next_sequence_would_see(dtype):
    """three rows of one head: the fourth place's mask is the next sequence's"""
    s = Step([(40, 3), (60, 6)], 2, 2, 128, 16, dtype, "tree", seed=25)
    s.masks = [np.array([True, False, False]), np.array([True, True, False]), np.array([True, True, False])] + [np.ones(6, bool)] * 6
    for x in (np.inf, np.nan):
        put(s, s.p.k, 0, 39, slice(None), 4, x)        # the step's row 2, which none of the three sees
        out, lse, weights = checked(s)
        assert np.isfinite(out).all() and np.isfinite(lse).all() and np.isfinite(weights).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,D,context", [(1, 128, 300), (9, 128, 300), (40, 128, 300), (40, 64, 300), (3, 200, 300), (1, 128, 9000), (40, 128, 9000)])
@pytest.mark.parametrize("most,sign", [(2.0 ** 21, 1), (2.0 ** 24, 1), (2.0 ** 25, -1), (2.0 ** 27, 1), (2.0 ** 30, -1), (2.0 ** 33, 1)])
def test_scores_of_any_size(most, sign, rows, D, context, dtype):
    """scores of c (1 - j / 64), j = 0 ... 31 in turns, of one product each, up to `most` or down from its negative: the difference of neighbours is far above a score's
    rounding, so that the keys of the largest score share the weight"""
    s = Step([(context, rows)], 4, 2, D, 32, dtype, "tree" if rows > 1 else "chain", seed=26)
    rng = np.random.default_rng(7)
    turn = rng.integers(0, 32, context)
    turn[:8] = np.arange(8)                            # the largest, and what comes next, before the step
    q, k = np.zeros(s.q.shape), np.zeros((context, 2, D))
    scale = 2.0 ** -4                                  # most = scale q k
    a = 2.0 ** np.ceil(np.log2(most / scale) / 2)
    q[..., 3], k[..., 3] = a, sign * (most / scale / a) * (1 - sign * turn[:, None] / 64)
    if max(a, np.abs(k).max()) > 60000 and dtype == "float16":
        pytest.skip("no such float16 numbers")
    s.q = ref.rounded(q, dtype)
    s.p.put(s.p.k, 0, range(context), ref.rounded(k, dtype))
    out, lse, weights = s.run(scale=scale)
    want, want_lse, _, _, by = ref.attention(s.p, ref.floats(s.q, dtype), s.starts, s.masks, scale)
    v = s.p.rows(s.p.v, 0, context)
    # weights of 1 / n: each is one rounding off its type, sums are exact but for float32's; the output's rounding
    spread = np.abs(v).max(axis=0)[np.arange(4) // 2][None]
    e = ref.EPS[dtype]
    assert np.isfinite(out).all() and (np.abs(out - want) <= (e + 2.0 ** -14) * spread).all()
    assert (np.abs(lse - want_lse) <= 2.0 ** -22 * np.abs(want_lse)).all()
