"""Attention over the four-bit cache at the ends of its ranges: windows, contexts and caps of any size, long sums, weights that have fallen to zero; and
prompts whose tiles are made once, with pages, rows and values missing."""
import numpy as np
import pytest

from tests.test_gpu_int4_cache import Attend

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------- windows
WIDE = [  # (context, rows): a few, many, and many enough for tiles made once; rows before position 0 among them
    ([(3, 5), (70, 2), (1, 4)], "float32"),
    ([(3, 5), (70, 2), (1, 4)], "bfloat16"),
    ([(20, 60), (150, 40)], "bfloat16"),
    ([(100, 220), (300, 200)], "bfloat16"),
    ([(100, 220), (300, 200)], "float16"),
]


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30, 64])
@pytest.mark.parametrize("portions,dtype", WIDE, ids=str)
def test_windows_of_any_size(portions, dtype, window):
    """a window that reaches below position -2^31 is no window: rows before position 0 see nothing, the others everything"""
    a = Attend(portions, 8, 2, 128, 16, dtype, window=window, seed=50)
    got = a.run()
    a.check(got)
    for (ctx, n), at in zip(a.portions, a.starts):
        assert (got[at:at + max(0, n - ctx)] == 0).all() and (got[at + max(0, n - ctx):at + n] != 0).any(-1).all()
    if window > 2 ** 29:
        a.window = 0
        assert np.array_equal(a.run(), got)
