"""Arguments at the ends of their types: what a 32-bit call would take for another number is refused, or is the number that it means.  No GPU."""
from types import SimpleNamespace

import pytest

from pygpukit_b200 import _lib, ops
from pygpukit_b200.core.dtypes import bfloat16, int32, uint8
from pygpukit_b200.llm.models.layered import LayeredCausalModel
from pygpukit_b200.ops import paged
from tests.test_int4_cache_cpu import arr


def call(**kw):
    a = dict(Q=arr((5, 8, 128), bfloat16), k_cache=arr((9, 2, 16, 72), uint8), v_cache=arr((9, 2, 16, 72), uint8), out=arr((5, 8, 128), bfloat16),
             page_table=arr((3, 4), int32), slots=arr((2,), int32), context_lens=arr((2,), int32), max_context=64, row_starts=arr((3,), int32), max_rows=5)
    a.update(kw)
    ops.sdpa_paged_int4(**a)


@pytest.mark.parametrize("bad", [dict(scale=float("inf")), dict(softcap=float("inf")), dict(scale=1e-60), dict(softcap=1e-60), dict(scale=1e39), dict(softcap=1e300)],
                         ids=str)
def test_numbers_that_float32_does_not_keep_are_refused(bad):
    """(a scale of 1e-60 would become the default one, a cap none)"""
    with pytest.raises(ValueError, match="sdpa_paged_int4"):
        call(**bad)


def test_windows_and_rows_above_32_bits_are_no_limit(monkeypatch):
    seen = []
    monkeypatch.setattr(paged.api, "kv4_attention", lambda *a: seen.append(a), raising=False)
    call(window=2 ** 32 + 5, max_rows=2 ** 32 + 1)                 # 5 and 1, cut to 32 bits
    call(window=2 ** 31 - 1, max_rows=2 ** 31 - 1)
    call(window=7, max_rows=3)
    got = [(a[22], a[16]) for a in seen]
    assert got == [(2 ** 31 - 1, 5), (2 ** 31 - 1, 5), (7, 3)]


def test_the_library_refuses_them_too():
    lib, p = _lib.load(), 1 << 20
    good = dict(q=p, q_ld=1024, kc=p, vc=p, out=p, o_ld=1024, pages=9, ps=16, table=p, slots=3, max_pages=4, seq=p, ctx=p, starts=None, seqs=5, tokens=5,
                max_rows=1, max_context=64, heads=8, kv=2, dim=128, scale=0.0, window=0, softcap=0.0, sinks=None, dtype=2, stream=None)
    for bad in (dict(scale=float("inf")), dict(scale=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(scale=2e38), dict(softcap=3e38)):
        assert lib.pgk_kv4_attention(*{**good, **bad}.values()) != 0, bad
        assert "kv4_attention failed" in _lib.last_error()


def test_an_array_is_there_twice_behind_one_without_bytes():
    x, none = arr((6, 4)), arr((6, 0))
    with pytest.raises(ValueError, match="twice"):
        ops.reorder_rows([none, x, x], arr((2, 3), int32))
    with pytest.raises(ValueError, match="twice"):
        ops.copy_rows([none, x, arr((6, 2)), x], arr((2,), int32), arr((2,), int32))


def test_a_model_refuses_a_cache_that_its_layers_do_not_read():
    m = LayeredCausalModel.__new__(LayeredCausalModel)
    m.cache = SimpleNamespace(int4=True, extend=None)              # nothing is appended before the refusal
    with pytest.raises(ValueError, match="four bits"):
        m.step_device([("a", [1, 2], [1])])
