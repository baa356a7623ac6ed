"""What the operators on the four-bit cache and of beam search refuse, and the format's own arithmetic: no GPU."""
import ctypes as C

import numpy as np
import pytest

from pygpukit_b200 import _lib, ops
from pygpukit_b200.core.array import GPUArray
from pygpukit_b200.core.dtypes import bfloat16, float16, float32, int32, int64, uint8
from tests import kv4_ref as ref


def arr(shape, dtype=float32):
    """an array that no call gets to read"""
    return GPUArray(shape, dtype, ptr=1 << 20)


def append(**kw):
    a = dict(q=arr((5, 8, 128), bfloat16), k=arr((5, 2, 128), bfloat16), v=arr((5, 2, 128), bfloat16), cos=arr((99, 128)), sin=arr((99, 128)),
             k_cache=arr((9, 2, 16, 72), uint8), v_cache=arr((9, 2, 16, 72), uint8), page_table=arr((3, 4), int32), slots=arr((5,), int32),
             positions=arr((5,), int32))
    a.update(kw)
    ops.rope_append_paged_int4(*a.values())


@pytest.mark.parametrize("bad", [
    dict(k=arr((5, 2, 128), uint8)), dict(k=arr((5, 256), bfloat16)), dict(v=arr((5, 2, 64), bfloat16)), dict(v=arr((5, 2, 128), float16)),
    dict(q=arr((4, 8, 128), bfloat16)), dict(q=arr((5, 8, 64), bfloat16)), dict(q=arr((5, 8, 128), float32)), dict(q=arr((5, 1024), bfloat16)),
    dict(cos=None), dict(sin=None), dict(cos=arr((99, 64))), dict(cos=arr((99, 128), bfloat16)), dict(cos=arr((99, 24)), sin=arr((99, 24))),
    dict(cos=arr((99, 144)), sin=arr((99, 144))), dict(cos=arr((0, 128)), sin=arr((0, 128))), dict(cos=arr((99, 0)), sin=arr((99, 0))),
    dict(k_cache=arr((9, 2, 16, 80), uint8)), dict(k_cache=arr((9, 4, 16, 72), uint8)), dict(k_cache=arr((9, 2, 16, 72), bfloat16)),
    dict(k_cache=arr((8, 2, 16, 72), uint8)), dict(k_cache=arr((9, 2, 24, 72), uint8), v_cache=arr((9, 2, 24, 72), uint8)),
    dict(k_cache=arr((9, 2, 0, 72), uint8), v_cache=arr((9, 2, 0, 72), uint8)), dict(k_cache=arr((9, 2 * 16 * 72), uint8)),
    dict(page_table=arr((12,), int32)), dict(page_table=arr((3, 4), int64)), dict(slots=arr((4,), int32)), dict(slots=arr((5,), int64)),
    dict(positions=arr((5, 1), int32)), dict(k=arr((5, 2, 80), bfloat16), v=arr((5, 2, 80), bfloat16), q=None),
], ids=str)
def test_append_refuses(bad):
    with pytest.raises(ValueError, match="rope_append_paged_int4|four bits"):
        append(**bad)


@pytest.mark.parametrize("bad", [dict(cache=arr((9, 2, 16, 70), uint8)), dict(cache=arr((9, 2, 72), uint8)), dict(cache=arr((9, 2, 16, 72))),
                                 dict(page_table=arr((3,), int32)), dict(slots=arr((5, 1), int32)), dict(positions=arr((6,), int32))], ids=str)
def test_read_refuses(bad):
    a = dict(cache=arr((9, 2, 16, 72), uint8), page_table=arr((3, 4), int32), slots=arr((5,), int32), positions=arr((5,), int32))
    a.update(bad)
    with pytest.raises(ValueError):
        ops.kv_read_paged_int4(*a.values(), out=arr((5, 2, 128), bfloat16))
    for out in (arr((5, 2, 64), bfloat16), arr((5, 2, 128), uint8)):
        with pytest.raises(ValueError):
            ops.kv_read_paged_int4(arr((9, 2, 16, 72), uint8), arr((3, 4), int32), arr((5,), int32), arr((5,), int32), out=out)


@pytest.mark.parametrize("bad", [
    dict(Q=arr((5, 8, 128), uint8)), dict(Q=arr((5, 1024), bfloat16)), dict(Q=arr((5, 7, 128), bfloat16), out=arr((5, 7, 128), bfloat16)),
    dict(out=arr((5, 8, 128), float32)), dict(out=arr((4, 8, 128), bfloat16)), dict(Q=arr((5, 8, 64), bfloat16), out=arr((5, 8, 64), bfloat16)),
    dict(k_cache=arr((9, 2, 16), uint8)), dict(v_cache=arr((9, 2, 32, 72), uint8)), dict(page_table=arr((3, 4), float32)), dict(slots=arr((4,), int32)),
    dict(slots=arr((5, 1), int32)), dict(context_lens=arr((5,), int64)), dict(max_context=-1), dict(max_context=65), dict(scale=-1.0), dict(scale=float("nan")),
    dict(row_starts=arr((5,), int32)), dict(row_starts=arr((6,), int32), max_rows=0), dict(max_rows=2), dict(window=-1), dict(softcap=-1.0),
    dict(softcap=float("nan")), dict(sinks=arr((7,))), dict(sinks=arr((8,), bfloat16)),
], ids=str)
def test_attention_refuses(bad):
    a = dict(Q=arr((5, 8, 128), bfloat16), k_cache=arr((9, 2, 16, 72), uint8), v_cache=arr((9, 2, 16, 72), uint8), out=arr((5, 8, 128), bfloat16),
             page_table=arr((3, 4), int32), slots=arr((5,), int32), context_lens=arr((5,), int32), max_context=64)
    a.update(bad)
    with pytest.raises(ValueError, match="sdpa_paged_int4"):
        ops.sdpa_paged_int4(**a)


@pytest.mark.parametrize("bad", [
    dict(logits=arr((6, 100), uint8)), dict(logits=arr((5, 100))), dict(logits=arr((600,))), dict(logits=arr((6, 0))), dict(scores=arr((6,))),
    dict(scores=arr((2, 3), bfloat16)), dict(scores=arr((2, 0)), logits=arr((0, 100))), dict(scores=arr((1, 65)), logits=arr((65, 100))), dict(n=0),
    dict(n=65), dict(n=7, logits=arr((6, 2))), dict(finished=arr((6,), int32)), dict(finished=arr((2, 3), uint8)),
    dict(finished=arr((2, 3), int32), pad_token=100), dict(finished=arr((2, 3), int32), pad_token=-1),
    dict(out=(arr((2, 3)), arr((2, 3), int32), arr((2, 4), int32))), dict(out=(arr((2, 3)), arr((2, 3)), arr((2, 3), int32))),
], ids=str)
def test_select_refuses(bad):
    a = dict(logits=arr((6, 100)), scores=arr((2, 3)))
    a.update(bad)
    with pytest.raises(ValueError, match="beam_select"):
        ops.beam_select(**a)


def test_rows_refuse():
    x = arr((6, 4))
    for parents in (arr((6,), int32), arr((2, 3), int64), arr((2, 2), int32), arr((1, 65), int32), arr((6, 0), int32)):
        with pytest.raises(ValueError, match="reorder_rows"):
            ops.reorder_rows([x], parents)
    for arrays in ([x, arr((5, 4))], [x, arr(())]):
        with pytest.raises(ValueError, match="reorder_rows"):
            ops.reorder_rows(arrays, arr((2, 3), int32))
    for call in (lambda a: ops.reorder_rows(a, arr((2, 3), int32)), lambda a: ops.copy_rows(a, arr((2,), int32), arr((2,), int32))):
        with pytest.raises(ValueError, match="twice"):              # its rows would move twice, at once
            call([x, arr((6, 2)), x])
    for src, dst in ((arr((3,), int64), arr((3,), int32)), (arr((3,), int32), arr((4,), int32)), (arr((3, 1), int32), arr((3, 1), int32))):
        with pytest.raises(ValueError, match="copy_rows"):
            ops.copy_rows([x], src, dst)


def test_the_library_refuses_what_the_operators_do():
    lib, p = _lib.load(), 1 << 20
    good = dict(q=p, k=p, v=p, q_ld=1024, k_ld=256, v_ld=256, cos=p, sin=p, rows=9, rot=128, pairs=0, kc=p, vc=p, pages=9, ps=16, table=p, slots=3, max_pages=4,
                row_slots=p, positions=p, tokens=5, heads=8, kv=2, dim=128, dtype=2, stream=None)
    for bad in (dict(dim=80), dict(dim=0), dict(ps=24), dict(ps=0), dict(ps=8192), dict(kc=p + 8), dict(vc=None), dict(table=None), dict(dtype=3), dict(rot=8),
                dict(rot=144), dict(rot=-16), dict(cos=None), dict(rows=0), dict(q_ld=1023), dict(k_ld=255), dict(q=None), dict(tokens=-1), dict(slots=0),
                dict(pages=0), dict(kv=0), dict(row_slots=None), dict(heads=65536, q_ld=65536 * 128), dict(max_pages=1 << 30)):
        assert lib.pgk_kv4_append(*{**good, **bad}.values()) != 0, bad
        assert "kv4_append failed" in _lib.last_error()
    assert lib.pgk_kv4_append(*{**good, "tokens": 0}.values()) == 0
    good = dict(q=p, q_ld=1024, kc=p, vc=p, out=p, o_ld=1024, pages=9, ps=16, table=p, slots=3, max_pages=4, seq=p, ctx=p, starts=None, seqs=5, tokens=5,
                max_rows=1, max_context=64, heads=8, kv=2, dim=128, scale=0.0, window=0, softcap=0.0, sinks=None, dtype=2, stream=None)
    for bad in (dict(dim=32), dict(ps=40), dict(q_ld=1000), dict(o_ld=1000), dict(heads=7), dict(heads=0), dict(max_rows=0), dict(max_rows=2), dict(seqs=6),
                dict(max_context=-1), dict(window=-1), dict(softcap=-1.0), dict(scale=float("nan")), dict(dtype=-1), dict(seq=None), dict(q=None),
                dict(starts=p, seqs=1 << 20, max_rows=1 << 12)):
        assert lib.pgk_kv4_attention(*{**good, **bad}.values()) != 0, bad
        assert "kv4_attention failed" in _lib.last_error()
    assert lib.pgk_kv4_attention(*{**good, "tokens": 0, "seqs": 0}.values()) == 0
    good = dict(x=p, ld=100, dtype=0, scores=p, finished=None, pad=0, groups=2, beams=3, vocab=100, n=6, s=p, b=p, t=p, stream=None)
    for bad in (dict(dtype=3), dict(beams=0), dict(beams=65), dict(n=0), dict(n=65), dict(ld=99), dict(vocab=0), dict(finished=p, pad=100), dict(groups=30000),
                dict(x=None), dict(t=None), dict(vocab=1, n=4), dict(vocab=4000000, ld=4000000)):
        assert lib.pgk_beam_select(*{**good, **bad}.values()) != 0, bad
        assert "beam_select failed" in _lib.last_error()
    assert lib.pgk_beam_select(*{**good, "groups": 0}.values()) == 0
    ptrs, sizes = (C.c_void_p * 2)(p, p), (C.c_int64 * 2)(64, 64)
    for bad in ((None, sizes, 2, 6, p, None, 6, 3), (ptrs, sizes, 2, 6, None, None, 6, 3), (ptrs, sizes, 2, 6, p, None, 6, 65), (ptrs, sizes, 2, 6, p, None, 6, 0),
                (ptrs, sizes, 2, 6, p, None, 7, 7), (ptrs, sizes, 2, 6, p, None, 5, 3), (ptrs, sizes, -1, 6, p, None, 6, 3),
                ((C.c_void_p * 2)(p, None), sizes, 2, 6, p, None, 6, 3), (ptrs, (C.c_int64 * 2)(64, -1), 2, 6, p, None, 6, 3)):
        assert lib.pgk_copy_rows(*bad, None) != 0, bad
        assert "copy_rows failed" in _lib.last_error()
    assert lib.pgk_copy_rows(None, None, 0, 0, None, None, 0, 1, None) == 0


def test_row_bytes():
    assert [ops.int4_row_bytes(d) for d in (64, 96, 128, 192, 256)] == [36, 54, 72, 108, 144]
    with pytest.raises(ValueError):
        ops.int4_row_bytes(80)


def test_the_format_is_within_its_steps_and_exact_in_bfloat16():
    """What a group stands for: zero is zero, no element is further off than a step, every value has eight significant bits."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((500, 128)) * 2.0 ** rng.integers(-20, 20, (500, 1)) + rng.standard_normal((500, 1))).astype(np.float32)
    x[:, 7] = 0.0
    words, groups = ref.encode(x)
    y = ref.decode(words, groups)
    scale = np.repeat(((groups.astype(np.uint32) & 0x7FF0) << 16).astype(np.uint32).view(np.float32).astype(np.float64), 32, -1)
    assert (np.abs(y - x) <= scale * (1 + 2.0 ** -20)).all() and (y[:, 7] == 0).all()
    assert np.array_equal(ref.floats(ref.rounded(y.astype(np.float32), "bfloat16"), "bfloat16").astype(np.float64), y)
    # most elements are within half a step: only those beside the group's ends are clipped
    assert (np.abs(y - x) <= 0.5001 * scale).mean() > 0.97
