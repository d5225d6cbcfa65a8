"""The C entry points of the paged cache refuse what their sizes do not allow,
before anything is computed from them (no GPU work)."""

import ctypes

import pytest


class Pages(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")]
                + [(n, ctypes.c_int64) for n in ("layer_stride", "page_stride", "head_stride", "row_stride")]
                + [(n, ctypes.c_int32) for n in ("layers", "pages", "heads", "page_size", "dim", "type")])


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("heads", ctypes.c_int64)]


I64, PTR = ctypes.c_int64, ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    from jasper_amd import build_lib
    if not build_lib.LIB.exists():
        build_lib.build(verbose=False)
    lib = ctypes.CDLL(str(build_lib.LIB))
    lib.jasper_last_error.restype = ctypes.c_char_p
    lib.jasperx_attention_workspace.restype = I64
    lib.jasperx_attention_workspace.argtypes = [I64, I64, ctypes.POINTER(Pages), I64, I64]
    lib.jasperx_retrieved_attention.restype = I64
    lib.jasperx_retrieved_attention.argtypes = (
        [ctypes.POINTER(Rows), ctypes.c_int32, I64, ctypes.POINTER(Pages), PTR, I64, I64, PTR, PTR, I64, I64, I64, I64,
         ctypes.c_double, PTR, PTR, PTR, I64, PTR])
    return lib


def pages(heads=8, dim=128):
    row = dim
    return Pages(layers=1, pages=4, heads=heads, page_size=16, dim=dim, type=0, row_stride=row, head_stride=16 * row,
                 page_stride=heads * 16 * row)


@pytest.mark.parametrize("lists", [1, 7, 9, 16, 31, 33, 64, 10 ** 12, 2 ** 63 - 1])
def test_workspace_refuses_lists_of_no_kind(lib, lists):
    """Lists are per query head (32) or per key head (8). More lists than query heads had ended the process."""
    assert lib.jasperx_attention_workspace(4, 32, ctypes.byref(pages()), 1000, lists) < 0
    assert b"lists must be" in lib.jasper_last_error()


@pytest.mark.parametrize("q_heads", [0, -8, 9, 65536, 2 ** 35])
def test_workspace_refuses_query_heads_that_the_calls_refuse(lib, q_heads):
    assert lib.jasperx_attention_workspace(4, q_heads, ctypes.byref(pages()), 1000, 8 if q_heads == 2 ** 35 else 0) < 0
    assert b"bad sizes" in lib.jasper_last_error()


BIG = 2 ** 63 - 1


@pytest.mark.parametrize("count,first,last", [
    (0, BIG, BIG), (2, BIG, BIG), (2 ** 31, BIG, 2 ** 63 - 2 ** 31), (BIG, 1, 0), (0, 2 ** 30, 0), (5, 0, 2 ** 62), (-1, 4, 4),
    (4, -1, 4), (4, 4, -1)])
def test_retrieved_refuses_sums_past_64_bits(lib, count, first, last):
    """The three numbers' sum counts a list's tokens; past 64 bits it wraps to a small one. (The addresses are never
    read: the call ends before.)"""
    somewhere = 4096
    p = pages()
    p.k = p.v = somewhere
    q = Rows(somewhere, 32 * 128, 128, 32)
    r = lib.jasperx_retrieved_attention(ctypes.byref(q), 0, 4, ctypes.byref(p), somewhere, 8, 8, somewhere, somewhere, 8,
                                        count, first, last, 1.0, somewhere, None, None, 0, None)
    assert r < 0 and b"first, last and count must be" in lib.jasper_last_error()


@pytest.mark.parametrize("tokens", [BIG, BIG - 6, BIG - 38, 2 ** 62])
def test_workspace_of_more_tokens_than_64_bits_round_up(lib, tokens):
    assert lib.jasperx_attention_workspace(4, 32, ctypes.byref(pages()), tokens, 0) < 0
    assert b"too large" in lib.jasper_last_error()
