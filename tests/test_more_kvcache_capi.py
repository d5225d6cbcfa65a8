"""The C entry points of shared prefixes, page tables on the GPU and positions
of several axes refuse what their sizes do not allow (no GPU work; addresses
are never read)."""

import ctypes

import pytest

from tests.test_kvcache_capi import BIG, I64, PTR, Pages, Rows, pages

I32 = ctypes.c_int32


class Table(ctypes.Structure):
    _fields_ = ([(n, PTR) for n in ("tables", "lens", "refs", "free_bits")]
                + [(n, I32) for n in ("sequences", "width", "pages", "page_size")])


SOMEWHERE = 4096


def table(sequences=4, width=8, pages=100, page_size=16, at=SOMEWHERE):
    return Table(at, at, at, at, sequences, width, pages, page_size)


@pytest.fixture(scope="module")
def lib():
    from jasper_amd import build_lib
    if not build_lib.LIB.exists():
        build_lib.build(verbose=False)
    lib = ctypes.CDLL(str(build_lib.LIB))
    lib.jasper_last_error.restype = ctypes.c_char_p
    for name, args in {
        "extend_tables": [ctypes.POINTER(Table), PTR, PTR, I64, I64, I64] + [PTR] * 9 + [I64, PTR],
        "extend_workspace": [I64, I64],
        "truncate_tables": [ctypes.POINTER(Table), PTR, PTR, I64, PTR],
        "fork_tables": [ctypes.POINTER(Table), PTR, PTR, I64, PTR],
        "shared_prefixes": [PTR, I64, I64, PTR, I64, I64, I64, PTR, PTR, PTR, I64, PTR],
        "prefixes_workspace": [I64],
        "shared_workspace": [I64, I64, ctypes.POINTER(Pages), I64, I64],
        "shared_attention": [ctypes.POINTER(Rows), I32, I64, ctypes.POINTER(Pages), PTR, I64, I64, PTR, I64, PTR, PTR, I64,
                             ctypes.c_double, PTR, PTR, PTR, I64, PTR],
        "rotary_by_axes": [ctypes.POINTER(Rows), ctypes.POINTER(Rows), I32, I64, I64, PTR, I32, PTR, I32, I32, PTR, PTR,
                           I64, I64, ctypes.c_uint32, PTR, PTR, PTR],
    }.items():
        f = getattr(lib, "jasperx_" + name)
        f.restype, f.argtypes = I64, args
    return lib


def refused(lib, result, text):
    assert result < 0 and text in lib.jasper_last_error().decode(), lib.jasper_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(page_size=0), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=512), "page_size"),
    (dict(sequences=-1), "at least 0"), (dict(pages=-5), "at least 0"), (dict(width=2 ** 28), "below 2^31"),
    (dict(at=None), "null")])
def test_page_tables_of_no_kind(lib, change, text):
    t = table(**change)
    x = SOMEWHERE
    refused(lib, lib.jasperx_extend_tables(ctypes.byref(t), x, x, 3, 5, 8, *[x] * 9, 2 ** 30, None), text)
    refused(lib, lib.jasperx_truncate_tables(ctypes.byref(t), x, x, 3, None), text)
    refused(lib, lib.jasperx_fork_tables(ctypes.byref(t), x, x, 3, None), text)


def test_extend_refuses(lib):
    t, x = table(), SOMEWHERE
    call = lambda n=3, tokens=5, width=8, at=x, bytes=2 ** 30: lib.jasperx_extend_tables(  # noqa: E731
        ctypes.byref(t), x, x, n, tokens, width, *[x] * 8, at, bytes, None)
    refused(lib, call(n=65536), "must be 0 to 65535")
    refused(lib, call(n=-1), "must be 0 to 65535")
    refused(lib, call(tokens=-1), "at least 0")
    refused(lib, call(tokens=2 ** 31), "too large")
    refused(lib, call(width=-1), "at least 0")
    refused(lib, call(width=2 ** 28), "below 2^31")
    refused(lib, call(width=BIG), "below 2^31")
    refused(lib, call(bytes=64), "workspace must")
    refused(lib, call(at=x + 4), "workspace must")
    refused(lib, lib.jasperx_extend_tables(None, x, x, 3, 5, 8, *[x] * 9, 2 ** 30, None), "null")
    many = table(sequences=2 ** 18 + 1)
    refused(lib, lib.jasperx_extend_tables(ctypes.byref(many), x, x, 3, 5, 8, *[x] * 9, 2 ** 30, None), "too large")
    refused(lib, lib.jasperx_truncate_tables(ctypes.byref(t), x, x, 65536, None), "must be 0 to 65535")
    refused(lib, lib.jasperx_fork_tables(ctypes.byref(t), x, x, -3, None), "must be 0 to 65535")


@pytest.mark.parametrize("n,count", [(-1, 5), (65536, 5), (5, -1), (5, 2 ** 31), (BIG, BIG)])
def test_extend_workspace_refuses(lib, n, count):
    refused(lib, lib.jasperx_extend_workspace(n, count), "must be")


def test_prefixes_refuse(lib):
    x = SOMEWHERE
    call = lambda width=8, batch=4, page=16, least=1, at=x, bytes=64: lib.jasperx_shared_prefixes(  # noqa: E731
        at, 8, width, at, batch, page, least, x, x, x, bytes, None)
    refused(lib, call(page=12), "page_size")
    refused(lib, call(width=-1), "below 2^31")
    refused(lib, call(width=2 ** 27), "below 2^31")
    refused(lib, call(least=-1), "least")
    refused(lib, call(at=None), "null")
    refused(lib, call(batch=65536), "must be 0 to 65535")
    refused(lib, call(bytes=8), "workspace must")
    refused(lib, lib.jasperx_prefixes_workspace(-1), "must be 0 to 65535")


def test_shared_attention_refuses(lib):
    x, p = SOMEWHERE, pages()
    p.k = p.v = x
    q = Rows(x, 32 * 128, 128, 32)
    call = lambda batch=4, max_len=128, groups=1, at=x, bytes=2 ** 40, ws=x: lib.jasperx_shared_attention(  # noqa: E731
        ctypes.byref(q), 0, batch, ctypes.byref(p), x, 8, 8, x, max_len, at, at, groups, 1.0, x, None, ws, bytes, None)
    refused(lib, call(groups=5), "groups must be")
    refused(lib, call(groups=-1), "groups must be")
    refused(lib, call(max_len=-1), "max_len must be")
    refused(lib, call(max_len=2 ** 31), "max_len must be")
    refused(lib, call(at=None), "null")
    refused(lib, call(batch=65536, groups=1), "batch must be")
    refused(lib, call(bytes=100), "workspace must")
    refused(lib, call(ws=x + 8), "workspace must")
    refused(lib, call(ws=None), "workspace must")


@pytest.mark.parametrize("batch,q_heads,max_len,groups", [
    (-1, 32, 100, 0), (65536, 32, 100, 0), (4, 0, 100, 1), (4, 33, 100, 1), (4, 65536, 100, 1), (4, 32, -1, 1),
    (4, 32, 2 ** 31, 1), (4, 32, 100, 5), (4, 32, 100, -1), (512, 32, 2 ** 31 - 1, 1)])
def test_shared_workspace_refuses(lib, batch, q_heads, max_len, groups):
    refused(lib, lib.jasperx_shared_workspace(batch, q_heads, ctypes.byref(pages()), max_len, groups), "too large")


def test_shared_workspace_refuses_more_rows_than_a_launch_joins(lib):
    p = pages()
    p.heads = 1
    most = (2 ** 32 - 1) // (512 * 256)  # rows of a launch have 256 threads each
    assert lib.jasperx_shared_workspace(512, most, ctypes.byref(p), 100, 1) > 0
    refused(lib, lib.jasperx_shared_workspace(512, most + 1, ctypes.byref(p), 100, 1), "too large")


def test_workspaces_that_are_given(lib):
    assert lib.jasperx_shared_workspace(0, 32, ctypes.byref(pages()), 100, 0) == 0
    assert lib.jasperx_shared_workspace(64, 32, ctypes.byref(pages()), 2 ** 20, 1) > 0
    assert lib.jasperx_extend_workspace(0, 0) == 0
    assert lib.jasperx_extend_workspace(10, 1000) >= 4 * 1000


@pytest.mark.parametrize("sections,n", [((10, 10, 11), 3), ((-1, 33, 0), 3), ((32, 0, 0), 0), ((8, 8, 8, 8), 5), ((32, 0), -1),
                                        ((2 ** 31 - 1, 2 ** 31 - 1, 34), 3), (None, 3)])
def test_rotary_refuses_sections(lib, sections, n):
    x = SOMEWHERE
    q = Rows(x, 64, 64, 1)
    s = (I32 * 5)(*(sections or ())) if sections else None
    r = lib.jasperx_rotary_by_axes(ctypes.byref(q), None, 0, 4, 64, x, 8, s, n, 0, x, x, 10, 64, 0, x, None, None)
    assert r < 0 and b"axes" in lib.jasper_last_error()
