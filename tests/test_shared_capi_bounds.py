"""The sizes that shared attention takes are those that decode_attention takes, but
for what a start costs (CPU; sizes only, no GPU work)."""

import ctypes

import pytest

from tests.test_kvcache_capi import I64, Pages, pages


@pytest.fixture(scope="module")
def lib():
    from jasper_amd import build_lib
    if not build_lib.LIB.exists():
        build_lib.build(verbose=False)
    lib = ctypes.CDLL(str(build_lib.LIB))
    lib.jasperx_shared_workspace.restype = I64
    lib.jasperx_shared_workspace.argtypes = [I64, I64, ctypes.POINTER(Pages), I64, I64]
    return lib


def test_a_batch_over_a_cache_of_a_million_tokens(lib):
    """256 sequences of 32 heads: a whole cache's tokens are what a GpuPagedCache without max_pages passes."""
    assert lib.jasperx_shared_workspace(256, 32, ctypes.byref(pages(heads=32)), 2 ** 20, 256) > 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,gh", [(1, 1), (1, 16), (1, 17), (8, 4), (32, 1), (2, 64), (1, 500), (128, 1)])
@pytest.mark.parametrize("batch", [1, 2, 37, 256, 512])
def test_it_takes_what_decode_takes(lib, dim, heads, gh, batch):
    p = pages(heads=heads, dim=dim)
    # the longest that decode_attention takes: a stream's tiles of 32 tokens and 2 for its start, below 2^31 in all
    longest = min(2 ** 31 - 1, 32 * ((2 ** 31 - 1) // (batch * heads * -(-gh // 16)) - 2))
    # a start: up to 8 + gh / 128 + 2 row tiles of 17 units, and 6 units more, of 32 tokens each
    start = 32 * ((10 + gh // 128) * 17 + 6)
    assert longest > start
    assert lib.jasperx_shared_workspace(batch, heads * gh, ctypes.byref(p), longest - start, 1) > 0
    if longest + 32 < 2 ** 31:
        assert lib.jasperx_shared_workspace(batch, heads * gh, ctypes.byref(p), longest + 32, 1) < 0
