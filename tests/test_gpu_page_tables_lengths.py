"""GPU tests that a GpuPagedCache's step reads what it stored, whatever max_len it was given."""

import pytest
import torch

from tests.test_gpu_kvcache import F16, randn
from tests.test_gpu_shared_attention import alike

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_len,stored", [(None, True), (20, True), (18, True), (17, True), (16, False), (0, False),
                                            (10 ** 6, True)])
def test_a_step_reads_all_that_it_stored(jasper, max_len, stored):
    heads, hq, dim, page = 2, 8, 64, 16
    cache = jasper.GpuPagedCache(40, 1, heads, dim, page_size=page, max_sequences=4, max_pages=5)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    step = cache.extend(ints([1, 2]), ints([20, 7]), 27, max_len=max_len)
    assert step.missing.item() == (0 if stored else -1)
    assert cache.length(1) == (20 if stored else 0)
    k, v = randn((27, heads, dim), F16, 1), randn((27, heads, dim), F16, 2)
    cache.append(0, step, None, k, v)
    q = randn((2, hq, dim), F16, 3, 2.0)
    got = cache.decode(0, step, q, return_lse=True)
    if not stored:
        assert (got[0] == 0).all()
        return
    full = cache.extend(ints([1, 2]), ints([0, 0]), 0)  # all that the tables have room for
    want = cache.decode(0, full, q, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    alike(cache.shared(0, step, q, cache.prefixes(step), return_lse=True), want, F16)
