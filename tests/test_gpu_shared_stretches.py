"""GPU tests of prefixes so long that a work-group reads more of them than it
holds pages of (1,024), where a page is longer than a tile of tokens, so that it
begins inside a page.

1,024 query rows of a key head are a team of eight work-groups, and 32 teams
share eight heads: each has about a quarter of a head's tokens, 70,000 to 150,000,
and all but the first of a head begin where they come to. The tables repeat the
pages of a small cache. Compared with decode_attention, which goes by a wave's
rows and holds no pages: 32 tokens read from elsewhere would be off by
(2 x 32 / prefix)^(1/2), 0.01 to 0.015 of the output's norm, against a bound of
3 x 2^-11.
"""

import pytest
import torch

from tests.test_gpu_kvcache import F8, F16, f8_scales, make_pages, randn
from tests.test_gpu_shared_attention import alike

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("outside", [(), (2000,), (37, 38, 1061, 1062, 1063, 3000)])
@pytest.mark.parametrize("dim,page,cache,prefix", [
    (256, 64, F16, 281_637), (256, 128, F16, 563_205), (128, 128, F16, 600_000), (256, 64, F8, 281_664),
    (256, 32, F16, 281_637)])
def test_stretches_that_begin_inside_a_page(jasper, dim, page, cache, prefix, outside):
    heads, gh, batch, pages = 8, 64, 16, 48
    kp, vp = make_pages(pages, heads, page, dim, cache, seed=60)
    ks, vs = f8_scales(heads, cache, 61)
    width = -(-prefix // page) + 1
    g = torch.Generator(device="cuda").manual_seed(62)
    table = torch.randint(0, pages, (width,), device="cuda", generator=g, dtype=torch.int32)
    for i, at in enumerate(outside):
        table[at] = (-1, pages, 2 ** 31 - 1)[i % 3]
    tables = table.expand(batch, width).contiguous()
    lens = prefix + torch.arange(batch, dtype=torch.int32, device="cuda") % 3
    q = randn((batch, heads * gh, dim), F16, 63, 2.0)
    groups = torch.tensor([0, batch], dtype=torch.int32, device="cuda")
    both = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    got = jasper.shared_attention(q, kp, vp, tables, lens, groups, both, k_scale=ks, v_scale=vs, return_lse=True)
    alike(got, jasper.decode_attention(q, kp, vp, tables, lens, k_scale=ks, v_scale=vs, return_lse=True), F16)


def test_tables_of_a_whole_cache_under_a_large_batch(jasper):
    """256 sequences of 32 heads whose tables have room for 2^20 tokens (refused before) are attended to as by decode."""
    batch, heads, page, dim = 256, 32, 16, 64
    kp, vp = make_pages(300, heads, page, dim, F16, seed=70)
    tables = torch.full((batch, 2 ** 20 // page), -1, dtype=torch.int32, device="cuda")
    own = torch.arange(batch, dtype=torch.int32, device="cuda")
    tables[:, :30] = torch.arange(260, 290, dtype=torch.int32, device="cuda")
    tables[:, 30] = own
    lens = 480 + own % 16
    q = randn((batch, heads, dim), F16, 71, 2.0)
    groups = torch.tensor([0, 10, 130, batch], dtype=torch.int32, device="cuda")
    both = torch.tensor([480, 33, 480], dtype=torch.int32, device="cuda")
    got = jasper.shared_attention(q, kp, vp, tables, lens, groups, both, return_lse=True)
    alike(got, jasper.decode_attention(q, kp, vp, tables, lens, return_lse=True), F16)
