"""GPU tests that attention over shared prefixes keeps decode_attention's bound
(tests/test_gpu_kvcache.py) under any number of query rows: the softmax weights
are held in two terms of their type, with an error below 2^-16 of a weight, and
the output is rounded once.

An element of the output then lies within half a step of its type, u |out|, and
2 e sum p|v| of the 64-bit value. Weights in one term are off by up to u_w of
themselves, u_w = 2^-8 (bf16) or 2^-11 (fp16, which e4m3 caches use); where few
tokens have most of the weight that is as much as the output's own rounding, and
takes outputs that lie near the middle of two neighbours over the bound.
"""

import pytest
import torch

from tests.test_gpu_kvcache import BF16, F8, F16, check, f8_scales, randn, ref_attention
from tests.test_gpu_shared_attention import build_shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,dtype,cache", [
    (64, F16, F16), (64, BF16, BF16), (64, F16, F8), (64, BF16, F8), (128, F16, F16), (128, BF16, BF16), (128, F16, F8),
    (128, BF16, F8), (96, BF16, BF16), (256, F16, F16), (256, BF16, BF16), (256, F16, F8), (200, BF16, BF16)])
@pytest.mark.parametrize("members,hq,heads,shared", [(17, 1, 1, 5), (9, 8, 2, 77), (40, 8, 1, 700)])
def test_wide_prefixes_are_as_exact_as_decode(jasper, dim, dtype, cache, members, hq, heads, shared):
    groups = [(shared, [shared + i % 4 for i in range(members)])]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, heads, 16, dim, cache, 10)
    q = randn((members, hq, dim), dtype, 11, 2.0)
    ks, vs = f8_scales(heads, cache, 12)
    ref = ref_attention(q, keys, values, dim ** -0.5, lambda i, j: torch.arange(keys[i].size(1)), dtype, ks, vs)
    check(jasper.shared_attention(q, kp, vp, tables, lens, starts, both, k_scale=ks, v_scale=vs, return_lse=True), ref)
