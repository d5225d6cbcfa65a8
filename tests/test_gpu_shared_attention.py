"""GPU tests of attention where sequences share a prefix, against a plain
64-bit one sequence by sequence.

The bound of an output is decode_attention's (tests/test_gpu_kvcache.py) and,
as a prefix under more than 16 query rows has its weights rounded to their type
once, u_w sum p|v| more, with u_w half the distance of neighbours of that type
(bf16 2^-8, fp16 2^-11, which e4m3 caches use). fp16 weights are 2^12 and more
of the largest, so that their smallest step adds 2^-37 max|v| a token at most.
"""

import math

import pytest
import torch

from tests.test_gpu_kvcache import (BF16, F8, F16, UNIT, build_cache, check, f8_scales, make_pages, near, randn, raw,
                                    ref_attention)

pytestmark = pytest.mark.gpu


def build_shared(groups, heads, page, dim, cache, seed, layout="heads"):
    """groups: (shared, the members' lengths). A cache in which the members' first tables entries are the first long
    enough member's; in a page that is shared in part the others have other rows, which are not to be read."""
    lens = [n for _, members in groups for n in members]
    kp, vp, tables, keys, values = build_cache(lens, heads, page, dim, cache, seed, layout)
    starts, at = [0], 0
    for shared, members in groups:
        long = [at + i for i, n in enumerate(members) if n >= shared]
        for i in long[1:]:
            tables[i, :shared // page] = tables[long[0], :shared // page]
            for x in (keys, values):
                x[i][:, :shared] = x[long[0]][:, :shared]
        at += len(members)
        starts.append(at)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return kp, vp, tables, ints(lens), ints(starts), ints([s for s, _ in groups]), keys, values


def ref_shared(q, keys, values, scale, dtype, cache, ks=None, vs=None, choose=None):
    choose = choose or (lambda i, j: torch.arange(keys[i].size(1)))
    out, tol, lse, ltol = ref_attention(q, keys, values, scale, choose, dtype, ks, vs)
    size = ref_attention(q, keys, [v.abs() for v in values], scale, choose, dtype, ks, vs)[0]
    most = max([v.abs().max().item() for v in values if v.numel()] + [0.0]) * (1.0 if vs is None else vs.max().item())
    longest = max(k.size(1) for k in keys)
    weights = BF16 if cache == BF16 else F16
    return out, tol + 1.001 * UNIT[weights] * size + longest * 2.0 ** -37 * most, lse, ltol


MIXED = [(64, [64, 70, 133]), (40, [55]), (0, [9, 0, 31]), (500, [500, 501, 499, 520, 0, 530, 777, 501, 600]),
         (130, [130 + i % 7 * 11 for i in range(21)]), (1, [1, 2]), (33, [20, 32]), (257, [300, 400, 10])]


@pytest.mark.parametrize("hq,heads,dim,page,dtype,cache,layout", [
    (8, 2, 128, 16, F16, F16, "heads"), (8, 2, 128, 16, BF16, BF16, "rows"), (4, 4, 64, 32, F16, F16, "pair"),
    (16, 1, 96, 8, BF16, BF16, "heads"), (17, 1, 128, 16, F16, F16, "heads"), (34, 2, 128, 64, BF16, F8, "heads"),
    (3, 3, 80, 16, F16, F8, "rows"), (6, 2, 256, 16, F16, F16, "heads"), (40, 1, 256, 8, BF16, BF16, "rows"),
    (2, 1, 8, 128, F16, F16, "heads"), (6, 2, 200, 256, BF16, BF16, "heads"), (4, 2, 256, 32, F16, F8, "heads"),
    (2, 2, 16, 8, BF16, F8, "pair"), (8, 1, 72, 16, F16, F16, "rows"), (10, 2, 64, 8, BF16, F8, "heads")])
def test_groups_of_all_sizes(jasper, hq, heads, dim, page, dtype, cache, layout):
    kp, vp, tables, lens, groups, shared, keys, values = build_shared(MIXED, heads, page, dim, cache, 10, layout)
    ks, vs = f8_scales(heads, cache, 11)
    q = randn((lens.numel(), hq, dim), dtype, 12, 2.0)
    ref = ref_shared(q, keys, values, dim ** -0.5, dtype, cache, ks, vs)
    got = jasper.shared_attention(q, kp, vp, tables, lens, groups, shared, k_scale=ks, v_scale=vs, return_lse=True)
    check(got, ref)
    out = jasper.shared_attention(q, kp, vp, tables, lens, groups, shared, k_scale=ks, v_scale=vs, max_len=777)
    near(out, ref[0], ref[1])


@pytest.mark.parametrize("shared", [1, 7, 8, 31, 32, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 383, 449])
@pytest.mark.parametrize("dim,cache", [(64, F16), (128, BF16), (128, F8), (256, F16)])
def test_ends_of_tiles(jasper, shared, dim, cache):
    dtype = F16 if cache == F8 else cache
    groups = [(shared, [shared + i % 3 for i in range(9)])]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, 1, 8, dim, cache, 20)
    q = randn((9, 4, dim), dtype, 21, 2.0)
    scales = f8_scales(1, cache, 22)
    ref = ref_shared(q, keys, values, dim ** -0.5, dtype, cache, *scales)
    check(jasper.shared_attention(q, kp, vp, tables, lens, starts, both, k_scale=scales[0], v_scale=scales[1],
                                  return_lse=True), ref)


@pytest.mark.parametrize("sizes,hq,heads", [
    ([130], 2, 1),           # three row tiles, a team of three
    ([75, 75], 8, 1),        # five each
    ([140], 8, 1),           # nine, in two blocks
    ([150, 3, 40, 12], 8, 2),  # unlike groups: no team for all of them
    ([300], 64, 1),          # more rows than eight work-groups have
    ([600, 90], 4, 2)])      # more sequences than one launch has, a group cut by it
def test_many_rows(jasper, sizes, hq, heads):
    shared, page, dim = 150, 16, 64
    groups = [(shared, [shared + i % 5 for i in range(n)]) for n in sizes]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, heads, page, dim, F16, 30)
    q = randn((sum(sizes), hq, dim), F16, 31, 2.0)
    check(jasper.shared_attention(q, kp, vp, tables, lens, starts, both, return_lse=True),
          ref_shared(q, keys, values, dim ** -0.5, F16, F16))


@pytest.mark.parametrize("shared", [1, 63, 64, 500, 2100, 9000, 40_000])
@pytest.mark.parametrize("hq,heads,dim,dtype,cache", [(4, 2, 64, F16, F16), (8, 1, 128, BF16, F8), (2, 1, 256, BF16, BF16)])
def test_few_rows(jasper, shared, hq, heads, dim, dtype, cache):
    """Waves have more tiles of longer prefixes, work-groups fewer of them; a long stream beside short ones."""
    groups = [(shared, [shared + 3, shared]), (0, [5]), (shared // 2, [shared // 2 + 1, shared // 2 + 40])]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, heads, 16, dim, cache, 34)
    q = randn((5, hq, dim), dtype, 35, 2.0)
    got = jasper.shared_attention(q, kp, vp, tables, lens, starts, both, return_lse=True)
    check(got, ref_shared(q, keys, values, dim ** -0.5, dtype, cache))


def test_a_group_that_begins_before_the_batch(jasper):
    """It begins with the batch, however far before it is said to, in every launch."""
    groups = [(40, [40 + i % 3 for i in range(600)])]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, 1, 8, 16, F16, 32)
    q = randn((600, 2, 16), F16, 33, 2.0)
    want = jasper.shared_attention(q, kp, vp, tables, lens, starts, both, return_lse=True)
    for first in (-1, -(2 ** 31)):
        starts[0] = first
        got = jasper.shared_attention(q, kp, vp, tables, lens, starts, both, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def alike(got, want, dtype):
    """Two attentions of the same inputs, each within its bound of the same values."""
    a, b = got[0].double(), want[0].double()
    assert a.isfinite().all()
    assert (a - b).norm() <= 3 * UNIT[dtype] * b.norm()
    assert (got[1].double() - want[1].double()).abs().max() <= 1e-4


@pytest.mark.parametrize("dim,page,dtype,cache,batch,heads,shared", [
    (64, 8, F16, F16, 9, 16, 131_000), (128, 8, BF16, BF16, 6, 8, 140_001), (128, 16, BF16, F8, 5, 4, 200_000),
    (256, 8, F16, F16, 20, 2, 70_000), (64, 64, BF16, F8, 3, 2, 100_003)])
def test_long_prefixes(jasper, dim, page, dtype, cache, batch, heads, shared):
    """More pages than a work-group holds at once; many work-groups to a stream."""
    gh = 4
    pages = -(-shared // page) + batch * 3
    kp, vp = make_pages(pages, heads, page, dim, cache, seed=40)
    ks, vs = f8_scales(heads, cache, 41)
    whole = shared // page
    tables = torch.empty((batch, whole + 3), dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, device="cuda").int()
    tables[:, :whole] = order[:whole]
    tables[:, whole:] = order[whole:whole + batch * 3].view(batch, 3)
    lens = torch.full((batch,), whole * page, dtype=torch.int32, device="cuda") + torch.arange(batch, device="cuda").int()
    q = randn((batch, heads * gh, dim), dtype, 42, 2.0)
    groups = torch.tensor([0, batch], dtype=torch.int32, device="cuda")
    both = torch.tensor([whole * page], dtype=torch.int32, device="cuda")
    got = jasper.shared_attention(q, kp, vp, tables, lens, groups, both, k_scale=ks, v_scale=vs, return_lse=True)
    alike(got, jasper.decode_attention(q, kp, vp, tables, lens, k_scale=ks, v_scale=vs, return_lse=True), dtype)


@pytest.mark.parametrize("members,hq,cache", [(3, 4, F16), (12, 4, F16), (12, 4, BF16), (12, 4, F8)])
def test_pages_outside_are_left_out(jasper, members, hq, cache):
    dtype = BF16 if cache == BF16 else F16
    groups = [(200, [200 + 9 * i for i in range(members)])]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, 1, 16, 128, cache, 50)
    tables[0, 3], tables[0, 9] = -9, kp.size(0)  # the leader's: the prefix has holes
    tables[1, 12] = 2 ** 31 - 1                   # a member's own page
    kept = torch.cat([torch.arange(48), torch.arange(64, 144), torch.arange(160, 10 ** 4)])

    def choose(i, j):
        t = kept[kept < keys[i].size(1)]
        return t[(t < 200) | (t >= 208)] if i == 1 else t

    q = randn((members, hq, 128), dtype, 51, 2.0)
    scales = f8_scales(1, cache, 52)
    ref = ref_shared(q, keys, values, 128 ** -0.5, dtype, cache, *scales, choose=choose)
    check(jasper.shared_attention(q, kp, vp, tables, lens, starts, both, k_scale=scales[0], v_scale=scales[1],
                                  return_lse=True), ref)
    tables.fill_(-1)  # no pages at all
    out, lse = jasper.shared_attention(q, kp, vp, tables, lens, starts, both, k_scale=scales[0], v_scale=scales[1],
                                       return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 40.0])
@pytest.mark.parametrize("members", [4, 20])
def test_scales(jasper, scale, members):
    """40: scores of several thousand, of which the largest changes late."""
    groups = [(300, [300 + i for i in range(members)])]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, 2, 16, 64, BF16, 60)
    q = randn((members, 4, 64), BF16, 61, 2.0)
    check(jasper.shared_attention(q, kp, vp, tables, lens, starts, both, scale=scale, return_lse=True),
          ref_shared(q, keys, values, scale, BF16, BF16))


def test_rows_far_apart(jasper):
    """A page's rows so far apart that a tile's offsets pass 32 bits: seen through strides, on pages that overlap."""
    page, dim, heads, pages = 256, 64, 1, 3
    stride = 2 ** 23 + 64
    store = randn((stride * (page - 1) + pages * dim,), F16, 70)
    kp = store.as_strided((pages, heads, page, dim), (dim, dim, stride, 1))
    vp = kp
    lens = torch.tensor([600, 610, 640, 700, 768], dtype=torch.int32, device="cuda")
    tables = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda").expand(5, 3).contiguous()
    q = randn((5, 6, dim), F16, 71, 2.0)
    rows = kp[tables[0].long(), 0].reshape(768, dim).double().cpu()
    keys = [rows[:n][None] for n in lens.tolist()]
    starts = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    both = torch.tensor([600], dtype=torch.int32, device="cuda")
    check(jasper.shared_attention(q, kp, vp, tables, lens, starts, both, return_lse=True),
          ref_shared(q, keys, keys, dim ** -0.5, F16, F16))


def test_queries_and_tables_as_slices(jasper):
    groups = [(100, [110, 120, 130, 140, 150])]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, 2, 16, 64, F16, 80)
    fused = randn((5, 13, 64), F16, 81, 2.0)
    wide = torch.zeros((5, 40), dtype=torch.int32, device="cuda")
    wide[:, 3:3 + tables.size(1)] = tables
    q = fused[:, 2:10]
    ref = ref_shared(q, keys, values, 0.125, F16, F16)
    check(jasper.shared_attention(q, kp, vp, wide[:, 3:3 + tables.size(1)], lens, starts, both, return_lse=True), ref)
    odd = torch.empty(5 * 8 * 64 + 1, dtype=F16, device="cuda")[1:].view(5, 8, 64).copy_(q)
    check(jasper.shared_attention(odd, kp, vp, tables, lens, starts, both, return_lse=True), ref)


def test_without_groups_it_is_decode(jasper):
    lens = [5, 0, 900, 33]
    kp, vp, tables, keys, values = build_cache(lens, 2, 16, 128, F16, 90)
    q = randn((4, 8, 128), F16, 91, 2.0)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = ref_attention(q, keys, values, 128 ** -0.5, lambda i, j: torch.arange(lens[i]), F16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for groups, shared in (([0], []), ([0, 4], [0]), ([2, 2], [50]), ([0, 1, 2, 3, 4], [5, 0, 800, 33]), ([1, 3], [10]),
                           ([0, 4, 4, 4, 4], [0, 7, 7, 7])):
        check(jasper.shared_attention(q, kp, vp, tables, tens, ints(groups), ints(shared), return_lse=True), ref)
    out, lse = jasper.shared_attention(q[:0], kp, vp, tables[:0], tens[:0], ints([0]), ints([]), return_lse=True)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    empty = kp[:0], vp[:0]
    out, lse = jasper.shared_attention(q, *empty, tables, tens, ints([0, 4]), ints([3]), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_large_values_and_hostile_rows_behind_the_prefix(jasper):
    """bf16 values at fp32's end stay finite; what the last shared page holds past the prefix may be anything."""
    groups = [(70, [70] * 30)]
    kp, vp, tables, lens, starts, both, keys, values = build_shared(groups, 1, 16, 128, BF16, 100)
    vp[tables[0, :4].long()] = 2.0 ** 126
    for v in values:
        v[:, :64] = 2.0 ** 126
    last = tables[0, 4].item()
    raw(kp)[last, :, 6:], raw(vp)[last, :, 6:] = float("nan"), float("inf")
    q = randn((30, 2, 128), BF16, 101, 2.0)
    check(jasper.shared_attention(q, kp, vp, tables, lens, starts, both, return_lse=True),
          ref_shared(q, keys, values, 128 ** -0.5, BF16, BF16))


def test_offsets_past_32_bits(jasper):
    """More than 2^32 bytes of keys: the prefix and the own tokens at their far end."""
    heads, page, dim, members = 8, 64, 128, 6
    pages = 2 ** 32 // (heads * page * dim * 2) + 70
    kp = torch.zeros((pages, heads, page, dim), dtype=F16, device="cuda")
    vp = torch.zeros_like(kp)
    far = torch.arange(pages - 8, pages, dtype=torch.int32, device="cuda")
    for x, seed in ((kp, 110), (vp, 111)):
        x[far.long()] = randn((8, heads, page, dim), F16, seed)
    tables = torch.stack([torch.cat([far[[7, 1]], far[2 + i:3 + i]]) for i in range(members)])
    lens = torch.tensor([130 + i for i in range(members)], dtype=torch.int32, device="cuda")
    q = randn((members, 32, dim), F16, 112, 2.0)
    keys, values = ([x[t.long()].transpose(0, 1).reshape(heads, -1, dim)[:, :n].double().cpu()
                     for t, n in zip(tables, lens.tolist())] for x in (kp, vp))
    starts = torch.tensor([0, members], dtype=torch.int32, device="cuda")
    both = torch.tensor([128], dtype=torch.int32, device="cuda")
    check(jasper.shared_attention(q, kp, vp, tables, lens, starts, both, return_lse=True),
          ref_shared(q, keys, values, dim ** -0.5, F16, F16))


def test_repeats_streams_and_graphs_give_the_same_bits(jasper):
    kp, vp, tables, lens, groups, shared, _, _ = build_shared(MIXED, 2, 16, 128, BF16, 120)
    q = randn((lens.numel(), 8, 128), BF16, 121, 2.0)

    def call():
        return jasper.shared_attention(q, kp, vp, tables, lens, groups, shared, return_lse=True)

    want = [x.clone() for x in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        with torch.cuda.stream(side):
            got = call()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):  # two graphs with workspaces of their own
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for i in range(4):
        q.copy_(randn(q.shape, BF16, 122 + i, 2.0))
        lens.sub_(1).clamp_(min=0)  # some members are then too short for their prefix
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs[i % 2]]
        assert all(torch.equal(a, b) for a, b in zip(got, call())), i
        torch.cuda.synchronize()


def test_refusals(jasper):
    kp, vp = make_pages(8, 2, 16, 64, F16, seed=130)
    q = randn((2, 4, 64), F16, 131)
    tables = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    groups, shared = torch.tensor([0, 2], dtype=torch.int32, device="cuda"), lens[:1]
    f = jasper.shared_attention
    bad = [
        lambda: f(q, kp, vp, tables, lens, groups.long(), shared), lambda: f(q, kp, vp, tables, lens, groups, shared.long()),
        lambda: f(q, kp, vp, tables, lens, groups[:1], shared), lambda: f(q, kp, vp, tables, lens, groups, lens),
        lambda: f(q, kp, vp, tables, lens, torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: f(q, kp, vp, tables, lens, groups.cpu(), shared), lambda: f(q, kp, vp, tables, lens, groups, shared.cpu()),
        lambda: f(q, kp, vp, tables, lens, groups[None], shared), lambda: f(q, kp, vp, tables, lens, groups, shared, max_len=-1),
        lambda: f(q.float(), kp, vp, tables, lens, groups, shared), lambda: f(q[:, :3], kp, vp, tables, lens, groups, shared),
        lambda: f(q, kp, vp, tables.long(), lens, groups, shared), lambda: f(q, kp, vp, tables, lens.long(), groups, shared),
        lambda: f(q, kp, vp[:4], tables, lens, groups, shared),
        lambda: f(q.detach().requires_grad_(), kp, vp, tables, lens, groups, shared),
        lambda: f(q, kp, vp, tables, lens, groups, shared, k_scale=torch.ones(2, device="cuda")),
        lambda: f(q, kp[:, :, :12], vp[:, :, :12], tables, lens, groups, shared),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    torch.cuda.synchronize()


def test_forks_of_a_paged_cache(jasper):
    """What PagedCache's forks share is found, and attended to as decode does."""
    layers, heads, hq, dim = 2, 2, 8, 128
    cache = jasper.PagedCache(400, layers, heads, dim, dtype=BF16, max_sequences=40)
    a, b = cache.new(), cache.new()
    step = cache.extend([a, b], [777, 200])
    for layer in range(layers):
        k, v = randn((977, heads, dim), BF16, 140 + layer), randn((977, heads, dim), BF16, 150 + layer)
        cache.append(layer, step, None, k, v)
    seqs = [a] + [cache.fork(a) for _ in range(12)] + [b] + [cache.fork(b) for _ in range(3)]
    for n in (1, 5, 20):
        step = cache.extend(seqs, n)
        prefixes = cache.prefixes(step)
        assert prefixes[0].tolist() == [0, 13] + [17] * 16
        assert prefixes[1].tolist() == [768, 192] + [0] * 15
        tokens = n * len(seqs)
        for layer in range(layers):
            cache.append(layer, step, None, randn((tokens, heads, dim), BF16, 160 + layer),
                         randn((tokens, heads, dim), BF16, 170 + layer))
            q = randn((len(seqs), hq, dim), BF16, 180 + layer, 2.0)
            alike(cache.shared(layer, step, q, prefixes, return_lse=True), cache.decode(layer, step, q, return_lse=True), BF16)


def test_what_requires_a_gradient_or_has_no_memory_is_refused(jasper):
    kp, vp = make_pages(8, 2, 16, 64, F16, seed=190)
    q = randn((2, 4, 64), F16, 191)
    tables = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    lens = torch.full((2,), 20, dtype=torch.int32, device="cuda")
    groups, shared = torch.tensor([0, 2], dtype=torch.int32, device="cuda"), lens[:1].clone()
    for i in range(3):
        args = [q, kp, vp]
        args[i] = args[i].detach().clone().requires_grad_()
        with pytest.raises(ValueError):
            jasper.shared_attention(*args, tables, lens, groups, shared)
        with torch.no_grad():
            jasper.shared_attention(*args, tables, lens, groups, shared)
    torch.cuda.synchronize()
