"""GPU tests of the paged cache's operators against plain 64-bit ones.

Tolerances come from the arithmetic, per output value:

- rotary: two products and a sum in 32 bits (3 half-ulps of 2^-24 of the
  products' sizes), then one rounding to the type: half the distance of
  neighbours, u = 2^-(stored bits + 1) of the value (fp16 2^-11, bf16 2^-8,
  e4m3 2^-4), or half the type's smallest step.
- attention: a score is dim products summed in 32 bits in any order, error at
  most (dim + 4) 2^-24 scale sum|q||k| plus 2^-22 of its distance from the
  maximum (exponential); a weight is held in two terms of the type (error
  below 2^-16), sums over T tokens add (T + 64) 2^-24. The weights' relative
  error e counts twice (numerator, denominator):
  |out error| <= u |out| + 2 e sum p|v|, |lse error| <= e + 2^-22 |lse|.
"""

import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F8: 2.0 ** -4}
STEP = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F8: 2.0 ** -10}  # half the smallest step


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g) * scale
    return x.to(dtype)


def raw(x):
    return x.view(torch.uint8) if x.dtype == F8 else x


def near(got, want, tol, what=""):
    got, want, tol = got.double().cpu(), want.cpu(), tol.cpu()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), what
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]), what
    off = (got - want)[fine].abs() - tol[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: over the bound by {off.max().item():.3g}"


# ---- rotary ----

def ref_rotary(x, positions, cos, sin, interleaved, back=False):
    """(value, size of the sums) in 64 bits on the CPU."""
    x, positions = x.double().cpu(), positions.cpu().long()
    c, s = cos.double().cpu()[positions][..., None, :], sin.double().cpu()[positions][..., None, :]
    if back:
        s = -s
    rot = 2 * cos.size(1)
    y, size = x.clone(), torch.zeros_like(x)
    half = rot // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        ci, si = c[..., i], s[..., i]
        y[..., a] = x[..., a] * ci - x[..., b] * si
        y[..., b] = x[..., b] * ci + x[..., a] * si
        size[..., a] = (x[..., a] * ci).abs() + (x[..., b] * si).abs()
        size[..., b] = (x[..., b] * ci).abs() + (x[..., a] * si).abs()
    return y, size


def rotary_tol(want, size, dtype):
    return UNIT[dtype] * 1.001 * want.abs() + 3 * 2.0 ** -24 * size + STEP[dtype]


@pytest.mark.parametrize("n,hq,hk,dim,rot,interleaved,dtype", [
    (1, 1, 1, 2, 2, False, F16), (1, 8, 2, 64, 64, True, BF16), (7, 3, 3, 80, 40, False, F16),
    (5, 2, 1, 80, 80, True, BF16), (33, 12, 4, 96, 48, True, F16), (130, 32, 8, 128, 128, False, BF16),
    (1500, 5, 5, 128, 64, False, F16), (2049, 4, 1, 256, 256, True, BF16), (1100, 2, 1, 10, 6, False, F16),
    (3, 1, 0, 34, 34, False, BF16), (6, 64, 8, 256, 96, False, F16)])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_rotary_values(jasper, n, hq, hk, dim, rot, interleaved, dtype, idx):
    cos, sin = jasper.rotary_table(5000, rot)
    q = randn((n, hq, dim), dtype, 1)
    k = randn((n, hk, dim), dtype, 2) if hk else None
    pos = torch.randint(0, 5000, (n,), device="cuda", dtype=idx)
    out = jasper.rotary(q, k, pos, cos, sin, interleaved=interleaved)
    for x, y in ((q, out[0]), (k, out[1])):
        if x is None:
            assert y is None
            continue
        want, size = ref_rotary(x, pos, cos, sin, interleaved)
        near(y, want, rotary_tol(want, size, dtype))
        assert torch.equal(y[..., rot:], x[..., rot:])


def test_rotary_shapes_strides_and_alignment(jasper):
    cos, sin = jasper.rotary_table(64, 64)
    pos = torch.arange(24, device="cuda").view(2, 12) * 2
    fused = randn((2, 12, 6, 65), F16, 3)
    q, k = fused[:, :, :4, 1:], fused[:, :, 4:, 1:]  # odd addresses and strides
    a, b = jasper.rotary(q, k, pos, cos, sin)
    c, d = jasper.rotary(q.contiguous(), k.contiguous(), pos, cos, sin)
    assert torch.equal(a, c) and torch.equal(b, d) and a.shape == q.shape
    t, _ = jasper.rotary(q.transpose(0, 1), None, pos.t(), cos, sin)
    assert torch.equal(t, a.transpose(0, 1))
    flipped = torch.stack([q[..., i] for i in range(64)], dim=0).permute(1, 2, 3, 0)  # values apart
    assert torch.equal(jasper.rotary(flipped, None, pos, cos, sin)[0], a)
    one, _ = jasper.rotary(q[0, 5], None, pos[0, 5], cos, sin)  # no leading size at all
    assert torch.equal(one, a[0, 5])
    none, _ = jasper.rotary(q[:0], None, pos[:0], cos, sin)
    assert none.shape == (0, 12, 4, 64)


def test_rotary_position_outside_the_tables(jasper):
    cos, sin = jasper.rotary_table(10, 32)
    q = randn((4, 2, 48), BF16, 4)
    y, _ = jasper.rotary(q, None, torch.tensor([0, 10, -1, 9], device="cuda"), cos, sin)
    assert y[1:3, :, :32].isnan().all() and y[[0, 3]].isfinite().all() and torch.equal(y[..., 32:], q[..., 32:])


def rotary_needs_no_graph(jasper, q, k, pos, cos, sin):
    with torch.no_grad():
        return any(x.requires_grad for x in jasper.rotary(q, k, pos, cos, sin))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot,scaling", [(64, 64, None), (96, 48, "yarn"), (128, 128, "ntk"), (20, 12, "linear")])
def test_rotary_gradient(jasper, dim, rot, scaling, interleaved):
    cos, sin = jasper.rotary_table(300, rot, scaling=scaling, factor=4.0 if scaling else 1.0, original=64)
    n = 37
    pos = torch.randint(0, 300, (n,), device="cuda")
    q = randn((n, 6, dim), F16, 5).requires_grad_()
    k = randn((n, 2, dim), F16, 6).requires_grad_()
    gq, gk = randn((n, 6, dim), F16, 7), randn((n, 2, dim), F16, 8)
    out = jasper.rotary(q, k, pos, cos, sin, interleaved=interleaved)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk), retain_graph=True)
    assert not rotary_needs_no_graph(jasper, q, k, pos, cos, sin)
    for g, d in ((gq, dq), (gk, dk)):
        want, size = ref_rotary(g, pos, cos, sin, interleaved, back=True)
        near(d, want, rotary_tol(want, size, F16))
    # differences: the map is linear, so a step of any size is exact but for rounding
    for at in range(0, dim, 5):
        step = torch.zeros_like(q)
        step[..., at] = 1.0
        up, _ = jasper.rotary((q + step).detach(), None, pos, cos, sin, interleaved=interleaved)
        dn, _ = jasper.rotary((q - step).detach(), None, pos, cos, sin, interleaved=interleaved)
        slope = ((up.double() - dn.double()) / 2 * gq.double()).sum(-1)
        # q +- 1 and the outputs are each rounded to fp16 (values below 8): 2^-8 each, over up to dim terms of |g|
        tol = 4 * 2.0 ** -8 * gq.double().abs().sum(-1)
        near(dq[..., at], slope.cpu(), tol)
    only, = torch.autograd.grad(out, (k,), (gq, gk), retain_graph=True)
    assert torch.equal(only, dk)
    again, _ = jasper.rotary(q, None, pos, cos, sin, interleaved=interleaved)
    assert torch.equal(torch.autograd.grad(again, q, gq)[0], dq)
    # the gradient is linear in gq: differentiated once more it is the rotation itself
    seed = gq.clone().requires_grad_()
    first, = torch.autograd.grad(out[0], q, seed, create_graph=True)
    other = randn((n, 6, dim), F16, 9)
    second, = torch.autograd.grad(first, seed, other)
    want, size = ref_rotary(other, pos, cos, sin, interleaved)
    near(second, want, rotary_tol(want, size, F16))


# ---- appending ----

def make_pages(pages, heads, page, dim, cache, seed=None, layout="heads"):
    """A pair of page tensors; layout rows: [n, page, heads, dim] seen with the heads first; pair: K beside V."""
    if layout == "rows":
        shape = (pages, page, heads, dim)
    elif layout == "pair":
        shape = (pages, 2, heads, page, dim)
    else:
        shape = (pages, heads, page, dim)
    scale = 32.0 if cache == F8 else 1.0
    out = []
    for i in range(1 if layout == "pair" else 2):
        out.append(torch.zeros(shape, dtype=cache, device="cuda") if seed is None
                   else randn(shape, cache, seed + i, scale))
    if layout == "rows":
        return [x.transpose(1, 2) for x in out]
    return [out[0][:, 0], out[0][:, 1]] if layout == "pair" else out


@pytest.mark.parametrize("n,hq,heads,dim,rot,interleaved,dtype,cache,page,layout", [
    (1, 8, 2, 64, 64, False, F16, F16, 8, "heads"), (1, 32, 8, 128, 128, False, BF16, BF16, 16, "rows"),
    (45, 5, 5, 80, 40, True, F16, F16, 16, "pair"), (300, 16, 2, 128, 64, False, BF16, F8, 32, "heads"),
    (2000, 4, 4, 96, 96, True, F16, F8, 64, "rows"), (70, 2, 1, 256, 256, False, F16, F16, 256, "heads"),
    (33, 0, 3, 128, 0, False, BF16, BF16, 16, "heads"), (19, 1, 1, 8, 6, False, F16, F16, 8, "heads"),
    (1030, 10, 10, 64, 62, False, BF16, F8, 16, "heads")])
def test_append_tokens(jasper, n, hq, heads, dim, rot, interleaved, dtype, cache, page, layout):
    pages = -(-n // page) + 3
    kp, vp = make_pages(pages, heads, page, dim, cache, layout=layout)
    qkv = randn((n, hq + 2 * heads, dim), dtype, 11)
    q, k, v = qkv.split([hq, heads, heads], dim=1)
    cos, sin = jasper.rotary_table(4096, rot) if rot else (None, None)
    pos = torch.randint(0, 4096, (n,), device="cuda") if rot else None
    slots = torch.randperm(pages * page, device="cuda")[:n]
    skipped = torch.zeros(n, dtype=torch.bool)
    if n > 10:
        slots[3], slots[7], slots[9] = -1, pages * page, -2 ** 40
        skipped[[3, 7, 9]] = True
    ks = vs = None
    if cache == F8:
        ks, vs = torch.rand(heads, device="cuda") * 0.01 + 0.004, torch.rand(heads, device="cuda") * 0.02 + 0.02
        ks[0] = 0.001  # values over 448 scales saturate
    out = jasper.append_tokens(q if hq else None, k, v, pos, slots, cos, sin, kp, vp, interleaved=interleaved,
                               k_scale=ks, v_scale=vs)
    if hq:
        want, size = ref_rotary(q, pos, cos, sin, interleaved) if rot else (q.double().cpu(), torch.zeros(1))
        near(out, want, rotary_tol(want, size, dtype))
    else:
        assert out is None
    kept = (~skipped).nonzero()[:, 0]
    at = slots.cpu()[kept]
    for store, x, scale, turned in ((kp, k, ks, bool(rot)), (vp, v, vs, False)):
        want, size = ref_rotary(x, pos, cos, sin, interleaved) if turned else (x.double().cpu(), torch.zeros(x.shape))
        if scale is not None:
            f = scale.double().cpu()[None, :, None]
            want, size = (want / f).clamp(-448, 448), size / f
            size = size + want.abs()  # the division rounds too
        tol = rotary_tol(want, size, cache)
        full = torch.zeros((pages, page, heads, dim), dtype=torch.float64)
        bound = torch.zeros_like(full)
        full[at // page, at % page] = want.expand(x.shape)[kept]
        bound[at // page, at % page] = tol.expand(x.shape)[kept]
        near(store.float().transpose(1, 2), full, bound)  # every other row is still zero


def test_append_e4m3_rounds_like_torch(jasper):
    """Every fp16 value, through an e4m3 cache without a scale."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).cuda().view(F16)
    k = bits.view(256, 1, 256)
    kp, vp = make_pages(32, 1, 8, 256, F8)
    jasper.append_tokens(None, k, k, None, torch.arange(256, device="cuda"), None, None, kp, vp)
    want = k.float().clamp(-448, 448).to(F8).float().view(-1)
    for store in (kp, vp):
        got = store.float().view(-1)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~got.isnan()], want[~got.isnan()])


# ---- pages ----

@pytest.mark.parametrize("cache", [F16, F8])
@pytest.mark.parametrize("layers,heads,page,dim,layout", [
    (1, 1, 8, 16, "heads"), (3, 2, 16, 80, "heads"), (2, 8, 16, 128, "rows"), (1, 5, 32, 96, "pair"), (32, 4, 64, 64, "heads")])
def test_copy_pages(jasper, cache, layers, heads, page, dim, layout):
    pages = 40
    pair = [make_pages(pages, heads, page, dim, cache, seed=20 + 2 * i, layout=layout) for i in range(layers)]
    if layout == "pair" or layers == 1:
        kp, vp = pair[0]
    else:
        kp, vp = (torch.stack([x[j] for x in pair]) for j in range(2))
        if layout == "rows":
            kp, vp = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (kp, vp))
    src = torch.tensor([3, 7, 3, 39, 50, 0, -1], dtype=torch.int32, device="cuda")
    dst = torch.tensor([4, 0, 9, 38, 1, -1, 2], dtype=torch.int32, device="cuda")
    want = []
    for x in (kp, vp):
        w = raw(x).clone()
        dim_of = x.ndim - 4
        for s, d in ((3, 4), (7, 0), (3, 9), (39, 38)):
            w.select(dim_of, d).copy_(raw(x).select(dim_of, s))
        want.append(w)
    jasper.copy_pages(kp, vp, src, dst)
    assert torch.equal(raw(kp), want[0]) and torch.equal(raw(vp), want[1])
    jasper.copy_pages(kp, vp, src[:0], dst[:0])
    assert torch.equal(raw(kp), want[0])


@pytest.mark.parametrize("moves,sequences,width", [(1, 1, 1), (513, 5, 77), (1025, 64, 130), (2500, 300, 33)])
@pytest.mark.parametrize("heads,page,dim", [(1, 8, 16), (3, 8, 40), (2, 64, 64)])
def test_copy_pages_moves_tables(jasper, moves, sequences, width, heads, page, dim):
    pages = 2 * moves + 100
    kp, vp = make_pages(pages, heads, page, dim, F16, seed=30)
    before = kp.clone()
    order = torch.randperm(pages)
    src, dst = order[:moves].int(), order[moves:2 * moves].int()
    owned = torch.cat([order[:moves], order[2 * moves:]])
    tables = owned[torch.randint(0, owned.numel(), (sequences, width))].int()
    tables[torch.rand(tables.shape) < 0.2] = -1
    to = torch.arange(pages).int()
    to[src.long()] = dst
    want = torch.where(tables < 0, tables, to[tables.clamp(min=0).long()])
    got = tables.cuda()
    jasper.copy_pages(kp, vp, src.cuda(), dst.cuda(), tables=got)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(kp[dst.long().cuda()], before[src.long().cuda()])


# ---- attention ----

def build_cache(lens, heads, page, dim, cache, seed, layout="heads", spare=3, hostile=True):
    """(k_pages, v_pages, tables, keys, values): pages in random order, and whatever no sequence owns is NaN or
    infinite; table entries past a sequence's pages are wild."""
    count = [-(-max(0, n) // page) for n in lens]
    pages = sum(count) + spare
    kp, vp = make_pages(pages, heads, page, dim, cache, seed=seed, layout=layout)
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g)
    tables = torch.randint(-5, 10 ** 6, (len(lens), max(count) + 2), dtype=torch.int32, generator=g)
    if hostile:
        tables[:, -1] = -2 ** 31
    owned = torch.zeros((pages, page), dtype=torch.bool)
    at, keys, values = 0, [], []
    for i, (n, c) in enumerate(zip(lens, count)):
        mine = order[at:at + c]
        at += c
        tables[i, :c] = mine.int()
        rows = torch.arange(max(0, n))
        owned[mine[rows // page], rows % page] = True
        keys.append(kp.float()[mine.cuda()].transpose(0, 1).reshape(heads, c * page, dim)[:, :max(0, n)].double().cpu())
        values.append(vp.float()[mine.cuda()].transpose(0, 1).reshape(heads, c * page, dim)[:, :max(0, n)].double().cpu())
    if hostile:
        free = (~owned).cuda()
        for x in (kp, vp):
            view = raw(x).transpose(1, 2)  # [pages, page, heads, dim]
            junk = 0x7F if cache == F8 else float("nan")
            view[free] = junk
            if cache != F8:
                view[free & (torch.arange(page, device="cuda") % 2 == 0)] = float("inf")
    return kp, vp, tables.cuda(), keys, values


def ref_attention(q, keys, values, scale, choose, dtype, k_scale=None, v_scale=None, lists=None):
    """Per sequence and list of query heads, in 64 bits: (out, its bound, lse, its bound)."""
    b, hq, dim = q.shape
    heads = keys[0].size(0)
    lists = lists or heads
    out, tol = torch.zeros((b, hq, dim), dtype=torch.float64), torch.zeros((b, hq, dim), dtype=torch.float64)
    lse, ltol = torch.full((b, hq), -math.inf, dtype=torch.float64), torch.zeros((b, hq), dtype=torch.float64)
    qd = q.double().cpu()
    for i, j in itertools.product(range(b), range(lists)):
        h, g = j * heads // lists, hq // lists
        at = choose(i, j)
        mine = slice(j * g, j * g + g)
        tol[i, mine] = STEP[dtype]
        if len(at) == 0:
            continue
        k, v = keys[i][h][at], values[i][h][at]
        if k_scale is not None:
            k, v = k * k_scale[h].double().cpu(), v * v_scale[h].double().cpu()
        s = qd[i, mine] @ k.T * scale
        size = (qd[i, mine].abs() @ k.abs().T * abs(scale)).amax(1, keepdim=True)
        p = torch.softmax(s, dim=1)
        out[i, mine] = p @ v
        lse[i, mine] = torch.logsumexp(s, dim=1)
        away = (s.amax(1, keepdim=True) - s).amax(1, keepdim=True).clamp(max=100)
        e = (dim + 4) * 2.0 ** -24 * size + 2.0 ** -22 * away + 2.0 ** -16 + (len(at) + 64) * 2.0 ** -24
        tol[i, mine] += UNIT[dtype] * 1.001 * out[i, mine].abs() + 2 * e * (p @ v.abs())
        ltol[i, mine] = (e + 2.0 ** -22 * lse[i, mine][:, None].abs())[:, 0]
    return out, tol, lse, ltol


EDGES = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1000, 2047, 2500]


def check(got, ref):
    near(got[0], ref[0], ref[1], "out")
    near(got[1], ref[2], ref[3], "lse")


def f8_scales(heads, cache, seed):
    if cache != F8:
        return None, None
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(heads, device="cuda", generator=g) * 0.02 + 0.02,
            torch.rand(heads, device="cuda", generator=g) * 0.02 + 0.02)


@pytest.mark.parametrize("hq,heads,dim,page,dtype,cache,layout", [
    (8, 2, 128, 16, F16, F16, "heads"), (32, 8, 128, 16, BF16, BF16, "rows"), (5, 5, 64, 32, F16, F16, "pair"),
    (16, 1, 96, 8, BF16, BF16, "heads"), (17, 1, 128, 16, F16, F16, "heads"), (64, 2, 128, 64, BF16, F8, "heads"),
    (3, 3, 80, 16, F16, F8, "rows"), (12, 4, 256, 16, F16, F16, "heads"), (40, 1, 256, 8, BF16, BF16, "heads"),
    (2, 1, 8, 128, F16, F16, "heads"), (6, 2, 200, 256, BF16, BF16, "heads"), (4, 2, 256, 32, F16, F8, "heads"),
    (2, 2, 16, 8, BF16, F8, "heads"), (7, 7, 72, 16, F16, F16, "heads")])
def test_decode_lengths(jasper, hq, heads, dim, page, dtype, cache, layout):
    kp, vp, tables, keys, values = build_cache(EDGES, heads, page, dim, cache, 40, layout)
    ks, vs = f8_scales(heads, cache, 41)
    q = randn((len(EDGES), hq, dim), dtype, 42, 2.0)
    lens = torch.tensor(EDGES, dtype=torch.int32, device="cuda")
    ref = ref_attention(q, keys, values, dim ** -0.5, lambda i, j: torch.arange(EDGES[i]), dtype, ks, vs)
    check(jasper.decode_attention(q, kp, vp, tables, lens, k_scale=ks, v_scale=vs, return_lse=True), ref)
    out = jasper.decode_attention(q, kp, vp, tables, lens, k_scale=ks, v_scale=vs, max_len=2500)
    near(out, ref[0], ref[1])


@pytest.mark.parametrize("window", [1, 5, 16, 33, 100, 1000, 10 ** 9])
@pytest.mark.parametrize("cache,page", [(F16, 16), (F8, 8)])
def test_decode_window(jasper, window, cache, page):
    kp, vp, tables, keys, values = build_cache(EDGES, 2, page, 64, cache, 50)
    ks, vs = f8_scales(2, cache, 51)
    q = randn((len(EDGES), 6, 64), F16, 52, 2.0)
    lens = torch.tensor(EDGES, dtype=torch.int32, device="cuda")
    ref = ref_attention(q, keys, values, 0.3, lambda i, j: torch.arange(max(0, EDGES[i] - window), EDGES[i]), F16, ks, vs)
    check(jasper.decode_attention(q, kp, vp, tables, lens, scale=0.3, window=window, k_scale=ks, v_scale=vs,
                                  return_lse=True), ref)


@pytest.mark.parametrize("batch,length,hq,heads,cache", [(1, 70_001, 8, 1, F16), (1, 33_333, 4, 2, F8), (2, 20_000, 2, 2, F16)])
def test_decode_long(jasper, batch, length, hq, heads, cache):
    lens = [length - 5 * i for i in range(batch)]
    kp, vp, tables, keys, values = build_cache(lens, heads, 16, 128, cache, 60)
    ks, vs = f8_scales(heads, cache, 61)
    q = randn((batch, hq, 128), F16, 62, 3.0)
    ref = ref_attention(q, keys, values, 128 ** -0.5, lambda i, j: torch.arange(lens[i]), F16, ks, vs)
    check(jasper.decode_attention(q, kp, vp, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), k_scale=ks,
                                  v_scale=vs, return_lse=True), ref)


def test_decode_large_scores_and_infinities(jasper):
    """Scores in the hundreds, of one sign; keys of minus infinity weigh nothing, NaN in a read row is seen."""
    lens = [300, 300, 40, 5]
    kp, vp, tables, keys, values = build_cache(lens, 1, 16, 64, BF16, 70, hostile=False)
    q = randn((4, 2, 64), BF16, 71, 40.0)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = ref_attention(q, keys, values, 1.0, lambda i, j: torch.arange(lens[i]), BF16)
    check(jasper.decode_attention(q, kp, vp, tables, tens, scale=1.0, return_lse=True), ref)
    q = q.abs().contiguous()
    for x, t in ((3, 10), (2, 7), (2, 39)):
        page = tables[x, t // 16].item() if t < lens[x] else None
        if page is not None:
            kp[page, 0, t % 16] = -math.inf
            keys[x][0][t] = -math.inf
    for t in range(5):
        kp[tables[3, 0].item(), 0, t] = -math.inf
    bad = tables[1, 2].item()
    vp[bad, 0, 3, 9] = math.nan
    kp[tables[0, 1].item(), 0, 3, 9] = math.nan
    out, lse = jasper.decode_attention(q, kp, vp, tables, tens, scale=1.0, return_lse=True)
    ref = ref_attention(q, keys, values, 1.0, lambda i, j: torch.arange(lens[i]) if i != 2 else
                        torch.tensor([t for t in range(40) if t not in (7, 39)]), BF16)
    near(out[2:3], ref[0][2:3], ref[1][2:3])
    assert (out[3] == 0).all() and (lse[3] == -math.inf).all()
    assert out[1, :, 9].isnan().all() and out[1, :, :9].isfinite().all()
    assert out[0].isnan().all() and lse[0].isnan().all()


def test_decode_pages_outside_and_query_strides(jasper):
    lens = [100, 64]
    kp, vp, tables, keys, values = build_cache(lens, 2, 16, 64, F16, 80)
    tables[0, 2], tables[1, 0] = -7, kp.size(0)  # lost pages: their tokens are left out
    fused = randn((2, 9, 64), F16, 81, 2.0)
    q = fused[:, 2:6]
    tens = torch.tensor([100, 0, 64, 0], dtype=torch.int32, device="cuda")[::2]
    ref = ref_attention(q, keys, values, 0.125, lambda i, j: torch.cat([torch.arange(32), torch.arange(48, 100)]) if i == 0
                        else torch.arange(16, 64), F16)
    check(jasper.decode_attention(q, kp, vp, tables, tens, return_lse=True), ref)
    odd = torch.empty(2 * 4 * 64 + 1, dtype=F16, device="cuda")[1:].view(2, 4, 64).copy_(q)
    check(jasper.decode_attention(odd, kp, vp, tables, tens, return_lse=True), ref)
    wide = torch.empty((2, 64, 4), dtype=F16, device="cuda").transpose(1, 2).copy_(q)
    check(jasper.decode_attention(wide, kp, vp, tables, tens, return_lse=True), ref)
    # lengths over what the table holds, and below zero
    out, lse = jasper.decode_attention(q, kp, vp, tables[:, :4].contiguous(),
                                       torch.tensor([1000, -3], dtype=torch.int32, device="cuda"), return_lse=True)
    cut = ref_attention(q, keys, values, 0.125, lambda i, j: torch.cat([torch.arange(32), torch.arange(48, 64)]), F16)
    near(out[:1], cut[0][:1], cut[1][:1])
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_offsets_past_32_bits(jasper):
    """More than 2^32 bytes of keys: rows at the far end are the ones read, written and copied."""
    heads, page, dim = 8, 64, 128
    pages = 2 ** 32 // (heads * page * dim * 2) + 70
    kp = torch.zeros((pages, heads, page, dim), dtype=F16, device="cuda")
    vp = torch.zeros_like(kp)
    n = 150
    k, v = randn((n, heads, dim), F16, 90), randn((n, heads, dim), F16, 91)
    table = torch.tensor([[pages - 1, 0, pages - 40]], dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = table[0, at // page].long() * page + at % page
    jasper.append_tokens(None, k, v, None, slots, None, None, kp, vp)
    q = randn((1, 16, dim), F16, 92, 2.0)
    keys, values = [k.double().cpu().transpose(0, 1)], [v.double().cpu().transpose(0, 1)]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    ref = ref_attention(q, keys, values, dim ** -0.5, lambda i, j: torch.arange(n), F16)
    check(jasper.decode_attention(q, kp, vp, table, lens, return_lse=True), ref)
    ids = torch.randperm(n)[:77].int()
    some = ref_attention(q, keys, values, dim ** -0.5, lambda i, j: ids.long(), F16)
    listed = ids.cuda().expand(1, heads, 77).contiguous()
    check(jasper.retrieved_attention(q, kp, vp, table, lens, listed, return_lse=True), some)
    moved = torch.tensor([pages - 1, pages - 40], dtype=torch.int32, device="cuda")
    to = torch.tensor([pages - 2, pages - 3], dtype=torch.int32, device="cuda")
    jasper.copy_pages(kp, vp, moved, to, tables=table)
    assert table.tolist() == [[pages - 2, 0, pages - 3]]
    kp[pages - 1], kp[pages - 40] = 0, 0
    check(jasper.decode_attention(q, kp, vp, table, lens, return_lse=True), ref)


@pytest.mark.parametrize("hq,heads,lists,dim,page,dtype,cache,count,first,last,layout", [
    (8, 2, 2, 128, 16, F16, F16, 100, 4, 20, "heads"), (8, 2, 8, 128, 16, BF16, BF16, 33, 0, 0, "rows"),
    (32, 8, 32, 128, 16, F16, F16, 128, 4, 64, "heads"), (4, 4, 4, 64, 32, BF16, F8, 300, 16, 256, "heads"),
    (24, 1, 1, 96, 8, F16, F16, 1, 1, 1, "pair"), (24, 1, 24, 80, 16, F16, F8, 7, 3, 0, "heads"),
    (6, 3, 3, 256, 16, BF16, BF16, 500, 0, 33, "heads"), (2, 1, 2, 8, 8, F16, F16, 50, 2, 2, "heads"),
    (16, 2, 2, 128, 16, F16, F16, 0, 5, 40, "heads"), (4, 2, 4, 256, 64, F16, F8, 64, 0, 7, "heads"),
    (4, 1, 1, 128, 16, F16, F16, 3000, 300, 700, "heads")])
def test_retrieved(jasper, hq, heads, lists, dim, page, dtype, cache, count, first, last, layout):
    lens = [0, 1, 5, 33, 64, 129, 700, 2500]
    kp, vp, tables, keys, values = build_cache(lens, heads, page, dim, cache, 100, layout)
    ks, vs = f8_scales(heads, cache, 101)
    q = randn((len(lens), hq, dim), dtype, 102, 2.0)
    g = torch.Generator().manual_seed(103)
    ids = torch.empty((len(lens), lists, count), dtype=torch.int32)
    for i, n in enumerate(lens):  # in order of no kind, some twice, some missing, some past the end
        ids[i] = torch.randint(0, max(1, n), (lists, count), generator=g, dtype=torch.int32)
    ids[torch.rand(ids.shape, generator=g) < 0.1] = -1
    ids[torch.rand(ids.shape, generator=g) < 0.05] = 2 ** 31 - 1
    ids[torch.rand(ids.shape, generator=g) < 0.05] = -2 ** 31
    ids[6] = -1  # a search that found nothing

    def choose(i, j):
        n = lens[i]
        a, z = min(first, n), max(n - last, min(first, n))
        mine = ids[i, j].long()
        return torch.cat([torch.arange(a), torch.arange(z, n), mine[(mine >= a) & (mine < z)]])

    ref = ref_attention(q, keys, values, dim ** -0.5, choose, dtype, ks, vs, lists)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    check(jasper.retrieved_attention(q, kp, vp, tables, tens, ids.cuda(), first=first, last=last, k_scale=ks,
                                     v_scale=vs, return_lse=True), ref)
    strided = ids.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    out = jasper.retrieved_attention(q, kp, vp, tables, tens, strided, first=first, last=last, k_scale=ks, v_scale=vs)
    near(out, ref[0], ref[1])


def test_retrieved_everything_is_decode(jasper):
    lens = [777, 50]
    kp, vp, tables, keys, values = build_cache(lens, 2, 16, 128, F16, 110)
    q = randn((2, 8, 128), F16, 111, 2.0)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ids = torch.randperm(777).int().cuda().expand(2, 2, 777).contiguous()
    ref = ref_attention(q, keys, values, 128 ** -0.5, lambda i, j: torch.arange(lens[i]), F16)
    check(jasper.retrieved_attention(q, kp, vp, tables, tens, ids, first=3, last=9, return_lse=True), ref)
    check(jasper.decode_attention(q, kp, vp, tables, tens, return_lse=True), ref)


def test_many_sequences(jasper):
    g = torch.Generator().manual_seed(120)
    lens = torch.randint(0, 60, (700,), generator=g).tolist()
    kp, vp, tables, keys, values = build_cache(lens, 1, 8, 64, F16, 121)
    q = randn((700, 2, 64), F16, 122, 2.0)
    ref = ref_attention(q, keys, values, 0.125, lambda i, j: torch.arange(lens[i]), F16)
    check(jasper.decode_attention(q, kp, vp, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                  return_lse=True), ref)


def test_repeats_and_streams_give_the_same_bits(jasper):
    lens = [5000, 3, 900]
    kp, vp, tables, _, _ = build_cache(lens, 2, 16, 128, BF16, 130)
    q = randn((3, 8, 128), BF16, 131, 2.0)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ids = torch.randint(0, 3, (3, 2, 100), dtype=torch.int32, device="cuda")

    def both():
        return (*jasper.decode_attention(q, kp, vp, tables, tens, return_lse=True),
                *jasper.retrieved_attention(q, kp, vp, tables, tens, ids, first=4, last=200, return_lse=True))

    want = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(side):
            got = both()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph_capture(jasper):
    """A serving step's calls in a graph, replayed on changed inputs with eager work in between."""
    heads, hq, dim, page, b = 2, 8, 128, 16, 3
    kp, vp = make_pages(3 * 40, heads, page, dim, F16)
    tables = torch.randperm(120).int().view(3, 40).cuda()
    cos, sin = jasper.rotary_table(700, dim)
    qkv = randn((b, hq + 2 * heads, dim), F16, 140)
    lens = torch.tensor([600, 17, 0], dtype=torch.int32, device="cuda")
    pos, slots = torch.zeros(b, dtype=torch.int64, device="cuda"), torch.zeros(b, dtype=torch.int64, device="cuda")
    ids = torch.zeros((b, heads, 50), dtype=torch.int32, device="cuda")
    src, dst = torch.tensor([5], dtype=torch.int32, device="cuda"), torch.tensor([-1], dtype=torch.int32, device="cuda")

    def step():
        q, k, v = qkv.split([hq, heads, heads], dim=1)
        q = jasper.append_tokens(q, k, v, pos, slots, cos, sin, kp, vp)
        jasper.copy_pages(kp, vp, src, dst)
        return (q, *jasper.decode_attention(q, kp, vp, tables, lens, return_lse=True),
                *jasper.retrieved_attention(q, kp, vp, tables, lens, ids, first=2, last=9, return_lse=True))

    kp.copy_(randn(kp.shape, F16, 141))
    vp.copy_(randn(vp.shape, F16, 142))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        lens += 1
        pos.copy_(lens.long() - 1)
        slots.copy_(tables.gather(1, (pos // page)[:, None])[:, 0].long() * page + pos % page)
        qkv.copy_(randn(qkv.shape, F16, 150 + i))
        ids.copy_(torch.randint(0, 600, ids.shape, dtype=torch.int32, device="cuda"))
        before = kp.clone(), vp.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out] + [kp.clone(), vp.clone()]
        kp.copy_(before[0])
        vp.copy_(before[1])
        want = [*step(), kp, vp]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


# ---- refusals ----

def test_refusals(jasper):
    kp, vp = make_pages(8, 2, 16, 64, F16, seed=160)
    q = randn((2, 4, 64), F16, 161)
    tables = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    ids = torch.zeros((2, 2, 5), dtype=torch.int32, device="cuda")
    scale = torch.ones(2, device="cuda")
    dec, ret = jasper.decode_attention, jasper.retrieved_attention
    bad = [
        lambda: dec(q.float(), kp, vp, tables, lens), lambda: dec(q.bfloat16(), kp, vp, tables, lens),
        lambda: dec(q[:, :3], kp, vp, tables, lens), lambda: dec(q[..., :32], kp, vp, tables, lens),
        lambda: dec(q.cpu(), kp, vp, tables, lens), lambda: dec(q, kp.cpu(), vp.cpu(), tables, lens),
        lambda: dec(q, kp, vp[:4], tables, lens), lambda: dec(q, kp, vp.bfloat16(), tables, lens),
        lambda: dec(q, kp, vp, tables.long(), lens), lambda: dec(q, kp, vp, tables[:1], lens),
        lambda: dec(q, kp, vp, tables, lens.long()), lambda: dec(q, kp, vp, tables, lens[:1]),
        lambda: dec(q, kp, vp, tables, lens, window=-1), lambda: dec(q, kp, vp, tables, lens, max_len=-1),
        lambda: dec(q, kp, vp, tables, lens, k_scale=scale), lambda: dec(q, kp[:, :, :12], vp[:, :, :12], tables, lens),
        lambda: dec(q, kp[0], vp[0], tables, lens), lambda: dec(q, kp.float(), vp.float(), tables, lens),
        lambda: dec(q.detach().requires_grad_(), kp, vp, tables, lens),
        lambda: dec(q, kp, vp, tables.t(), lens[:1].expand(4)),
        lambda: dec(q, kp, vp.transpose(1, 2).contiguous().transpose(1, 2), tables, lens),
        lambda: dec(q[..., :60], kp[..., :60], vp[..., :60], tables, lens),
        lambda: dec(q[..., :56], kp[..., 4:60], vp[..., 4:60], tables, lens),
        lambda: ret(q, kp, vp, tables, lens, ids.long()), lambda: ret(q, kp, vp, tables, lens, ids[:, :1]),
        lambda: ret(q, kp, vp, tables, lens, ids[:1]), lambda: ret(q, kp, vp, tables, lens, ids, first=-1),
        lambda: ret(q, kp, vp, tables, lens, ids, last=2 ** 30),
        lambda: jasper.copy_pages(kp, vp, lens, lens[:1]), lambda: jasper.copy_pages(kp, vp, lens.long(), lens.long()),
        lambda: jasper.copy_pages(kp, vp, lens, lens, tables=tables.long()),
        lambda: jasper.copy_pages(kp, vp, lens, lens, tables=tables.t()),
        lambda: jasper.copy_pages(kp.cpu(), vp.cpu(), lens.cpu(), lens.cpu()),
    ]
    cos, sin = jasper.rotary_table(16, 64)
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    k = q[:, :2]
    bad += [
        lambda: jasper.rotary(q.float(), None, pos, cos, sin), lambda: jasper.rotary(q, k.bfloat16(), pos, cos, sin),
        lambda: jasper.rotary(q, None, pos[:1], cos, sin), lambda: jasper.rotary(q, None, pos.float(), cos, sin),
        lambda: jasper.rotary(q[..., :62], None, pos, cos, sin), lambda: jasper.rotary(q, None, pos, cos, None),
        lambda: jasper.rotary(q, None, pos, cos.half(), sin.half()), lambda: jasper.rotary(q, None, pos, cos, sin[:5]),
        lambda: jasper.rotary(q, None, pos.cpu(), cos, sin), lambda: jasper.rotary(q[..., :63], None, pos, cos, sin),
        lambda: jasper.append_tokens(q, k, k, pos, pos, cos, sin, kp.bfloat16(), vp.bfloat16()),
        lambda: jasper.append_tokens(q, q, q, pos, pos, cos, sin, kp, vp),
        lambda: jasper.append_tokens(q, k, k[:1], pos, pos, cos, sin, kp, vp),
        lambda: jasper.append_tokens(q, k, k, None, pos, cos, sin, kp, vp),
        lambda: jasper.append_tokens(q, k, k, pos, pos[:1], cos, sin, kp, vp),
        lambda: jasper.append_tokens(q, k, k, pos, pos.float(), cos, sin, kp, vp),
        lambda: jasper.append_tokens(q, k, k, pos, pos, cos, sin, kp, vp, k_scale=scale),
        lambda: jasper.append_tokens(q.detach().requires_grad_(), k, k, pos, pos, cos, sin, kp, vp),
        lambda: jasper.rotary_table(4, 3), lambda: jasper.rotary_table(4, 4, scaling="other"),
        lambda: jasper.rotary_table(4, 4, scaling="yarn", factor=2.0),
        lambda: jasper.rotary_table(4, 4, scaling="linear", factor=0.5),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was accepted")
    torch.cuda.synchronize()


def test_empty_calls(jasper):
    kp, vp = make_pages(8, 2, 16, 64, F16, seed=170)
    tables = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    lens = torch.zeros(0, dtype=torch.int32, device="cuda")
    out, lse = jasper.decode_attention(randn((0, 4, 64), F16, 1), kp, vp, tables, lens, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    ids = torch.zeros((0, 2, 5), dtype=torch.int32, device="cuda")
    assert jasper.retrieved_attention(randn((0, 4, 64), F16, 1), kp, vp, tables, lens, ids).shape == (0, 4, 64)
    none = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    out, lse = jasper.decode_attention(randn((2, 4, 64), F16, 1), kp, vp, none,
                                       torch.tensor([3, 0], dtype=torch.int32, device="cuda"), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    empty, _ = make_pages(0, 2, 16, 64, F16)
    out = jasper.decode_attention(randn((1, 4, 64), F16, 1), empty, empty, torch.zeros((1, 4), dtype=torch.int32, device="cuda"),
                                  torch.tensor([9], dtype=torch.int32, device="cuda"))
    assert (out == 0).all()


@pytest.mark.parametrize("hq,heads,dim,dtype,cache", [
    (130, 1, 128, F16, F16), (64, 2, 64, BF16, F8), (130, 1, 256, BF16, BF16), (66, 2, 96, F16, F16), (33, 1, 16, F16, F8)])
def test_many_heads_to_a_key_head(jasper, hq, heads, dim, dtype, cache):
    lens = [3000, 0, 1, 900, 4100]
    kp, vp, tables, keys, values = build_cache(lens, heads, 16, dim, cache, 190)
    ks, vs = f8_scales(heads, cache, 191)
    q = randn((len(lens), hq, dim), dtype, 192, 2.0)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = ref_attention(q, keys, values, dim ** -0.5, lambda i, j: torch.arange(lens[i]), dtype, ks, vs)
    check(jasper.decode_attention(q, kp, vp, tables, tens, k_scale=ks, v_scale=vs, return_lse=True), ref)
    ids = torch.arange(3500, dtype=torch.int32, device="cuda").flip(0).expand(len(lens), heads, 3500).contiguous()
    ref = ref_attention(q, keys, values, dim ** -0.5,
                        lambda i, j: torch.tensor([t for t in range(lens[i]) if t < 3500 or t >= lens[i] - 7], dtype=torch.int64),
                        dtype, ks, vs)
    check(jasper.retrieved_attention(q, kp, vp, tables, tens, ids, first=1, last=7, k_scale=ks, v_scale=vs,
                                     return_lse=True), ref)


SHORT = [0, 1, 5, 8, 17, 31, 32, 33, 64, 100, 129, 255, 300, 500]


@pytest.mark.parametrize("hq,heads,dim,page,dtype,cache", [
    (8, 2, 128, 16, F16, F16), (32, 8, 128, 16, BF16, BF16), (20, 1, 128, 16, BF16, F8), (5, 5, 64, 32, F16, F16),
    (16, 1, 64, 8, F16, F16), (3, 3, 80, 16, F16, F8), (16, 1, 96, 8, BF16, BF16), (12, 4, 256, 16, F16, F16),
    (17, 1, 256, 8, BF16, F8), (6, 2, 200, 64, BF16, BF16), (2, 1, 8, 128, F16, F16), (4, 2, 16, 8, BF16, F8)])
@pytest.mark.parametrize("repeat", [1, 20])
def test_decode_short(jasper, hq, heads, dim, page, dtype, cache, repeat):
    """Tables that hold few tokens; few sequences, and many."""
    lens = SHORT * repeat
    kp, vp, tables, keys, values = build_cache(lens, heads, page, dim, cache, 180)
    tables = tables[:, :-(-500 // page)]  # rows of a wider table
    ks, vs = f8_scales(heads, cache, 181)
    q = randn((len(lens), hq, dim), dtype, 182, 2.0)
    ref = ref_attention(q, keys, values, dim ** -0.5, lambda i, j: torch.arange(lens[i]), dtype, ks, vs)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    check(jasper.decode_attention(q, kp, vp, tables, tens, k_scale=ks, v_scale=vs, return_lse=True), ref)


def test_rotary_gradient_of_broadcast_rows(jasper):
    """One key head seen by four: their gradients add up in it."""
    n, dim = 9, 32
    cos, sin = jasper.rotary_table(64, dim)
    pos = torch.arange(n, device="cuda") * 5
    q = randn((n, 4, dim), BF16, 200)
    one = randn((n, 1, dim), BF16, 201).requires_grad_()
    g = randn((n, 4, dim), BF16, 202)
    _, k = jasper.rotary(q, one.expand(n, 4, dim), pos, cos, sin)
    want, _ = ref_rotary(one.detach().expand(n, 4, dim), pos, cos, sin, False)
    near(k.detach(), want, rotary_tol(want, want.abs() * 2, BF16))
    got, = torch.autograd.grad(k, one, g)
    each, size = ref_rotary(g, pos, cos, sin, False, back=True)
    # four rounded gradients, added with three roundings
    tol = rotary_tol(each, size, BF16).sum(1, keepdim=True) + 3 * UNIT[BF16] * each.abs().sum(1, keepdim=True)
    near(got, each.sum(1, keepdim=True), tol)
    flat = randn((1, 4, dim), BF16, 203).requires_grad_()  # one row for all positions
    out, _ = jasper.rotary(flat.expand(n, 4, dim), None, pos, cos, sin)
    got, = torch.autograd.grad(out, flat, g)
    tol = rotary_tol(each, size, BF16).sum(0, keepdim=True) + n * UNIT[BF16] * each.abs().sum(0, keepdim=True)
    near(got, each.sum(0, keepdim=True), tol)


@pytest.mark.parametrize("scale", [-0.4, 0.0, 1e-6])
def test_decode_scales(jasper, scale):
    lens = [1500, 70, 1]
    kp, vp, tables, keys, values = build_cache(lens, 2, 16, 128, BF16, 210)
    q = randn((3, 6, 128), BF16, 211, 2.0)
    ref = ref_attention(q, keys, values, scale, lambda i, j: torch.arange(lens[i]), BF16)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    check(jasper.decode_attention(q, kp, vp, tables, tens, scale=scale, return_lse=True), ref)


def test_flat_softmax_over_many_tokens_keeps_its_tail(jasper):
    """One token far above 100,000 equal ones whose weights are 2^-26 of its: together 0.15% of the sum."""
    n = 100_001
    kp, vp, tables, keys, values = build_cache([n], 1, 16, 64, F16, 220)
    kp.zero_()
    keys[0].zero_()
    page = tables[0, 5000 // 16].item()
    kp[page, 0, 5000 % 16, 0] = 26 * math.log(2.0)
    keys[0][0, 5000, 0] = kp[page, 0, 5000 % 16, 0].double().cpu()
    q = torch.zeros((1, 1, 64), dtype=F16, device="cuda")
    q[0, 0, 0] = 1.0
    vp.copy_(vp.abs() + 1.0)
    values[0].copy_(vp.float()[tables[0, :-(-n // 16)].long()].transpose(0, 1).reshape(1, -1, 64)[:, :n].double().cpu())
    ref = ref_attention(q, keys, values, 1.0, lambda i, j: torch.arange(n), F16)
    tens = torch.tensor([n], dtype=torch.int32, device="cuda")
    check(jasper.decode_attention(q, kp, vp, tables, tens, scale=1.0, return_lse=True), ref)


@pytest.mark.parametrize("batch,window", [(65, 0), (130, 0), (700, 0), (700, 50), (2000, 0)])
def test_many_unlike_sequences(jasper, batch, window):
    """Tables wide enough that the waves share out all sequences' tokens among them: runs of short sequences, of
    empty ones, and long ones between."""
    g = torch.Generator().manual_seed(230)
    lens = torch.randint(0, 90, (batch,), generator=g)
    lens[torch.rand(batch, generator=g) < 0.2] = 0
    lens[batch // 3], lens[-1], lens[batch // 2:batch // 2 + 20] = 9000, 4321, 0
    lens = lens.tolist()
    kp, vp, tables, keys, values = build_cache(lens, 2, 16, 64, F16, 231)
    q = randn((batch, 4, 64), F16, 232, 2.0)
    tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = ref_attention(q, keys, values, 0.125, lambda i, j: torch.arange(max(0, lens[i] - window) if window else 0, lens[i]),
                        F16)
    check(jasper.decode_attention(q, kp, vp, tables, tens, window=window, return_lse=True), ref)
    ids = torch.arange(7000, dtype=torch.int32, device="cuda").expand(3, 2, 7000).contiguous()
    few = torch.tensor([0, batch // 3, batch - 1], device="cuda")
    rows = few.tolist()
    ref = ref_attention(q[few], [keys[i] for i in rows], [values[i] for i in rows], 0.125,
                        lambda i, j: torch.arange(min(7000, lens[rows[i]])), F16)
    check(jasper.retrieved_attention(q[few], kp, vp, tables[few], tens[few], ids, return_lse=True), ref)


def test_copy_pages_in_several_launches(jasper):
    """More than 32 GB are copied in several launches (here of pages that are all the same memory), and the table
    entries of every part are rewritten."""
    kp, vp = (randn((1, 64, 256, 256), F16, 240 + i).expand(5000, -1, -1, -1) for i in range(2))
    before = kp[0].clone(), vp[0].clone()
    src = torch.arange(2100, dtype=torch.int32, device="cuda")
    tables = torch.arange(5000, dtype=torch.int32, device="cuda").flip(0).contiguous()
    jasper.copy_pages(kp, vp, src, src + 2500, tables=tables)
    want = torch.arange(5000, device="cuda").flip(0)
    assert torch.equal(tables.long(), torch.where(want < 2100, want + 2500, want))
    assert torch.equal(kp[0], before[0]) and torch.equal(vp[0], before[1])


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 15, 16])
@pytest.mark.parametrize("heads", [1, 8])
def test_parts_of_a_stream_start_on_16_bytes(jasper, group, heads):
    """What a wave leaves for the join is written and read 16 bytes at a time. The workspace is a list of ends, whole
    16s, then two parts to a work-group. As many work-groups are taken for 64 values as for 128, so the difference
    tells their number: 64 values more per query head and part."""
    import ctypes
    from tests.test_kvcache_capi import I64, Pages
    lib = ctypes.CDLL(str(jasper.library_path()))
    fn = lib.jasperx_attention_workspace
    fn.restype, fn.argtypes = I64, [I64, I64, ctypes.POINTER(Pages), I64, I64]
    sizes = []
    for dim in (64, 128):
        p = Pages(layers=1, pages=4, heads=heads, page_size=16, dim=dim, type=0, row_stride=dim, head_stride=16 * dim,
                  page_stride=heads * 16 * dim)
        sizes.append(fn(1, heads * group, ctypes.byref(p), 100_000, 0))
    ends = -(-heads * 8 // 16) * 16
    work_groups, rest = divmod(sizes[1] - sizes[0], 2 * 64 * 4 * group)
    assert rest == 0 and work_groups > 0
    for dim, size in zip((64, 128), sizes):
        values = group * (dim + 2)
        part = -(-values // 4) * 16
        assert size == ends + work_groups * 2 * part


def test_rotary_refuses_tables_that_require_a_gradient(jasper):
    cos, sin = jasper.rotary_table(16, 64)
    q = randn((3, 2, 64), F16, 250)
    pos = torch.arange(3, device="cuda")
    for c, s in ((cos.clone().requires_grad_(), sin), (cos, sin.clone().requires_grad_())):
        for rows in (q, q.clone().requires_grad_()):
            with pytest.raises(ValueError, match="no gradient for cos and sin"):
                jasper.rotary(rows, None, pos, c, s)
        with torch.no_grad():
            assert torch.equal(jasper.rotary(q, None, pos, c, s)[0], jasper.rotary(q, None, pos, cos, sin)[0])


def test_append_and_copy_refuse_what_requires_a_gradient(jasper):
    """Rows, tables, pages and scales alike; without gradients they are what they always were."""
    heads, page, dim = 2, 16, 64
    given = dict(zip(("q", "k", "v"), (randn((3, h, dim), F16, 260 + h) for h in (4, heads, heads))))
    given["cos"], given["sin"] = jasper.rotary_table(16, dim)
    at = torch.arange(3, device="cuda")
    pair = torch.tensor([0], dtype=torch.int32, device="cuda")
    for cache in (F16, F8):
        given["k_pages"], given["v_pages"] = make_pages(4, heads, page, dim, F16)
        if cache == F8:
            given |= {"k_scale": torch.ones(heads, device="cuda"), "v_scale": torch.ones(heads, device="cuda")}
            given["k_pages"], given["v_pages"] = make_pages(4, heads, page, dim, F8)
        want = jasper.append_tokens(positions=at, slots=at, **given)
        for name in given:
            asked = given | {name: given[name].detach().clone().requires_grad_()}
            with pytest.raises(ValueError, match="append_tokens has no gradient"):
                jasper.append_tokens(positions=at, slots=at, **asked)
            if name.endswith("pages"):
                with pytest.raises(ValueError, match="copy_pages has no gradient"):
                    jasper.copy_pages(asked["k_pages"], asked["v_pages"], pair, pair + 1)
            with torch.no_grad():
                assert torch.equal(jasper.append_tokens(positions=at, slots=at, **asked), want), name


def test_attention_refuses_what_requires_a_gradient(jasper):
    tables = torch.tensor([[2, 1, 0], [3, 0, 0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 9], dtype=torch.int32, device="cuda")
    ids = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 2, 3)
    for cache in (F16, F8):
        given = {"q": randn((2, 4, 64), F16, 270)}
        given["k_pages"], given["v_pages"] = make_pages(4, 2, 16, 64, cache, seed=271)
        if cache == F8:
            given |= {"k_scale": torch.full((2,), 0.03, device="cuda"), "v_scale": torch.full((2,), 0.03, device="cuda")}
        for f in (lambda **x: jasper.decode_attention(tables=tables, lens=lens, **x),
                  lambda **x: jasper.retrieved_attention(tables=tables, lens=lens, ids=ids, first=1, **x)):
            want = f(**given)
            for name in given:
                asked = given | {name: given[name].detach().clone().requires_grad_()}
                with pytest.raises(ValueError, match="has no gradient"):
                    f(**asked)
                with torch.no_grad():
                    assert torch.equal(f(**asked), want), name


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_forward_mode(jasper, interleaved, grad):
    """The map is linear: the tangent of the result is the rotation of the tangent. With rows that require a gradient
    too, the tangent is differentiable as the result is."""
    import torch.autograd.forward_ad as fwd
    n, dim, rot = 19, 96, 48
    cos, sin = jasper.rotary_table(300, rot)
    pos = torch.randint(0, 300, (n,), device="cuda")
    q, k = randn((n, 6, dim), F16, 280), randn((n, 2, dim), F16, 281)
    tq, tk = randn((n, 6, dim), F16, 282), randn((n, 2, dim), F16, 283)
    plain = jasper.rotary(q, k, pos, cos, sin, interleaved=interleaved)
    if grad:
        q, k, tq = q.requires_grad_(), k.requires_grad_(), tq.requires_grad_()
    wants = [ref_rotary(t.detach(), pos, cos, sin, interleaved) for t in (tq, tk)]
    with fwd.dual_level():
        dq, dk = fwd.make_dual(q, tq), fwd.make_dual(k, tk)
        out = jasper.rotary(dq, dk, pos, cos, sin, interleaved=interleaved)
        for y, same, (want, size) in zip(out, plain, wants):
            value, tangent = fwd.unpack_dual(y)
            assert torch.equal(value, same)
            near(tangent.detach(), want, rotary_tol(want, size, F16))
        only_k = jasper.rotary(q, dk, pos, cos, sin, interleaved=interleaved)
        assert fwd.unpack_dual(only_k[0]).tangent is None
        assert torch.equal(fwd.unpack_dual(only_k[1]).tangent, fwd.unpack_dual(out[1]).tangent)
        alone, none = jasper.rotary(dq, None, pos, cos, sin, interleaved=interleaved)
        assert none is None and torch.equal(fwd.unpack_dual(alone).tangent, fwd.unpack_dual(out[0]).tangent)
        if grad:
            g = randn((n, 6, dim), F16, 284)
            value, tangent = fwd.unpack_dual(out[0])
            want, size = ref_rotary(g, pos, cos, sin, interleaved, back=True)
            for y, x in ((value, q), (tangent, tq)):
                near(torch.autograd.grad(y, x, g, retain_graph=True)[0], want, rotary_tol(want, size, F16))
        for c, s in ((fwd.make_dual(cos, sin), sin), (cos, fwd.make_dual(sin, cos))):
            with pytest.raises(ValueError, match="no gradient for cos and sin"):
                jasper.rotary(q, k, pos, c, s)
    again = jasper.rotary(q, k, pos, cos, sin, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(again, plain))


def test_tangents_are_refused_where_none_come_out(jasper):
    """append_tokens, copy_pages and the attentions have no forward-mode derivative either, with gradients on or off."""
    import torch.autograd.forward_ad as fwd
    q, k = randn((2, 4, 64), F16, 290), randn((2, 2, 64), F16, 291)
    kp, vp = make_pages(4, 2, 16, 64, F16, seed=292)
    cos, sin = jasper.rotary_table(16, 64)
    at = torch.arange(2, device="cuda")
    i32 = torch.arange(2, dtype=torch.int32, device="cuda")
    with fwd.dual_level(), torch.no_grad():
        def dual(x):
            return fwd.make_dual(x, torch.ones_like(x))
        for rows in ((dual(q), k, k), (q, dual(k), k), (q, k, dual(k))):
            with pytest.raises(ValueError, match="append_tokens has no gradient"):
                jasper.append_tokens(*rows, at, at, cos, sin, kp, vp)
        with pytest.raises(ValueError, match="append_tokens has no gradient"):
            jasper.append_tokens(q, k, k, at, at, dual(cos), sin, kp, vp)
        with pytest.raises(ValueError, match="copy_pages has no gradient"):
            jasper.copy_pages(kp, dual(vp), i32, i32 + 2)
        for pages, rows in (((kp, vp), dual(q)), ((dual(kp), vp), q), ((kp, dual(vp)), q)):
            with pytest.raises(ValueError, match="has no gradient"):
                jasper.decode_attention(rows, *pages, i32[:, None], i32)
            with pytest.raises(ValueError, match="has no gradient"):
                jasper.retrieved_attention(rows, *pages, i32[:, None], i32, i32.expand(2, 2, 2).contiguous())
        plain = jasper.decode_attention(q, kp, vp, i32[:, None], i32)
        assert torch.equal(jasper.decode_attention(dual(q).detach(), kp, vp, i32[:, None], i32), plain)


def test_writes_in_place_are_counted(jasper):
    """Autograd has to know that pages and tables changed: what it saved of them before is stale."""
    store = [torch.zeros((2, 4, 2, 16, 64), dtype=F16, device="cuda") for _ in range(2)]
    kp, vp = store[0][1], store[1][1]  # a layer of larger tensors
    k = randn((2, 2, 64), F16, 300)
    at = torch.arange(2, device="cuda")
    src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 3))
    tables = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    w = randn(kp.shape, F16, 301).requires_grad_()
    tensors = [*store, kp, vp, tables]

    def counts():
        return [t._version for t in tensors]

    saved, before = (kp * w).sum(), counts()
    jasper.append_tokens(None, k, k, None, at, None, None, kp, vp)
    assert [b > a for a, b in zip(before, counts())] == [True] * 4 + [False]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    for given, moved in ((None, False), (tables, True)):
        saved, before = (vp * w).sum(), counts()
        jasper.copy_pages(*store, src, dst, tables=given)
        assert [b > a for a, b in zip(before, counts())] == [True] * 4 + [moved]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()
    saved, before = (vp * w).sum(), counts()
    jasper.decode_attention(randn((2, 4, 64), F16, 302), kp, vp, tables, dst.expand(2).contiguous())
    assert counts() == before
    saved.backward()
    with torch.inference_mode():  # such tensors are not counted, and still written
        free = torch.zeros_like(kp), torch.zeros_like(vp)
    jasper.append_tokens(None, k, k, None, at, None, None, *free)
    jasper.copy_pages(*free, src, dst)
    assert torch.equal(free[0][0, :, :2], k.transpose(0, 1)) and torch.equal(free[1][3], free[1][0])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_e4m3_quotients_are_a_division_s(jasper, dtype):
    """Every value of the type over ordinary scales, tiny, huge, infinite and zero ones: the bits of a division in 32
    bits, saturated and rounded, the sign of a zero among them."""
    scales = [0.001, 1 / 3, -0.02, 7.3, 448.0, 2.0 ** -79, 2.0 ** 79, 1.3 * 2.0 ** -81, 1.7 * 2.0 ** 81, 2.0 ** -126,
              2.0 ** -127, 2.0 ** -129, 3 * 2.0 ** -134, 3e38, math.inf, 0.0]
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    k = bits.view(256, 1, 256).expand(256, len(scales), 256)
    scale = torch.tensor(scales, dtype=torch.float32)
    kp, vp = make_pages(32, len(scales), 8, 256, F8)
    jasper.append_tokens(None, k.cuda(), k.cuda(), None, torch.arange(256, device="cuda"), None, None, kp, vp,
                         k_scale=scale.cuda(), v_scale=scale.cuda())
    want = (k.float() / scale[None, :, None]).clamp(-448, 448).to(F8)
    for store in (kp, vp):
        got = store.transpose(1, 2).reshape(want.shape).cpu()
        nan = want.float().isnan()
        assert torch.equal(got.float().isnan(), nan)
        off = (got.view(torch.uint8) != want.view(torch.uint8)) & ~nan
        assert not off.any(), [(scales[i], int(n)) for i, n in enumerate(off.sum((0, 2)).tolist()) if n]


def test_every_page_of_several_launches_is_copied(jasper):
    """2,100 pages of 8 MB of keys and as much of values: 2,048 go in the first launch, the others in the second.
    No page shares memory with another, and each holds its own numbers."""
    torch.cuda.empty_cache()
    moves, shape = 2100, (4201, 64, 256, 256)
    kp, vp = (torch.empty(shape, dtype=F16, device="cuda") for _ in range(2))
    words = [x.view(torch.int64).view(shape[0], -1) for x in (kp, vp)]
    g = torch.Generator(device="cuda").manual_seed(310)
    for x in words:
        x.random_(generator=g)
    sums = [x.sum(1) for x in words]
    order = torch.randperm(shape[0], device="cuda", generator=g)
    src, dst, spare = order[:moves], order[moves:2 * moves], order[2 * moves:]
    tables = order.flip(0).int().contiguous()
    jasper.copy_pages(kp, vp, src.int(), dst.int(), tables=tables)
    for x, before in zip(words, sums):
        for i in range(0, moves, 70):
            assert torch.equal(x[dst[i:i + 70]], x[src[i:i + 70]]), i
        after = x.sum(1)
        assert torch.equal(after[dst], before[src]) and torch.equal(after[src], before[src])
        assert torch.equal(after[spare], before[spare])
    to = torch.arange(shape[0], device="cuda")
    to[src] = dst
    assert torch.equal(tables.long(), to[order.flip(0)])
    del kp, vp, words, x
    torch.cuda.empty_cache()


def test_caches_without_layers_or_heads_are_refused_as_arguments(jasper):
    kp, vp = (torch.zeros((0, 4, 2, 16, 64), dtype=F16, device="cuda") for _ in range(2))
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="at least one layer"):
        jasper.copy_pages(kp, vp, one, one + 1)
    kp, vp = (torch.zeros((4, 0, 16, 64), dtype=F16, device="cuda") for _ in range(2))
    rows = torch.zeros((1, 0, 64), dtype=F16, device="cuda")
    with pytest.raises(ValueError, match="one head"):
        jasper.append_tokens(None, rows, rows, None, one, None, None, kp, vp)


def test_every_position_is_outside_of_empty_tables(jasper):
    cos, sin = jasper.rotary_table(0, 32)
    q = randn((3, 2, 48), F16, 320)
    y, _ = jasper.rotary(q, None, torch.arange(3, device="cuda"), cos, sin)
    assert y[..., :32].isnan().all() and torch.equal(y[..., 32:], q[..., 32:])


@pytest.mark.filterwarnings("ignore")
def test_what_has_no_memory_is_refused_and_compiled_code_calls_through(jasper):
    from torch._subclasses.fake_tensor import FakeTensorMode
    q, k = randn((3, 4, 64), F16, 330), randn((3, 2, 64), F16, 331)
    kp, vp = make_pages(4, 2, 16, 64, F16, seed=332)
    at = torch.arange(3, device="cuda")
    cos, sin = jasper.rotary_table(8, 64)
    tables, lens = torch.zeros((3, 1), dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    ids = torch.zeros((3, 2, 1), dtype=torch.int32, device="cuda")
    calls = [lambda q, k: jasper.rotary(q, k, at, cos, sin)[0],
             lambda q, k: jasper.append_tokens(q, k, k, at, at, cos, sin, kp, vp),
             lambda q, k: jasper.decode_attention(q, kp, vp, tables, lens),
             lambda q, k: jasper.retrieved_attention(q, kp, vp, tables, lens, ids)]
    module = jasper.kvcache._kv()
    for f in calls:
        want = f(q, k)
        twice = torch.compile(lambda q, k, f=f: 2 * f(q, k), backend="eager")
        assert torch.equal(twice(q, k), 2 * want)
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(torch.stack([q, q]), torch.stack([k, k]))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.jvp(lambda q, f=f: f(q, k), (q,), (q,))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.grad(lambda q, f=f: f(q, k).float().sum())(q)
        with FakeTensorMode() as mode, pytest.raises((RuntimeError, ValueError)):
            f(mode.from_tensor(q), mode.from_tensor(k))
    assert jasper.kvcache._kv() is module
    torch.cuda.synchronize()


@pytest.mark.parametrize("batch,heads,count,dim,cache", [(64, 8, 1300, 128, F16), (128, 8, 1700, 128, F8), (200, 4, 3000, 64, F16),
                                                         (130, 4, 900, 256, BF16)])
def test_lists_longer_than_a_wave_stages_at_once(jasper, batch, heads, count, dim, cache):
    """So many lists that a wave of a group has more tiles than it keeps row offsets of."""
    g = torch.Generator().manual_seed(340)
    lens = torch.randint(count, 2 * count, (batch,), generator=g).tolist()
    lens[3], lens[7] = 0, 40
    dtype = F16 if cache == F8 else cache
    pages = [-(-n // 16) for n in lens]
    total = sum(pages) + 1
    kp, vp = make_pages(total, heads, 16, dim, cache, seed=341)
    order = torch.randperm(total, generator=g)
    tables = torch.zeros((batch, max(pages)), dtype=torch.int32)
    for i, n in enumerate(pages):
        tables[i, :n] = order[sum(pages[:i]):sum(pages[:i]) + n].int()
    ks, vs = f8_scales(heads, cache, 342)
    q = randn((batch, heads, dim), dtype, 343, 2.0)
    ids = torch.stack([torch.stack([torch.randperm(max(lens), generator=g)[:count] for _ in range(heads)])
                       for _ in range(batch)]).int()
    out = jasper.retrieved_attention(q, kp, vp, tables.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), ids.cuda(),
                                     first=3, last=30, k_scale=ks, v_scale=vs, return_lse=True)
    some = [0, 3, 7, batch // 2, batch - 1]
    keys, values = [], []
    for i in some:
        mine = tables[i, :pages[i]].long().cuda()
        for held, store in ((keys, kp), (values, vp)):
            held.append(raw(store)[mine].view(cache).transpose(0, 1).reshape(heads, -1, dim)[:, :lens[i]].double().cpu())

    def choose(i, j):
        n = lens[some[i]]
        a, z = min(3, n), max(n - 30, min(3, n))
        mine = ids[some[i], j].long()
        return torch.cat([torch.arange(a), torch.arange(z, n), mine[(mine >= a) & (mine < z)]])

    at = torch.tensor(some, device="cuda")
    check([x[at] for x in out], ref_attention(q[at], keys, values, dim ** -0.5, choose, dtype, ks, vs, heads))


def test_threads_with_streams_of_their_own(jasper):
    import threading
    cos, sin = jasper.rotary_table(4000, 128)
    errors = []

    def work(x):
        try:
            lens = [3000 + x, 5, 700]
            kp, vp, tables, _, _ = build_cache(lens, 2, 16, 128, F16, 350 + x)
            q = randn((3, 8, 128), F16, 360 + x, 2.0)
            tens = torch.tensor(lens, dtype=torch.int32, device="cuda")
            ids = torch.randint(0, 700, (3, 2, 90), dtype=torch.int32, device="cuda")
            pos = tens.long() - 1

            def step():
                turned, _ = jasper.rotary(q, None, pos, cos, sin)
                return (turned, *jasper.decode_attention(turned, kp, vp, tables, tens, return_lse=True),
                        *jasper.retrieved_attention(turned, kp, vp, tables, tens, ids, first=2, last=9, return_lse=True))

            want = step()
            torch.cuda.current_stream().synchronize()
            stream = torch.cuda.Stream()
            for _ in range(30):
                with torch.cuda.stream(stream):
                    got = step()
                    with pytest.raises(ValueError):
                        jasper.decode_attention(q, kp, vp, tables[:1], tens)
                stream.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as e:  # noqa: BLE001  a thread's own error is told below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(x,)) for x in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("width", [8, 4000])
@pytest.mark.parametrize("step", [1.0, 2.0, 5.0])
def test_large_bf16_values_stay_finite(jasper, width, step):
    """Values near bf16's end, the later ones with the higher scores: no weight may be over one. So many sequences that
    a wave has several tiles of one, under short tables (a work-group to a stream) and wide ones."""
    n, batch = 120, 3000
    kp, vp = (torch.zeros((9, 1, 16, 64), dtype=BF16, device="cuda") for _ in range(2))
    tables = torch.zeros((batch, width), dtype=torch.int32, device="cuda")
    tables[:, :8] = torch.arange(1, 9)
    for i, t in enumerate((3, 50, 90)):
        page, row = 1 + t // 16, t % 16
        kp[page, 0, row, 0] = step * i
        vp[page, 0, row] = 1e38 * (1 - 0.1 * i)
    q = torch.zeros((batch, 2, 64), dtype=BF16, device="cuda")
    q[:, :, 0] = 1.0
    keys, values = ([x[1:].float().transpose(0, 1).reshape(1, -1, 64)[:, :n].double().cpu()] for x in (kp, vp))
    ref = ref_attention(q[:1], keys, values, 1.0, lambda i, j: torch.arange(n), BF16)
    out, lse = jasper.decode_attention(q, kp, vp, tables, torch.full((batch,), n, dtype=torch.int32, device="cuda"), scale=1.0,
                                       return_lse=True)
    for i in range(0, batch, 99):
        check((out[i:i + 1], lse[i:i + 1]), ref)
