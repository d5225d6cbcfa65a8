"""GPU tests of rotary positions with several axes, against 64-bit ones pair by
pair; bounds as in tests/test_gpu_kvcache.py."""

import pytest
import torch

from tests.test_gpu_kvcache import BF16, F8, F16, make_pages, near, randn, raw, rotary_tol

pytestmark = pytest.mark.gpu


def axes(sections, cyclic):
    """The axis of each pair."""
    if not cyclic:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while sum(left):
        for a in range(len(left)):
            if left[a] > 0:
                out.append(a)
                left[a] -= 1
    return out


def ref_axes(x, positions, cos, sin, sections, cyclic, interleaved, back=False):
    """(value, size of the sums) in 64 bits on the CPU; positions [axes, ...]."""
    x, positions = x.double().cpu(), positions.cpu().long()
    y, size = x.clone(), torch.zeros_like(x)
    half = cos.size(1)
    for i, a in enumerate(axes(sections, cyclic)):
        c = cos[:, i].double().cpu()[positions[a]][..., None]
        s = sin[:, i].double().cpu()[positions[a]][..., None] * (-1 if back else 1)
        u, v = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y[..., u] = x[..., u] * c - x[..., v] * s
        y[..., v] = x[..., v] * c + x[..., u] * s
        size[..., u] = (x[..., u] * c).abs() + (x[..., v] * s).abs()
        size[..., v] = (x[..., v] * c).abs() + (x[..., u] * s).abs()
    return y, size


CASES = [
    ((16, 24, 24), False), ((24, 20, 20), True), ((1, 62, 1), True), ((64,), False), ((64,), True), ((0, 64), False),
    ((32, 32), True), ((16, 16, 16, 16), True), ((13, 0, 40, 11), True), ((5, 59, 0, 0), False), ((0, 0, 0, 64), True)]


@pytest.mark.parametrize("sections,cyclic", CASES)
@pytest.mark.parametrize("interleaved,dtype,idx", [(False, F16, torch.int64), (True, BF16, torch.int32)])
def test_values(jasper, sections, cyclic, interleaved, dtype, idx):
    cos, sin = jasper.rotary_table(3000, 128)
    q, k = randn((200, 6, 160), dtype, 1), randn((200, 2, 160), dtype, 2)
    pos = torch.randint(0, 3000, (len(sections), 200), device="cuda", dtype=idx)
    out = jasper.rotary(q, k, pos, cos, sin, interleaved=interleaved, sections=sections, cyclic=cyclic)
    for x, y in ((q, out[0]), (k, out[1])):
        want, size = ref_axes(x, pos, cos, sin, sections, cyclic, interleaved)
        near(y, want, rotary_tol(want, size, dtype))
        assert torch.equal(y[..., 128:], x[..., 128:])


@pytest.mark.parametrize("n,hq,hk,dim,sections,cyclic,interleaved", [
    (1, 1, 1, 2, (1, 0), False, False), (1, 8, 2, 64, (12, 10, 10), True, True), (7, 3, 3, 80, (7, 7, 6), False, False),
    (33, 12, 4, 96, (9, 8, 7), True, True), (1500, 5, 5, 128, (16, 8, 8), False, False),
    (2049, 2, 1, 256, (43, 43, 42), True, False), (300, 2, 1, 10, (1, 1, 1), True, False), (3, 1, 0, 34, (9, 8), True, True),
    (5, 70, 8, 256, (3, 40, 5), False, True), (9, 2, 2, 2048, (500, 300, 224), True, False)])
def test_sizes(jasper, n, hq, hk, dim, sections, cyclic, interleaved):
    cos, sin = jasper.rotary_table(500, 2 * sum(sections))
    q, k = randn((n, hq, dim), F16, 3), randn((n, hk, dim), F16, 4) if hk else None
    pos = torch.randint(0, 500, (len(sections), n), device="cuda")
    out = jasper.rotary(q, k, pos, cos, sin, interleaved=interleaved, sections=sections, cyclic=cyclic)
    for x, y in ((q, out[0]), (k, out[1])):
        if x is not None:
            want, size = ref_axes(x, pos, cos, sin, sections, cyclic, interleaved)
            near(y, want, rotary_tol(want, size, F16))


def test_one_position_for_all_axes_is_one_axis(jasper):
    cos, sin = jasper.rotary_table(400, 64)
    q = randn((3, 50, 4, 96), BF16, 5)
    pos = torch.randint(0, 400, (3, 50), device="cuda")
    want, _ = jasper.rotary(q, None, pos, cos, sin)
    for sections, cyclic in (((10, 12, 10), False), ((10, 12, 10), True), ((32,), False)):
        got, _ = jasper.rotary(q, None, torch.stack([pos] * len(sections)), cos, sin, sections=sections, cyclic=cyclic)
        assert torch.equal(got, want)


def test_tables_put_together_give_axes_their_own_frequencies(jasper):
    parts = [jasper.rotary_table(90, 2 * s) for s in (8, 12, 12)]
    cos, sin = (torch.cat([p[i] for p in parts], dim=1).contiguous() for i in range(2))
    q = randn((40, 2, 64), F16, 6)
    pos = torch.randint(0, 90, (3, 40), device="cuda")
    got, _ = jasper.rotary(q, None, pos, cos, sin, interleaved=True, sections=(8, 12, 12))
    at = 0
    for (c, s), n, p in zip(parts, (8, 12, 12), pos):
        want, _ = jasper.rotary(q[..., 2 * at:2 * at + 2 * n].contiguous(), None, p, c, s, interleaved=True)
        assert torch.equal(got[..., 2 * at:2 * at + 2 * n], want)
        at += n


def test_a_position_outside_is_its_axis_s_affair(jasper):
    cos, sin = jasper.rotary_table(10, 32)
    q = randn((3, 2, 48), BF16, 7)
    pos = torch.tensor([[0, 9, 10], [-1, 3, 3], [2 ** 40, 2, 1]], device="cuda")
    y, _ = jasper.rotary(q, None, pos, cos, sin, sections=(6, 6, 4))
    of = torch.tensor(axes((6, 6, 4), False) * 2, device="cuda")
    assert y[0][:, :32][:, of == 0].isfinite().all() and y[0][:, :32][:, of != 0].isnan().all()
    assert y[1].isfinite().all()
    assert y[2][:, :32][:, of == 0].isnan().all() and y[2][:, :32][:, of != 0].isfinite().all()
    assert torch.equal(y[..., 32:], q[..., 32:])


@pytest.mark.parametrize("sections,cyclic,interleaved", [((6, 5, 5), True, False), ((8, 8), False, True)])
def test_gradients(jasper, sections, cyclic, interleaved):
    """Against the formula's and, the rotation being linear, against differences."""
    cos, sin = jasper.rotary_table(100, 32)
    q, k = randn((30, 4, 40), BF16, 8).requires_grad_(), randn((30, 2, 40), BF16, 9).requires_grad_()
    pos = torch.randint(0, 100, (len(sections), 30), device="cuda")
    call = lambda a, b: jasper.rotary(a, b, pos, cos, sin, interleaved=interleaved, sections=sections, cyclic=cyclic)  # noqa: E731
    out = call(q, k)
    gq, gk = randn(q.shape, BF16, 10), randn(k.shape, BF16, 11)
    grads = torch.autograd.grad(out, (q, k), (gq, gk), retain_graph=True)
    for g, got in zip((gq, gk), grads):
        want, size = ref_axes(g, pos, cos, sin, sections, cyclic, interleaved, back=True)
        near(got, want, rotary_tol(want, size, BF16))
    x, dx = q.detach().double().cpu(), randn(q.shape, BF16, 12).double().cpu()
    f = lambda x: (ref_axes(x, pos, cos, sin, sections, cyclic, interleaved)[0] * gq.double().cpu()).sum()  # noqa: E731
    change = (f(x + dx) - f(x - dx)) / 2
    # every gradient is off by half a step at most
    assert (change - (grads[0].double().cpu() * dx).sum()).abs() <= (2.0 ** -8 * grads[0].double().cpu().abs() * dx.abs()).sum() + 1e-3
    # twice: linear in the gradients too
    gq2 = gq.clone().requires_grad_()
    first, = torch.autograd.grad(call(q, None)[0], q, gq2, create_graph=True)
    back, = torch.autograd.grad(first, gq2, gq)
    want, size = ref_axes(gq, pos, cos, sin, sections, cyclic, interleaved)
    near(back, want, rotary_tol(want, size, BF16))
    # broadcast gradients, only one of the two wanted
    only, = torch.autograd.grad(call(q.detach(), k)[1].sum(), k)
    want, size = ref_axes(torch.ones(k.shape), pos, cos, sin, sections, cyclic, interleaved, back=True)
    near(only, want, rotary_tol(want, size, BF16))


def test_forward_mode(jasper):
    cos, sin = jasper.rotary_table(100, 32)
    q, dq = randn((9, 2, 40), F16, 13), randn((9, 2, 40), F16, 14)
    pos = torch.randint(0, 100, (3, 9), device="cuda")
    with torch.autograd.forward_ad.dual_level():
        y, _ = jasper.rotary(torch.autograd.forward_ad.make_dual(q, dq), None, pos, cos, sin, sections=(6, 5, 5))
        value, tangent = torch.autograd.forward_ad.unpack_dual(y)
    assert torch.equal(value, jasper.rotary(q, None, pos, cos, sin, sections=(6, 5, 5))[0])
    assert torch.equal(tangent, jasper.rotary(dq, None, pos, cos, sin, sections=(6, 5, 5))[0])


@pytest.mark.parametrize("n,hq,heads,dim,sections,cyclic,interleaved,dtype,cache,page", [
    (1, 32, 8, 128, (24, 20, 20), True, False, BF16, BF16, 16), (77, 4, 2, 64, (10, 11, 11), False, True, F16, F16, 8),
    (300, 16, 2, 128, (8, 12, 12), True, False, BF16, F8, 32), (45, 5, 5, 80, (7, 6, 7), True, False, F16, F8, 16)])
def test_append(jasper, n, hq, heads, dim, sections, cyclic, interleaved, dtype, cache, page):
    """The same bits as rotary and an append without rotation."""
    cos, sin = jasper.rotary_table(2000, 2 * sum(sections))
    qkv = randn((n, hq + 2 * heads, dim), dtype, 15)
    q, k, v = qkv.split([hq, heads, heads], dim=1)
    pos = torch.randint(0, 2000, (len(sections), n), device="cuda")
    slots = torch.randperm(-(-n // page) * page, device="cuda")[:n]
    slots[::9] = -1
    scales = (torch.rand(heads, device="cuda") * 0.02 + 0.01,) * 2 if cache == F8 else (None, None)
    got, want = (make_pages(-(-n // page), heads, page, dim, cache) for _ in range(2))
    out = jasper.append_tokens(q, k, v, pos, slots, cos, sin, *got, interleaved=interleaved, k_scale=scales[0],
                               v_scale=scales[1], sections=sections, cyclic=cyclic)
    turned = jasper.rotary(q, k, pos, cos, sin, interleaved=interleaved, sections=sections, cyclic=cyclic)
    assert torch.equal(out, turned[0])
    if cache != F8:  # there the rotated key is rounded once, not twice
        jasper.append_tokens(None, turned[1], v, None, slots, None, None, *want)
        assert torch.equal(raw(got[0]), raw(want[0]))
    else:
        kept = slots >= 0
        held = got[0].float().transpose(1, 2).reshape(-1, heads, dim)[slots[kept]].double().cpu()
        value, size = ref_axes(k[kept], pos[:, kept], cos, sin, sections, cyclic, interleaved)
        s = scales[0].double().cpu()[None, :, None]
        near(held, (value / s).clamp(-448, 448), rotary_tol(value / s, size / s, F8))
    jasper.append_tokens(None, k, v, None, slots, None, None, *want, k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(raw(got[1]), raw(want[1]))


def test_graph_capture(jasper):
    cos, sin = jasper.rotary_table(300, 64)
    q, pos = randn((20, 4, 64), F16, 16), torch.randint(0, 300, (3, 20), device="cuda")
    call = lambda: jasper.rotary(q, None, pos, cos, sin, sections=(12, 10, 10), cyclic=True)[0]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        q.copy_(randn(q.shape, F16, 17 + i))
        pos.copy_(torch.randint(0, 300, pos.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def test_refusals(jasper):
    cos, sin = jasper.rotary_table(16, 64)
    q = randn((2, 4, 64), F16, 20)
    kp, vp = make_pages(8, 2, 16, 64, F16)
    k, slots = q[:, :2], torch.zeros(2, dtype=torch.int64, device="cuda")
    pos = torch.zeros((3, 2), dtype=torch.int64, device="cuda")
    f = lambda sections, pos=pos, **more: jasper.rotary(q, None, pos, cos, sin, sections=sections, **more)  # noqa: E731
    g = lambda sections, pos=pos, **more: jasper.append_tokens(q, k, k, pos, slots, cos, sin, kp, vp, sections=sections, **more)  # noqa: E731
    for call in (f, g):
        for bad in (lambda: call(()), lambda: call((10, 10, 11)), lambda: call((10, -2, 24)), lambda: call((8, 8, 8, 4, 4)),
                    lambda: call((16, 16)), lambda: call((32,)), lambda: call((10, 10, 12), pos=pos[:, :1]),
                    lambda: call((10, 10, 12), pos=pos.t().contiguous()), lambda: call((10, 10, 12), pos=pos.float()),
                    lambda: call(None, pos=pos[0], cyclic=True), lambda: call((2 ** 40, 1, 31)), lambda: call(None)):
            with pytest.raises(ValueError):
                bad()
    torch.cuda.synchronize()
