"""GPU tests of PagedCache: sequences that grow, fork, are freed and compacted
read back what was appended to them, and the example that puts the operators
together."""

import importlib.util
import math
from pathlib import Path

import pytest
import torch

from tests.test_gpu_kvcache import F8, F16, check, ref_attention, ref_rotary

pytestmark = pytest.mark.gpu


class Reference:
    """Per sequence and layer the rows that should be in the cache, in 64 bits."""

    def __init__(self):
        self.rows = {}

    def add(self, seq, k, v):
        old = self.rows.get(seq)
        self.rows[seq] = (k, v) if old is None else tuple(torch.cat([a, b], dim=2) for a, b in zip(old, (k, v)))


@pytest.mark.parametrize("dtype,page,dim,rot", [(F16, 16, 64, 32), (F8, 8, 128, 128)])
def test_sequences_keep_their_tokens(jasper, dtype, page, dim, rot):
    layers, heads, hq = 3, 2, 4
    scales = {}
    if dtype == F8:
        scales = {x: torch.rand((layers, heads), device="cuda") * 0.02 + 0.02 for x in ("k_scale", "v_scale")}
    cache = jasper.PagedCache(90, layers, heads, dim, page_size=page, dtype=dtype, max_sequences=6, **scales)
    cache.k_pages.view(torch.uint8).fill_(0x7F)  # NaN in every type
    cache.v_pages.view(torch.uint8).fill_(0x7F)
    cos, sin = jasper.rotary_table(500, rot)
    g = torch.Generator().manual_seed(7)
    want, live = {}, []

    def grow(seqs, counts):
        step = cache.extend(seqs, counts)
        n = int(sum(counts))
        assert step.positions.numel() == step.slots.numel() == n
        for layer in range(layers):
            qkv = torch.randn((n, hq + 2 * heads, dim), generator=g).half().cuda()
            q, k, v = qkv.split([hq, heads, heads], dim=1)
            out = cache.append(layer, step, q, k, v, cos, sin)
            assert out.shape == q.shape
            held_k, held_v = (x[layer].float().transpose(1, 2).reshape(-1, heads, dim)[step.slots].double().cpu()
                              for x in (cache.k_pages, cache.v_pages))
            turned, _ = ref_rotary(k, step.positions, cos, sin, False)
            if dtype == F16:
                assert ((held_k - turned).abs() < 2.0 ** -8).all() and torch.equal(held_v, v.double().cpu())
            at = 0
            for s, c in zip(seqs, counts):
                old = want[s].get(layer)
                new = held_k[at:at + c].transpose(0, 1), held_v[at:at + c].transpose(0, 1)
                want[s][layer] = new if old is None else tuple(torch.cat(x, dim=1) for x in zip(old, new))
                at += c
        return step

    def read(step):
        q = torch.randn((len(step.seqs), hq, dim), generator=g).half().cuda()
        for layer in range(layers):
            keys = [want[s][layer][0] for s in step.seqs.tolist()]
            values = [want[s][layer][1] for s in step.seqs.tolist()]
            ks, vs = (scales[x][layer] if scales else None for x in ("k_scale", "v_scale"))
            ref = ref_attention(q, keys, values, dim ** -0.5, lambda i, j: torch.arange(keys[i].size(1)), F16, ks, vs)
            check(cache.decode(layer, step, q, return_lse=True), ref)
            ids = torch.arange(400, dtype=torch.int32, device="cuda").expand(len(keys), heads, 400).contiguous()
            check(cache.retrieved(layer, step, q, ids, first=2, last=5, return_lse=True), ref)

    def new():
        s = cache.new()
        want[s] = {}
        live.append(s)
        return s

    a, b = new(), new()
    grow([a, b], [37, 120])
    c = cache.fork(b)
    want[c] = dict(want[b])
    live.append(c)
    d = cache.fork(c)
    want[d] = dict(want[c])
    live.append(d)
    for _ in range(3):
        read(grow([d, a, b, c], [1, 2, 1, 1]))
    cache.free([b])
    live.remove(b)
    read(grow([a, c, d], [30, 1, 0]))
    f = new()
    assert f == b
    grow([f], [64])
    cache.free([a])  # the lowest pages among them: pages above take their places
    live.remove(a)
    assert cache.compact() > 0
    used = cache.k_pages.size(1) - cache.n_free
    cache.k_pages.view(torch.uint8)[:, used:] = 0x7F
    cache.v_pages.view(torch.uint8)[:, used:] = 0x7F
    read(grow([d, c, f], [0, 0, 0]))
    e = new()
    assert e == a
    read(grow([f, e, d], [1, 100, 3]))
    for layer in range(layers):
        got = cache.keys(layer, d).double().cpu()
        held = want[d][layer][0]
        if scales:
            held = (held * scales["k_scale"][layer].double().cpu()[:, None, None])
            assert ((got - held).abs() <= 2.0 ** -11 * 1.001 * held.abs() + 2.0 ** -24).all()
        else:
            assert torch.equal(got, held)
    assert cache.length(e) == 100
    before = cache.n_free
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.extend([c, e], [1200, 1000] if page == 16 else [500, 500])
    assert cache.n_free == before and cache.length(e) == 100
    cache.free(live)
    assert cache.n_free == 90


def test_paged_cache_refusals(jasper):
    for bad in (dict(page_size=12), dict(page_size=4), dict(dim=60), dict(dim=264), dict(dtype=torch.float32),
                dict(dim=72, dtype=F8), dict(k_scale=torch.ones(1, 2)), dict(n_layers=0),
                dict(dtype=F8, dim=64, k_scale=torch.ones(2))):
        args = dict(n_pages=4, n_layers=1, kv_heads=2, dim=64) | bad
        with pytest.raises(ValueError):
            jasper.PagedCache(**args)
    cache = jasper.PagedCache(4, 1, 2, 64, max_pages=2)
    with pytest.raises(ValueError, match="too large"):
        cache.extend([cache.new()], 33)


@pytest.mark.parametrize("exact", [False, True])
def test_example(jasper, exact):
    spec = importlib.util.spec_from_file_location("long_context", Path(__file__).parent.parent / "examples/long_context.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    args = ["--tokens", "3000", "--steps", "2", "--topics", "60", "--quiet"] + (["--exact"] if exact else [])
    weight, error = example.main(args)
    assert 0 < weight <= 1 + 1e-4 and math.isfinite(error)
    # every token read: the full attention itself, but for the types' rounding
    weight, error = example.main(args + ["--last", "4000"])
    assert abs(weight - 1) < 1e-4 and error < 2.0 ** -9


@pytest.mark.parametrize("dtype", [F16, torch.bfloat16, F8])
def test_keys_are_rows_for_an_index(jasper, dtype):
    """Whatever type the pages have, the index takes the keys: the search finds what the rows' products say."""
    heads, dim, n = 2, 64, 700
    rows_type = F16 if dtype == F8 else dtype
    scale = torch.tensor([[0.02, 0.03]], device="cuda") if dtype == F8 else None
    cache = jasper.PagedCache(50, 1, heads, dim, dtype=dtype, k_scale=scale)
    g = torch.Generator(device="cuda").manual_seed(11)
    k = torch.randn((n, heads, dim), device="cuda", generator=g).to(rows_type)
    seq = cache.new()
    cache.append(0, cache.extend([seq], n), None, k, k)
    keys = cache.keys(0, seq)
    assert keys.dtype == F16 and keys.shape == (heads, n, dim) and keys.is_contiguous()
    held = k.double().transpose(0, 1)
    if dtype == F8:  # to 4 bits of 448 scales' worth, then to fp16
        assert ((keys.double() - held).abs() <= held.abs() * (2.0 ** -4 + 2.0 ** -10) + 0.03 * 2.0 ** -9).all()
    else:  # bf16's 8 bits fit fp16's 11 but below its smallest normal value
        assert ((keys.double() - held).abs() <= 2.0 ** -25).all()
    q = torch.randn((5, dim), device="cuda", generator=g).half()
    for h in range(heads):
        found = jasper.bruteforce_knn(keys[h], q, 10, distance="ip")[0]
        products = q.double() @ keys[h].double().T
        best = products.topk(10, dim=1).values
        # products of 64 terms, summed in 32 bits and held in 16
        assert (products.gather(1, found.long()) >= best[:, -1:] - 2.0 ** -9 * best.abs().amax()).all()
        graph = jasper.Graph.build(keys[h], n_neighbors=32, distance="ip")
        assert graph.search(q, k=10)[0].shape == (5, 10)


def test_keys_past_the_range_of_float16(jasper):
    """bf16 keys reach further: rows for the index stay finite; what is no number stays so."""
    cache = jasper.PagedCache(4, 1, 1, 8, dtype=torch.bfloat16)
    k = torch.tensor([[1e38, -1e38, 65504.0, 66000.0, -70000.0, math.inf, -math.inf, math.nan]], device="cuda").bfloat16()
    seq = cache.new()
    cache.append(0, cache.extend([seq], 1), None, k[:, None], k[:, None])
    got = cache.keys(0, seq)[0, 0].tolist()
    assert got[:7] == [65504.0, -65504.0, 65504.0, 65504.0, -65504.0, math.inf, -math.inf] and math.isnan(got[7])


@pytest.mark.parametrize("exact", [False, True])
def test_example_reads_every_token_after_the_document(jasper, exact):
    """An answer longer than the window: with the whole document retrieved, nothing may be missing."""
    spec = importlib.util.spec_from_file_location("long_context", Path(__file__).parent.parent / "examples/long_context.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    weight, error = example.main(["--tokens", "100", "--k", "100", "--first", "100", "--last", "2", "--steps", "40",
                                  "--topics", "2", "--quiet"] + (["--exact"] if exact else []))
    assert abs(weight - 1) < 1e-4 and error < 2.0 ** -9
