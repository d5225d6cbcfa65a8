"""The paged cache's host side (no GPU): which pages sequences have, and the
rotary tables."""

import math

import numpy as np
import pytest
import torch

from jasper_amd.kvcache import PageTable, rotary_table


class Model:
    """Sequences as lists of tokens and pages as dicts: what PageTable has to keep true."""

    def __init__(self, table):
        self.table, self.tokens, self.memory, self.count = table, {}, {}, 0

    def read(self, seq):
        t = self.table
        return [self.memory[int(t.pages[seq, i // t.page_size]), i % t.page_size] for i in range(int(t.lens[seq]))]

    def extend(self, seqs, counts):
        positions, slots, copies, changed = self.table.extend(seqs, counts)
        ps = self.table.page_size
        for src, dst in copies:
            for r in range(ps):
                if (src, r) in self.memory:
                    self.memory[dst, r] = self.memory[src, r]
        at = 0
        for s, c in zip(seqs, counts):
            for i in range(c):
                assert positions[at] == len(self.tokens[s])
                self.count += 1
                self.memory[int(slots[at]) // ps, int(slots[at]) % ps] = self.count
                self.tokens[s].append(self.count)
                at += 1
        assert at == len(positions) == len(slots)
        for s, i, page in changed:
            assert self.table.pages[s, i] == page

    def check(self):
        t = self.table
        refs = np.zeros_like(t.refs)
        for s, tokens in self.tokens.items():
            assert t.lens[s] == len(tokens) and self.read(s) == tokens
            np.add.at(refs, t.pages[s, :-(-len(tokens) // t.page_size)], 1)
        assert np.array_equal(refs, t.refs)
        assert sorted(t._free) == np.flatnonzero(refs == 0).tolist()


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page", [1, 4, 16])
def test_page_table_against_a_model(seed, page):
    rng = np.random.default_rng(seed)
    t = PageTable(60, page, 9, 40)
    m = Model(t)
    refused = 0
    for _ in range(300):
        live = list(m.tokens)
        do = rng.integers(0, 10)
        if do < 2 and len(live) < 9:
            m.tokens[t.new()] = []
        elif do < 4 and live and len(live) < 9:
            s = int(rng.choice(live))
            m.tokens[t.fork(s)] = list(m.tokens[s])
        elif do < 8 and live:
            seqs = [int(x) for x in rng.permutation(live)[:rng.integers(1, len(live) + 1)]]
            counts = [int(x) for x in rng.integers(0, 2 * page + 2, len(seqs))]
            before = (t.pages.copy(), t.lens.copy(), t.refs.copy(), list(t._free))
            try:
                m.extend(seqs, counts)
            except (RuntimeError, ValueError):
                refused += 1
                for a, b in zip(before, (t.pages, t.lens, t.refs, t._free)):
                    assert np.array_equal(a, b)
                gone = int(rng.choice(live))
                t.free([gone])
                del m.tokens[gone]
        elif do == 8 and live:
            gone = [int(x) for x in rng.permutation(live)[:rng.integers(1, 3)]]
            t.free(gone)
            for s in gone:
                del m.tokens[s]
        else:
            src, dst = t.compact()
            assert not set(src.tolist()) & set(dst.tolist())
            for a, b in zip(src.tolist(), dst.tolist()):
                for r in range(page):
                    if (a, r) in m.memory:
                        m.memory[b, r] = m.memory[a, r]
            assert np.array_equal(np.flatnonzero(t.refs > 0), np.arange((t.refs > 0).sum()))
        m.check()
    assert refused or page > 1


def test_last_owner_keeps_its_page():
    t = PageTable(4, 8, 4, 4)
    a = t.new()
    t.extend([a], 5)
    b, c = t.fork(a), t.fork(a)
    assert t.refs[0] == 3
    _, _, copies, _ = t.extend([a, b, c], 1)  # three pages in all, with one free to spare
    assert len(copies) == 2 and t.n_free == 1 and sorted(t.pages[[a, b, c], 0].tolist()) == [0, 1, 2]
    d = t.fork(a)
    t.free([a])
    _, _, copies, _ = t.extend([d], 1)
    assert copies == []


def test_page_table_refusals():
    t = PageTable(4, 8, 2, 3)
    a = t.new()
    for seqs in ([a, a], [1], [-1], [2], [[a]]):
        with pytest.raises(ValueError):
            t.extend(seqs, 1)
    with pytest.raises(ValueError):
        t.extend([a], -1)
    with pytest.raises(ValueError, match="too large"):
        t.extend([a], 25)
    t.extend([a], 24)
    b = t.new()
    with pytest.raises(RuntimeError, match="out of pages"):
        t.extend([b], 9)
    with pytest.raises(RuntimeError, match="in use"):
        t.new()
    t.free(a)
    with pytest.raises(ValueError):
        t.free([a])
    t.extend([b], 9)
    with pytest.raises(ValueError):
        PageTable(0, 8, 1, 1)


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (96, 500000.0)])
def test_rotary_table_values(rot, base):
    cos, sin = rotary_table(1000, rot, base=base, device="cpu")
    assert cos.shape == sin.shape == (1000, rot // 2) and cos.dtype == sin.dtype == torch.float32
    for p in (0, 1, 7, 999):
        for i in range(rot // 2):
            angle = p * base ** (-2 * i / rot)
            # rounded once to 32 bits; the angle's own error: 2^-50 of up to 1000
            assert abs(cos[p, i] - math.cos(angle)) <= 2.0 ** -24
            assert abs(sin[p, i] - math.sin(angle)) <= 2.0 ** -24


def test_rotary_table_scalings():
    plain = rotary_table(4096, 64, device="cpu")
    linear = rotary_table(4096, 64, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(linear[0][::4], plain[0][:1024]) and torch.equal(linear[1][::4], plain[1][:1024])
    # ntk: the fastest pair is as it was, the slowest is divided by the factor
    ntk = rotary_table(4096, 64, scaling="ntk", factor=4.0, device="cpu")
    assert torch.equal(ntk[0][:, 0], plain[0][:, 0])
    slow = 10000.0 ** (-62 / 64) / 4
    want = torch.sin(torch.arange(4096, dtype=torch.float64) * slow)
    assert (ntk[1][:, 31].double() - want).abs().max() <= 2.0 ** -24 + 1e-12
    # yarn: pairs of many turns kept, of few divided, and the size 0.1 ln(factor) + 1
    size = 0.1 * math.log(4.0) + 1
    yarn = rotary_table(4096, 64, scaling="yarn", factor=4.0, original=2048, device="cpu")
    assert ((yarn[0][:, 0] - plain[0][:, 0] * size).abs() <= 2.0 ** -22).all()
    want = torch.sin(torch.arange(4096, dtype=torch.float64) * slow) * size
    assert (yarn[1][:, 31].double() - want).abs().max() <= 2.0 ** -22
    length = yarn[0].double() ** 2 + yarn[1].double() ** 2
    assert (length - size ** 2).abs().max() <= 2.0 ** -21
    one = rotary_table(100, 64, scaling="yarn", factor=1.0, original=2048, device="cpu")
    assert torch.equal(one[0], plain[0][:100])


def test_library_is_required_to_be_on_the_gpu():
    """Every operator refuses CPU tensors: there is no CPU form of them."""
    import jasper_amd
    from jasper_amd import build_lib
    if not build_lib.BINDING.exists():
        build_lib.build(verbose=False)
    x = torch.zeros((2, 2, 64), dtype=torch.float16)
    pages = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    i32, i64 = torch.zeros((2, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    cos, sin = rotary_table(4, 64, device="cpu")
    for f in (lambda: jasper_amd.rotary(x, x, i64, cos, sin),
              lambda: jasper_amd.append_tokens(x, x, x, i64, i64, cos, sin, pages, pages),
              lambda: jasper_amd.copy_pages(pages, pages, i32[:, 0], i32[:, 0]),
              lambda: jasper_amd.decode_attention(x, pages, pages, i32, i32[:, 0]),
              lambda: jasper_amd.retrieved_attention(x, pages, pages, i32, i32[:, 0], i32[:, :, None])):
        with pytest.raises(ValueError, match="CUDA tensor"):
            f()


@pytest.mark.parametrize("rot,base,original,factor", [
    (64, 10000.0, 131072, 4.0), (128, 10000.0, 131072, 4.0), (16, 10000.0, 32768, 4.0), (64, 10000.0, 2048, 16.0),
    (128, 500000.0, 8192, 8.0), (96, 10000.0, 10 ** 7, 2.0)])
def test_yarn_blends_between_its_two_bounds(rot, base, original, factor):
    """Every pair's frequency against the formula. The blend ends at the pair that turns beta_slow times within the
    original context, also where that is past the last pair: then no pair is divided outright."""
    cos, sin = rotary_table(2, rot, base=base, scaling="yarn", factor=factor, original=original, device="cpu")
    size = 1 + 0.1 * math.log(factor)

    def place(turns):  # where original * base^(-2i / rot) = 2 pi turns
        return rot / 2 * math.log(original / (2 * math.pi * turns), base)

    low, high = max(math.floor(place(32)), 0), min(math.ceil(place(1)), rot - 1)
    for i in range(rot // 2):
        plain = base ** (-2 * i / rot)
        divided = 0.0 if i <= low else 1.0 if i >= high else (i - low) / (high - low)
        want = plain * (1 - divided) + plain / factor * divided
        # sine and cosine of position 1 are rounded to 32 bits, 2^-24 of each: twice that in the angle's tangent
        got = math.atan2(sin[1, i].item(), cos[1, i].item())
        assert abs(got - want) <= 2.0 ** -22 * want, i
        assert abs(math.hypot(sin[1, i].item(), cos[1, i].item()) - size) <= 2.0 ** -23 * size
        if original * plain / (2 * math.pi) > 1:
            assert got > plain / factor * (1 + 2.0 ** -20), i


def test_cache_refuses_tables_of_no_pages():
    """max_pages 0 is no default."""
    from jasper_amd import PagedCache
    for bad in (0, -1):
        with pytest.raises(ValueError, match="max_pages"):
            PagedCache(4, 1, 2, 64, max_pages=bad, device="cpu")
    assert PagedCache(4, 1, 2, 64, device="cpu").tables.shape == (64, 4)
