"""GPU tests of the page tables kept on the GPU, against a model on the host
that does the same request by request: every number has to be the same."""

import random

import numpy as np
import pytest
import torch

from tests.test_gpu_kvcache import BF16, F16, randn
from tests.test_gpu_shared_attention import alike

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Model:
    """tables, lens and refs as lists, and the same as tensors for the calls."""

    def __init__(self, sequences, width, pages, page):
        self.page, self.width, self.pages = page, width, pages
        self.tables = np.full((sequences, width), -1, dtype=np.int64)
        self.lens, self.refs = np.zeros(sequences, dtype=np.int64), np.zeros(pages, dtype=np.int64)
        bits = np.packbits(np.arange(-(-pages // 32) * 32) < pages, bitorder="little").view(np.int32)
        self.gpu = [torch.full((sequences, width), -1, dtype=torch.int32, device="cuda"), ints([0] * sequences),
                    ints([0] * pages), torch.from_numpy(bits).cuda()]

    def count(self, n):
        return -(-n // self.page)

    def same(self):
        tables, lens, refs, free = (x.cpu().numpy() for x in self.gpu)
        assert np.array_equal(tables, self.tables) and np.array_equal(lens, self.lens) and np.array_equal(refs, self.refs)
        bits = np.unpackbits(free.view(np.uint8), bitorder="little")
        assert np.array_equal(bits[:self.pages], self.refs == 0) and not bits[self.pages:].any()

    def extend(self, seqs, counts, n_tokens, width=None):
        """The outputs as lists; the state changes only when all can be done."""
        width = self.width if width is None else width
        real = [(i, s, c) for i, (s, c) in enumerate(zip(seqs, counts)) if 0 <= s < len(self.lens)]
        bad = len({s for _, s, _ in real}) < len(real) or any(c < 0 for _, _, c in real)
        bad = bad or any(self.lens[s] + c > min(width, self.width) * self.page for _, s, c in real)
        bad = bad or sum(c for _, _, c in real) > n_tokens
        n = len(seqs)
        src, dst, missing = [-1] * n, [-1] * n, -1 if bad else 0
        if not bad:
            free = [p for p in range(self.pages) if self.refs[p] == 0]
            tables, refs, used = self.tables.copy(), self.refs.copy(), 0
            take = lambda k: free[k] if k < len(free) else -1  # noqa: E731
            for i, s, c in real:
                have, need = self.count(self.lens[s]), self.count(self.lens[s] + c)
                if c and self.lens[s] % self.page and refs[tables[s, have - 1]] > 1:
                    src[i], dst[i] = tables[s, have - 1], take(used)
                    refs[src[i]] -= 1
                    refs[dst[i]] = 1
                    tables[s, have - 1] = dst[i]
                    used += 1
                for j in range(have, need):
                    tables[s, j] = take(used)
                    refs[tables[s, j]] = 1
                    used += 1
            missing = max(0, used - len(free))
        if missing:
            src, dst, counts = [-1] * n, [-1] * n, [0] * n
        else:
            self.tables, self.refs = tables, refs
        positions, slots, starts = [], [], [0]
        step, lens = np.full((n, width), -1), [0] * n
        for i, (s, c) in enumerate(zip(seqs, counts)):
            if 0 <= s < len(self.lens):
                for t in range(self.lens[s], self.lens[s] + c):
                    positions.append(t)
                    slots.append(self.tables[s, t // self.page] * self.page + t % self.page)
                self.lens[s] += c
                lens[i] = self.lens[s]
                k = min(width, self.count(lens[i]))
                step[i, :k] = self.tables[s, :k]
            starts.append(len(positions))
        pad = n_tokens - len(positions)
        return positions + [0] * pad, slots + [-1] * pad, starts, step, lens, src, dst, [missing]

    def truncate(self, seqs, to):
        seen = set()
        for s, n in zip(seqs, to):
            if not 0 <= s < len(self.lens) or s in seen:
                continue
            seen.add(s)
            if not 0 <= n < self.lens[s]:
                continue
            for j in range(self.count(n), self.count(self.lens[s])):
                self.refs[self.tables[s, j]] -= 1
                self.tables[s, j] = -1
            self.lens[s] = n

    def fork(self, seqs, into):
        n = len(self.lens)
        ok = lambda x: 0 <= x < n  # noqa: E731
        pairs = []
        for i, (s, t) in enumerate(zip(seqs, into)):
            real = [(a, b) for a, b in zip(seqs, into) if ok(a) and ok(b)]
            if not ok(s) or not ok(t) or self.lens[t] or t in seqs or s in [b for _, b in real]:
                continue
            if t in [b for a, b in zip(seqs[:i], into[:i]) if ok(a) and ok(b)]:
                continue
            pairs.append((s, t))
        for s, t in pairs:
            k = self.count(self.lens[s])
            self.tables[t, :k] = self.tables[s, :k]
            self.lens[t] = self.lens[s]
            np.add.at(self.refs, self.tables[s, :k], 1)


def extend(jasper, m, seqs, counts, n_tokens, width=None):
    got = jasper.extend_tables(*m.gpu, ints(seqs), ints(counts), m.page, n_tokens, width)
    want = m.extend(seqs, counts, n_tokens, width)
    for name, a, b in zip(("positions", "slots", "starts", "tables", "lens", "src", "dst", "missing"), got, want):
        assert np.array_equal(a.cpu().numpy(), np.asarray(b).reshape(a.shape)), name
    m.same()
    return want[-1][0]


@pytest.mark.parametrize("sequences,width,pages,page,seed", [
    (6, 9, 40, 8, 1), (20, 30, 300, 16, 2), (40, 64, 1000, 32, 3), (3, 1, 2, 256, 4), (100, 40, 5000, 8, 5),
    (64, 200, 33, 64, 6)])
def test_a_life_of_a_table(jasper, sequences, width, pages, page, seed):
    """Random growth, cuts and forks; pages run out now and then, and what cannot be is asked for."""
    r = random.Random(seed)
    m = Model(sequences, width, pages, page)
    seen = set()
    for _ in range(60):
        what = r.random()
        n = r.randrange(1, sequences + 1)
        seqs = r.sample(range(sequences), n)
        if what < 0.5:
            most = r.choice([1, 1, 3, page, 3 * page])
            counts = [r.randrange(most + 1) for _ in seqs]
            if r.random() < 0.1:
                seqs[r.randrange(n)] = r.choice([-1, sequences, 2 ** 31 - 1, seqs[0]])
            total = sum(counts) + r.choice([0, 0, 5])
            if r.random() < 0.1:
                counts[r.randrange(n)] = r.choice([-1, -2 ** 31, width * page + 1, 2 ** 31 - 1])
            seen.add(min(1, extend(jasper, m, seqs, counts, total, r.choice([None, None, max(1, width // 2), width + 3]))))
        elif what < 0.75:
            to = [r.choice([0, int(m.lens[s]) // 2, int(m.lens[s]) + 1, -1]) for s in seqs]
            seqs = seqs + r.choice([[], seqs[:1], [-5, sequences]])
            to = to + [0] * (len(seqs) - len(to))
            jasper.truncate_tables(*m.gpu, ints(seqs), ints(to), page)
            m.truncate(seqs, to)
            m.same()
        else:
            into = [r.choice([s for s in range(-1, sequences + 1)]) for _ in seqs]
            jasper.fork_tables(*m.gpu, ints(seqs), ints(into), page)
            m.fork(seqs, into)
            m.same()
    assert 0 in seen


@pytest.mark.parametrize("batch,old,new,page,pages,pad", [
    (700, 0, 300, 16, 20_000, 10), (1500, 20, 1, 16, 5000, 0), (3000, 0, 9, 8, 70_001, 1), (2, 0, 50_000, 16, 7000, 0),
    (65, 100, 700, 64, 130_000, 17), (1025, 7, 2, 8, 4097, 0)])
def test_large_requests(jasper, batch, old, new, page, pages, pad):
    r = random.Random(7)
    width = -(-(old + new) // page) + 2
    m = Model(batch + 9, width, pages, page)
    seqs = r.sample(range(batch + 9), batch)
    if old:
        extend(jasper, m, seqs, [old] * batch, old * batch)
    counts = [r.randrange(1, new + 1) for _ in seqs]
    assert extend(jasper, m, seqs, counts, sum(counts) + pad) == 0
    jasper.truncate_tables(*m.gpu, ints(seqs[::2]), ints([old] * len(seqs[::2])), page)
    m.truncate(seqs[::2], [old] * len(seqs[::2]))
    m.same()
    assert extend(jasper, m, seqs[::2], counts[::2], sum(counts[::2])) == 0


@pytest.mark.parametrize("forks", [1, 3, 200, 4300])
def test_many_forks_of_one_page(jasper, forks):
    """All but the last owner that grows copy the page; more of them than are held at once."""
    m = Model(forks + 2, 2, forks + 10, 8)
    extend(jasper, m, [0], [11], 11)
    jasper.fork_tables(*m.gpu, ints([0] * forks), ints(list(range(1, forks + 1))), 8)
    m.fork([0] * forks, list(range(1, forks + 1)))
    m.same()
    some = list(range(0, forks + 1, 2))
    extend(jasper, m, some, [1] * len(some), len(some))
    everyone = list(range(forks + 1))[::-1]
    extend(jasper, m, everyone, [1] * len(everyone), len(everyone))
    assert m.refs.max() == forks + 1  # the first page is everyone's


def test_very_many_sequences_and_pages(jasper):
    """As many sequences as a call takes, and more pages than the bitmap's words that waves give out by themselves."""
    m = Model(2 ** 18, 3, 300_000, 8)
    seqs = [2 ** 18 - 1, 0, 131_071, 77]
    assert extend(jasper, m, seqs, [20, 1, 24, 9], 60) == 0
    assert extend(jasper, m, seqs[::-1], [1, 0, 7, 4], 12) == 0
    wide = Model(10, 20_000, 290_000, 8)
    assert extend(jasper, wide, [3, 9, 1], [150_000, 1, 77_777], 230_000) == 0
    jasper.truncate_tables(*wide.gpu, ints([3]), ints([9]), 8)
    wide.truncate([3], [9])
    assert extend(jasper, wide, [2, 3], [160_000, 100_001], 260_001) == 0


def ref_prefixes(tables, lens, page, least):
    groups, shared = [], []
    for b in range(len(lens)):
        run = 0
        if b:
            whole = min(max(0, lens[b]), max(0, lens[b - 1])) // page
            while run < min(whole, tables.shape[1]) and tables[b, run] == tables[b - 1, run]:
                run += 1
        if run and run * page >= least:
            shared[-1] = run * page if shared[-1] is None else min(shared[-1], run * page)
        else:
            groups.append(b)
            shared.append(None)
    k = len(lens) - len(groups)
    return groups + [len(lens)] * (k + 1), [s or 0 for s in shared] + [0] * k


@pytest.mark.parametrize("batch,width,page,seed", [(1, 5, 16, 1), (2, 40, 8, 2), (33, 70, 16, 3), (400, 30, 16, 4),
                                                   (90, 1500, 8, 5), (3000, 40, 32, 6)])
@pytest.mark.parametrize("least", [0, 1, 100])
def test_shared_prefixes(jasper, batch, width, page, seed, least):
    r = np.random.RandomState(seed)
    tables = np.empty((batch, width), dtype=np.int32)
    lens = np.empty(batch, dtype=np.int32)
    b = 0
    while b < batch:
        n = min(batch - b, r.choice([1, 1, 2, 5, 9, 70]))
        tables[b:b + n] = r.randint(0, 10 ** 6, (n, width))
        tables[b:b + n, :r.randint(0, width + 1)] = r.randint(0, 10 ** 6)
        lens[b:b + n] = r.choice([r.randint(0, width * page + 50), width * page], n)
        b += n
    lens[r.rand(batch) < 0.1] = r.choice([0, -1, 3])
    padded = torch.from_numpy(np.pad(tables, ((0, 0), (2, 1)))).cuda()
    got = jasper.shared_prefixes(padded[:, 2:-1], torch.from_numpy(lens).cuda(), page, least)
    want = ref_prefixes(tables, lens.tolist(), page, least)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]


def test_empty_calls(jasper):
    m = Model(4, 3, 10, 16)
    none = ints([])
    assert extend(jasper, m, [], [], 3) == 0
    jasper.truncate_tables(*m.gpu, none, none, 16)
    jasper.fork_tables(*m.gpu, none, none, 16)
    assert extend(jasper, m, [-1, 7], [5, 2 ** 31 - 1], 0) == 0
    m.same()
    groups, shared = jasper.shared_prefixes(m.gpu[0][:0], none, 16)
    assert groups.tolist() == [0] and shared.tolist() == []
    nothing = Model(2, 0, 0, 8)
    assert extend(jasper, nothing, [0, 1], [0, 0], 1) == 0
    assert extend(jasper, nothing, [0], [1], 1) == -1


def test_refusals(jasper):
    m = Model(4, 3, 40, 16)
    t, lens, refs, free = m.gpu
    s, c = ints([0, 1]), ints([1, 1])
    ext, cut, fork = jasper.extend_tables, jasper.truncate_tables, jasper.fork_tables
    bad = [
        lambda: ext(t.long(), lens, refs, free, s, c, 16, 2), lambda: ext(t, lens[:3], refs, free, s, c, 16, 2),
        lambda: ext(t, lens, refs, free[:1], s, c, 16, 2), lambda: ext(t, lens, refs.long(), free, s, c, 16, 2),
        lambda: ext(t, lens, refs, free, s, c[:1], 16, 2), lambda: ext(t, lens, refs, free, s.long(), c, 16, 2),
        lambda: ext(t, lens, refs, free, s, c, 12, 2), lambda: ext(t, lens, refs, free, s, c, 0, 2),
        lambda: ext(t, lens, refs, free, s, c, 512, 2), lambda: ext(t, lens, refs, free, s, c, 16, -1),
        lambda: ext(t, lens, refs, free, s, c, 16, 2 ** 31), lambda: ext(t, lens, refs, free, s, c, 16, 2, width=-1),
        lambda: ext(t, lens, refs, free, s, c, 16, 2, width=2 ** 28), lambda: ext(t.cpu(), lens, refs, free, s, c, 16, 2),
        lambda: ext(t, lens, refs, free, s.cpu(), c, 16, 2), lambda: ext(t.t(), lens[:3], refs, free, s, c, 16, 2),
        lambda: ext(t, lens, refs, free, ints([0] * 65536), ints([0] * 65536), 16, 2),
        lambda: cut(t, lens, refs, free, s, c[:1], 16), lambda: cut(t, lens, refs, free, s[None], c[None], 16),
        lambda: cut(t, lens, refs, free, s, c, 7), lambda: fork(t, lens, refs, free, s, c.long(), 16),
        lambda: fork(t, lens, refs, free, s, c.cpu(), 16), lambda: fork(t, lens, refs[:, None], free, s, c, 16),
        lambda: jasper.shared_prefixes(t, lens[:1], 16), lambda: jasper.shared_prefixes(t, lens, 10),
        lambda: jasper.shared_prefixes(t.long(), lens, 16), lambda: jasper.shared_prefixes(t, lens, 16, -1),
        lambda: jasper.shared_prefixes(t.t(), lens[:3], 16),
        lambda: jasper.GpuPagedCache(4, 1, 1, 64).extend(s, c, 2, max_len=-1),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    m.same()


def test_writes_in_place_are_counted(jasper):
    m = Model(4, 3, 40, 16)
    before = [x._version for x in m.gpu]
    extend(jasper, m, [0], [20], 20)
    jasper.fork_tables(*m.gpu, ints([0]), ints([1]), 16)
    jasper.truncate_tables(*m.gpu, ints([1]), ints([0]), 16)
    assert all(x._version > v for x, v in zip(m.gpu, before))


def test_a_captured_serving_loop(jasper):
    """Prompts, forks, drafts that are rejected and sequences that end, every step one replayed graph: the same bits as
    without one, and what a PagedCache on the host reads."""
    layers, heads, hq, dim, page, n = 2, 2, 8, 64, 16, 6
    cos, sin = jasper.rotary_table(600, 32)
    sections = (6, 5, 5)

    def cache():
        return jasper.GpuPagedCache(120, layers, heads, dim, page_size=page, dtype=F16, max_sequences=12, max_pages=20)

    def start(c):
        prompt = c.extend(ints([3, 8]), ints([150, 37]), 200)
        for layer in range(layers):
            k = randn((200, heads, dim), F16, 10 + layer)
            c.append(layer, prompt, None, k, randn((200, heads, dim), F16, 20 + layer), cos, sin,
                     positions=torch.stack([prompt.positions] * 3), sections=sections, cyclic=True)
        c.fork(ints([3, 3, 3, 8]), ints([0, 1, 2, 5]))

    seqs, counts, back = ints([0, 1, 2, 3, 5, 8]), ints([0] * n), ints([0] * n)
    qkv = torch.zeros((layers, 4 * n, hq + 2 * heads, dim), dtype=F16, device="cuda")

    def step(c):
        s = c.extend(seqs, counts, 4 * n)
        prefixes = c.prefixes(s)
        outs = [s.tables, s.lens, s.slots, s.missing, *prefixes]
        for layer in range(layers):
            q, k, v = qkv[layer].split([hq, heads, heads], dim=1)
            q = c.append(layer, s, q, k, v, cos, sin, positions=torch.stack([s.positions] * 3), sections=sections,
                         cyclic=True)
            q = q.index_select(0, (s.starts[1:].long() - 1).clamp(min=0))  # each sequence's last token
            outs += [*c.shared(layer, s, q, prefixes, return_lse=True), *c.decode(layer, s, q, return_lse=True)]
        c.truncate(seqs, back)
        return outs

    eager, captured, warm = cache(), cache(), cache()
    for c in (eager, captured, warm):
        for x in (c.k_pages, c.v_pages):
            x.zero_()
        start(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(captured)
    r = random.Random(1)
    lens = [150, 150, 150, 150, 37, 37]
    for i in range(7):
        new = [r.randrange(1, 5) for _ in range(n)]
        keep = [a + r.randrange(1, b + 1) for a, b in zip(lens, new)]  # drafts that were rejected
        lens = keep
        counts.copy_(ints(new))
        back.copy_(ints(keep))
        qkv.copy_(randn(qkv.shape, F16, 40 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        want = step(eager)
        torch.cuda.synchronize()
        for j, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (i, j)
        assert got[3].item() == 0 and got[4].tolist() == [0, 4] + [n] * 5 and got[5][:2].tolist() == [144, 32]
        for x, y in zip(eager._state() + (eager.k_pages, eager.v_pages), captured._state() + (captured.k_pages, captured.v_pages)):
            assert torch.equal(x, y)
        for layer in range(layers):
            shared, decode = got[6 + 4 * layer:8 + 4 * layer], got[8 + 4 * layer:10 + 4 * layer]
            alike(shared, decode, F16)
    assert [captured.length(s) for s in seqs.tolist()] == lens
    assert captured.keys(0, 8).shape == (heads, lens[-1], dim)
    captured.free(seqs)
    assert captured.n_free == 120


def test_a_full_cache_stores_nothing(jasper):
    cache = jasper.GpuPagedCache(4, 1, 1, 64, page_size=16, dtype=BF16, max_sequences=4)
    step = cache.extend(ints([0, 1]), ints([40, 30]), 70)
    assert step.missing.item() == 1 and (step.slots == -1).all() and step.lens.tolist() == [0, 0] and cache.n_free == 4
    for x in (cache.k_pages, cache.v_pages):
        x.zero_()
    cache.append(0, step, None, randn((70, 1, 64), BF16, 1), randn((70, 1, 64), BF16, 2))
    assert not cache.k_pages.any() and not cache.v_pages.any()
    out = cache.decode(0, step, randn((2, 2, 64), BF16, 3))
    assert (out == 0).all()
    with pytest.raises(NotImplementedError):
        cache.compact()
    with pytest.raises(NotImplementedError):
        cache.new()
