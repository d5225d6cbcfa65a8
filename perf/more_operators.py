"""Operators for batches that share a long prefix, for tables kept on the GPU and
for positions of several axes, as cases that can be timed.

A case names an operator, its sizes and types:

  shared  shared_attention(): one new token per sequence, where neighbours in
          the batch share their first tokens' pages, read once for all
  tables  extend_tables() and truncate_tables(): a step's new tokens given
          pages, slots and tables, and taken back (drafts that were rejected);
          with forks, fork_tables() and shared_prefixes() too
  rotary  rotary() with positions of several axes, and the gradients back
  append  append_tokens() with positions of several axes

`plain_*` below are the operators in elementary torch operations, in 32 bits;
`exact` computes them in 64 bits (tables are whole numbers and have no such
values). Data: normal keys and values, queries twice as wide, so that a softmax
over many tokens is neither flat nor one token.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn}
F8_MAX = 448.0


def listed():
    return [
        # Four continuations of one short conversation: latency.
        {"name": "shared-few", "op": "shared", "batch": 4, "groups": 1, "prefix_from": 2000, "prefix": 2000, "tail_from": 1, "tail": 40,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "type": "f16", "cache": "f16", "page": 16},
        # A server's step: 64 users of one long system prompt, each some way
        # into an answer.
        {"name": "shared-batch", "op": "shared", "batch": 64, "groups": 1, "prefix_from": 16_384, "prefix": 16_384,
         "tail_from": 5, "tail": 1500, "q_heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "cache": "bf16", "page": 16},
        # Seven documents of unlike lengths with one to eleven questions each;
        # a key head of its own for every query head.
        {"name": "shared-documents", "op": "shared", "batch": 41, "groups": 7, "prefix_from": 900, "prefix": 12_345,
         "tail_from": 1, "tail": 333, "q_heads": 12, "kv_heads": 12, "dim": 64, "type": "f16", "cache": "f16", "page": 32},
        # 16 samples of an answer about a book, in a cache of 8 bits.
        {"name": "shared-long", "op": "shared", "batch": 16, "groups": 1, "prefix_from": 131_000, "prefix": 131_000,
         "tail_from": 100, "tail": 700, "q_heads": 64, "kv_heads": 8, "dim": 128, "type": "bf16", "cache": "f8", "page": 64},
        # The next token of 48 sequences: latency.
        {"name": "tables-step", "op": "tables", "batch": 48, "forks": 0, "old_from": 17, "old": 8192, "new_from": 1, "new": 1, "pad": 0,
         "page": 16, "pages": 20_000, "sequences": 64, "width": 600},
        # 64 sequences forked into three drafts each, five tokens more of all,
        # every last page copied on its first write.
        {"name": "tables-drafts", "op": "tables", "batch": 64, "forks": 3, "old_from": 100, "old": 6000, "new_from": 5, "new": 5, "pad": 3,
         "page": 16, "pages": 30_000, "sequences": 300, "width": 384},
        # A burst of 700 prompts, admitted at once to a large cache.
        {"name": "tables-prompts", "op": "tables", "batch": 700, "forks": 0, "old_from": 0, "old": 0, "new_from": 1, "new": 4000,
         "pad": 100, "page": 16, "pages": 130_000, "sequences": 1024, "width": 256},
        # A training batch of 4 sequences of 2048 tokens with images: time,
        # height and width take 16, 24 and 24 of the 64 pairs.
        {"name": "axes-train", "op": "rotary", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "sections": "16 24 24", "type": "bf16", "interleaved": False, "cyclic": False},
        # A short batch of an odd length; the pairs are neighbours and are dealt
        # to the axes in turn, and 48 of each 80 values are rotated.
        {"name": "axes-partial", "op": "rotary", "tokens": 1021, "q_heads": 12, "kv_heads": 12, "dim": 80,
         "sections": "10 7 7", "type": "f16", "interleaved": True, "cyclic": True},
        # One user's next token: latency.
        {"name": "axes-token", "op": "append", "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "sections": "24 20 20", "type": "bf16", "cache": "bf16", "page": 16, "interleaved": False, "cyclic": True},
        # A video's tokens, of an odd number, into a cache of 8 bits.
        {"name": "axes-video", "op": "append", "tokens": 6007, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "sections": "16 24 24", "type": "f16", "cache": "f8", "page": 32, "interleaved": False, "cyclic": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["shared", "shared", "tables", "rotary", "append"])
    if op == "tables":
        page = rng.choice([8, 16, 16, 32, 64])
        forks = rng.choice([0, 0, 1, 3])
        batch = _log(rng, 1, 700 // (1 + forks))
        width = max(2, _log(rng, 8, 512) * 16 // page)
        old = _log(rng, 1, max(1, width * page // 2)) if rng.random() < 0.7 or forks else 0
        new = rng.choice([1, 1, rng.randrange(1, 9), _log(rng, 1, max(1, width * page - old))])
        new = min(new, max(1, 300_000 // (batch * (1 + forks))), width * page - old)
        pages = batch * (1 + forks) * (-(-(old + new) // page) + 1) + rng.randrange(1000)
        return {"op": op, "batch": batch, "forks": forks, "old_from": rng.choice([old, min(1, old)]), "old": old,
                "new_from": rng.choice([new, 1]), "new": new, "pad": rng.choice([0, 0, 17]), "page": page, "pages": pages,
                "sequences": batch * (1 + forks) + rng.randrange(100), "width": width}
    kv_heads = rng.choice([1, 2, 4, 5, 8, 10])
    c = {"op": op, "kv_heads": kv_heads, "q_heads": kv_heads * rng.choice([1, 2, 3, 4, 8]),
         "dim": rng.choice([64, 80, 96, 128, 128, 256]), "type": rng.choice(["f16", "bf16"])}
    if op != "rotary":
        c |= {"cache": rng.choice([c["type"], c["type"], "f8"]), "page": rng.choice([8, 16, 16, 32, 64])}
    width = c["kv_heads"] * c["dim"]
    if op == "shared":
        c["batch"] = _log(rng, 1, 128)
        c["groups"] = rng.choice([1, 1, 1 + c["batch"] // 4, 1 + c["batch"] // 16])
        most = 96_000 * 8 * 128 // width // (1 if c["cache"] == "f8" else 2)  # by the bytes of all prefixes
        most = min(most // c["groups"], 131_000 * 1024 * 128 // (c["batch"] * c["q_heads"] * c["dim"]), 131_000)
        longest = _log(rng, 1, max(1, most))
        c |= {"prefix_from": rng.choice([longest, max(1, longest // 5)]), "prefix": longest}
        tail = _log(rng, 1, max(1, min(3000, 64 * 500 * 8 * 128 // (width * c["batch"]))))
        c |= {"tail_from": rng.choice([1, tail]), "tail": tail}
        return c
    rot = c["dim"] // rng.choice([1, 1, 2])
    axes = rng.choice([2, 3, 3, 4])
    cuts = sorted(rng.randrange(rot // 2 + 1) for _ in range(axes - 1))
    sections = " ".join(str(b - a) for a, b in zip([0] + cuts, cuts + [rot // 2]))
    c |= {"sections": sections, "interleaved": rng.random() < 0.5,
          "cyclic": rng.random() < 0.5}
    if op == "rotary":
        c["tokens"] = _log(rng, 1, min(16_384, 8192 * 40 * 128 // (width + c["q_heads"] * c["dim"])))
    else:
        c["tokens"] = _log(rng, 1, min(8192, 6007 * 48 * 128 // (2 * width + c["q_heads"] * c["dim"])))
    return c


def _sections(case):
    return [int(n) for n in case["sections"].split()]


def _spread(case, name, n):
    """n numbers from the case's least to its largest, evenly spread in their logarithm."""
    lo, hi = case[name + "_from"], case[name]
    if not hi:
        return [0] * n
    lo = max(lo, 1)
    if n == 1 or lo == hi:
        return [hi] * n
    return [round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1))) for i in range(n)]


def _sizes(case):
    """The groups' sizes: unlike, all of at least one sequence."""
    n, k = case["batch"], case["groups"]
    cuts = [round(n * (i + 1) * (i + 2) / (k * (k + 1))) for i in range(k)]
    cuts = [max(c, i + 1) for i, c in enumerate(cuts)]
    cuts = [min(c, n - (k - 1 - i)) for i, c in enumerate(cuts)]
    return [b - a for a, b in zip([0] + cuts, cuts)]


def _prefixes(case):
    """The tokens each group shares: whole pages of its prompt; and the prompts' lengths."""
    prompts = _spread(case, "prefix", case["groups"])
    return [p // case["page"] * case["page"] for p in prompts], prompts


def _shuffled(x, seed):
    return [x[i] for i in torch.randperm(len(x), generator=torch.Generator().manual_seed(seed)).tolist()]


def _normal(shape, dtype, gen, scale=1.0):
    """Normal values of a type; 8-bit ones by way of 16 bits, in pieces."""
    if dtype != torch.float8_e4m3fn:
        return torch.randn(shape, dtype=dtype, device="cuda", generator=gen).mul_(scale)
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        part = flat[at:at + (1 << 28)]
        part.copy_(torch.randn(part.numel(), dtype=torch.float16, device="cuda", generator=gen).mul_(scale))
    return out


def _table(positions, rot):
    """cos and sin of position times 10000^(-2i / rot), [positions, rot / 2], made in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _grid(case, gen):
    """Positions [axes, tokens]: text, where all axes go on together, then images 28 wide and 20 high."""
    axes, n = len(_sections(case)), case["tokens"]
    start = torch.randint(0, 1000, (1,), device="cuda", generator=gen)
    at = torch.arange(n, device="cuda")
    text = n // 8
    i = (at - text).clamp(min=0)
    image = torch.stack([i // 560, i // 28 % 20, i % 28, i % 7][:axes])
    return torch.where(at < text, at, text + image) + start


def _pack(flags):
    """Truth values as the bits of int32 words, the lowest first."""
    n = -(-flags.numel() // 32)
    bits = torch.zeros(32 * n, dtype=torch.int64, device=flags.device)
    bits[:flags.numel()] = flags.long()
    word = (bits.view(n, 32) << torch.arange(32, device=flags.device)).sum(dim=1)
    return torch.where(word >= 1 << 31, word - (1 << 32), word).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "tables":
        return _prepare_tables(s, seed, gen)
    heads, dim, dtype, hq = case["kv_heads"], case["dim"], TYPES[case["type"]], case["q_heads"]
    if case["op"] == "shared":
        return _prepare_shared(s, seed, gen)
    s["sections"] = _sections(case)
    n, rot = case["tokens"], 2 * sum(s["sections"])
    s["positions"] = _grid(case, gen)
    s["cos"], s["sin"] = _table(1100 + n, rot)
    if case["op"] == "rotary":
        s["q"], s["gq"] = (_normal((n, hq, dim), dtype, gen) for _ in range(2))
        s["k"], s["gk"] = (_normal((n, heads, dim), dtype, gen) for _ in range(2))
        return s
    # the projection's output: queries, keys and values of a token side by side
    qkv = _normal((n, hq + 2 * heads, dim), dtype, gen)
    s["q"], s["k"], s["v"] = qkv.split([hq, heads, heads], dim=1)
    pages = -(-n // case["page"]) + 8
    s["k_pages"], s["v_pages"] = (torch.zeros((pages, heads, case["page"], dim), dtype=TYPES[case["cache"]],
                                              device="cuda") for _ in range(2))
    order = torch.randperm(pages, device="cuda", generator=gen)
    at = torch.arange(n, device="cuda")
    s["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
    s["k_scale"] = s["v_scale"] = None
    if case["cache"] == "f8":
        s["k_scale"], s["v_scale"] = (0.01 + 0.02 * torch.rand(heads, device="cuda", generator=gen) for _ in range(2))
    return s


def _prepare_shared(s, seed, gen):
    heads, dim, page, cache = s["kv_heads"], s["dim"], s["page"], TYPES[s["cache"]]
    sizes, (shared, prompts) = _sizes(s), _prefixes(s)
    s["sizes"], s["shared_of"] = sizes, shared
    tails = _shuffled(_spread(s, "tail", s["batch"]), seed)
    lens = [p for n, p in zip(sizes, prompts) for _ in range(n)]
    s["lengths"] = lens = [a + b for a, b in zip(lens, tails)]
    count = [-(-n // page) for n in lens]
    both = [x // page for n, x in zip(sizes, shared) for _ in range(n)]
    pages = sum(x // page for x in shared) + sum(c - b for c, b in zip(count, both)) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).int()
    s["tables"] = torch.zeros((s["batch"], max(count)), dtype=torch.int32, device="cuda")
    at = i = 0
    for n, x in zip(sizes, shared):
        first = order[at:at + x // page]
        at += x // page
        for j in range(i, i + n):
            s["tables"][j, :x // page] = first
            s["tables"][j, x // page:count[j]] = order[at:at + count[j] - x // page]
            at += count[j] - x // page
        i += n
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["groups"] = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], dtype=torch.int32, device="cuda")
    s["shared"] = torch.tensor(shared, dtype=torch.int32, device="cuda")
    s["q"] = _normal((s["batch"], s["q_heads"], dim), TYPES[s["type"]], gen, 2.0)
    s["k_scale"] = s["v_scale"] = None
    if s["cache"] == "f8":  # a value of deviation 1 is held as one of deviation 32
        s["k_scale"], s["v_scale"] = (0.02 + 0.02 * torch.rand(heads, device="cuda", generator=gen) for _ in range(2))
    wide = 32.0 if s["cache"] == "f8" else 1.0
    s["k_pages"], s["v_pages"] = (_normal((pages, heads, page, dim), cache, gen, wide) for _ in range(2))
    return s


def _prepare_tables(s, seed, gen):
    """A cache in use: sequences on pages anywhere, the rest free. A step's sequences are listed drafts first, the
    sequence that they were forked from after them."""
    n, page, per = s["batch"], s["page"], 1 + s["forks"]
    olds = _shuffled(_spread(s, "old", n), seed)
    rows = torch.randperm(s["sequences"], device="cuda", generator=gen)[:n * per].int()
    s["seqs"] = rows
    s["parents"] = rows.view(n, per)[:, -1:].expand(n, per - 1).reshape(-1).contiguous()
    s["children"] = rows.view(n, per)[:, :-1].reshape(-1).contiguous()
    count = [-(-x // page) for x in olds]
    order = torch.randperm(s["pages"], device="cuda", generator=gen).int()
    s["tables"] = torch.full((s["sequences"], s["width"]), -1, dtype=torch.int32, device="cuda")
    s["lens"] = torch.zeros(s["sequences"], dtype=torch.int32, device="cuda")
    owners = rows.view(n, per)[:, -1].long()
    at = torch.arange(s["width"], device="cuda")
    counts = torch.tensor(count, device="cuda")
    begin = counts.cumsum(0) - counts
    held = torch.where(at < counts[:, None], order[(begin[:, None] + at).clamp(max=s["pages"] - 1)], -1)
    s["tables"][owners] = held
    s["lens"][owners] = torch.tensor(olds, dtype=torch.int32, device="cuda")
    s["refs"] = torch.zeros(s["pages"], dtype=torch.int32, device="cuda")
    s["refs"][order[:sum(count)].long()] = 1
    s["free"] = _pack(s["refs"] == 0)
    news = _shuffled(_spread(s, "new", n * per), seed + 1)
    s["counts"] = torch.tensor(news, dtype=torch.int32, device="cuda")
    s["total"] = sum(news) + s["pad"]
    back = torch.zeros((n, per), dtype=torch.int32, device="cuda")
    back[:, -1] = s["lens"][owners]
    s["back"] = back.view(-1)  # drafts are given up, the others are as before
    return s


# ---- the plain forms ----

def axis_of(sections, cyclic):
    """The axis of each pair: section after section, or dealt in turn, each until it has its share."""
    if not cyclic:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def _angles(s):
    axis = torch.tensor(axis_of(s["sections"], s["cyclic"]), device="cuda")
    at = s["positions"][axis].T  # [tokens, pairs]
    pair = torch.arange(axis.numel(), device="cuda")
    return s["cos"][at, pair], s["sin"][at, pair]


def plain_turn(x, angles, interleaved, back=False):
    """x [n, heads, dim] with its first pairs rotated by angles (cos, sin) [n, pairs]; back: by the opposite ones."""
    c, t = (a[:, None, :] for a in angles)
    if back:
        t = -t
    rot = 2 * c.size(2)
    x = x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, v = a * c - b * t, b * c + a * t
    turned = torch.stack([u, v], dim=-1).flatten(-2) if interleaved else torch.cat([u, v], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _store(pages, slots, rows, scale):
    page = pages.size(2)
    if scale is not None:
        rows = (rows / scale[None, :, None]).clamp(-F8_MAX, F8_MAX)
    rows = rows.to(pages.dtype)
    if pages.dtype == torch.float8_e4m3fn:
        pages, rows = pages.view(torch.uint8), rows.view(torch.uint8)
    pages[slots // page, :, slots % page] = rows


def plain_rotary(s):
    angles, mode = _angles(s), s["interleaved"]
    return [plain_turn(s["q"], angles, mode).to(s["q"].dtype), plain_turn(s["k"], angles, mode).to(s["k"].dtype),
            plain_turn(s["gq"], angles, mode, True).to(s["q"].dtype),
            plain_turn(s["gk"], angles, mode, True).to(s["k"].dtype)]


def plain_append(s):
    angles, mode = _angles(s), s["interleaved"]
    _store(s["k_pages"], s["slots"], plain_turn(s["k"], angles, mode), s["k_scale"])
    _store(s["v_pages"], s["slots"], s["v"].float(), s["v_scale"])
    return [plain_turn(s["q"], angles, mode).to(s["q"].dtype), s["k_pages"], s["v_pages"]]


def plain_shared(s):
    """Group by group: the prefix once under all its sequences' queries, the rest sequence by sequence."""
    page, dim, heads = s["page"], s["dim"], s["kv_heads"]
    gh = s["q_heads"] // heads

    def rows(pages, table, scale):
        """[..., n] pages as [..., heads, n * page, dim]."""
        if pages.dtype == torch.float8_e4m3fn:
            x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn)
        else:
            x = pages[table]
        x = x.transpose(-4, -3).flatten(-3, -2).float()
        return x if scale is None else x * scale[:, None, None]

    outs, logs, i = [], [], 0
    for n, shared in zip(s["sizes"], s["shared_of"]):
        wide = -(-max(s["lengths"][i:i + n]) // page)
        table, lens, q = s["tables"][i:i + n, :wide].long(), s["lens"][i:i + n], s["q"][i:i + n].float() * dim ** -0.5
        first, rest = table[0, :shared // page], table[:, shared // page:]
        k0, v0 = rows(s["k_pages"], first, s["k_scale"]), rows(s["v_pages"], first, s["v_scale"])
        k1, v1 = rows(s["k_pages"], rest, s["k_scale"]), rows(s["v_pages"], rest, s["v_scale"])
        q = q.view(n, heads, gh, dim)
        s0 = torch.matmul(q.transpose(0, 1).reshape(heads, n * gh, dim), k0.transpose(1, 2).contiguous())
        s1 = torch.matmul(q, k1.transpose(2, 3).contiguous())
        valid = shared + torch.arange(k1.size(2), device="cuda") < lens[:, None]
        s1 = torch.where(valid[:, None, None, :], s1, -math.inf)
        s0 = s0.view(heads, n, gh, -1).transpose(0, 1)
        top = s1.amax(dim=-1, keepdim=True)
        if shared:
            top = torch.maximum(top, s0.amax(dim=-1, keepdim=True))
        p0, p1 = torch.exp(s0 - top), torch.exp(s1 - top)
        total = p0.sum(dim=-1, keepdim=True) + p1.sum(dim=-1, keepdim=True)
        v1 = torch.where(valid[:, None, :, None], v1, 0.0)
        o = torch.matmul(p0.transpose(0, 1).reshape(heads, n * gh, -1), v0).view(heads, n, gh, dim).transpose(0, 1)
        outs.append(((o + torch.matmul(p1, v1)) / total).reshape(n, s["q_heads"], dim).to(s["q"].dtype))
        logs.append((top + torch.log(total)).reshape(n, s["q_heads"]))
        i += n
    return [torch.cat(outs), torch.cat(logs)]


def plain_fork(tables, lens, refs, seqs, into, page):
    seqs, into = seqs.long(), into.long()
    have = (lens[seqs] + page - 1) // page
    mine = torch.arange(tables.size(1), device="cuda") < have[:, None]
    held = tables[seqs]
    tables[into] = torch.where(mine, held, tables[into])
    lens[into] = lens[seqs]
    refs.index_add_(0, held.clamp(min=0).flatten().long(), mine.flatten().int())


def plain_extend(s):
    """Requests in order, each first the page that it no longer shares, then its new ones: the lowest free pages."""
    tables, lens, refs, page, total = s["tables"], s["lens"], s["refs"], s["page"], s["total"]
    rows, counts = s["seqs"].long(), s["counts"].long()
    n, width = rows.numel(), tables.size(1)
    old = lens[rows].long()
    new = old + counts
    have, need = (old + page - 1) // page, (new + page - 1) // page
    held = tables[rows]
    last = held.gather(1, (have - 1).clamp(min=0)[:, None])[:, 0]
    growing = (counts > 0) & (old % page != 0) & (refs[last.clamp(min=0).long()] > 1)
    earlier = (last[:, None] == last) & growing & torch.ones((n, n), dtype=torch.bool, device="cuda").tril(-1)
    copied = growing & (refs[last.clamp(min=0).long()] - earlier.sum(dim=1) > 1)  # the last owner keeps the page
    take = need - have + copied
    begin = take.cumsum(0) - take
    free = ((s["free"][:, None] >> torch.arange(32, device="cuda")) & 1).flatten()[:refs.numel()]
    rank = free.cumsum(0) - 1
    order = torch.zeros(refs.numel() + 1, dtype=torch.int64, device="cuda")
    order.scatter_(0, torch.where(free == 1, rank, refs.numel()), torch.arange(refs.numel(), device="cuda"))
    order[-1] = 0
    # the step's tables: kept pages, the copy, new pages, -1
    at = torch.arange(width, device="cuda")
    fresh = at >= (have - copied.long())[:, None]
    given = order[(begin[:, None] + copied[:, None] + at - have[:, None]).clamp(0, refs.numel() - 1)].int()
    step = torch.where(at < need[:, None], torch.where(fresh, given, held), -1)
    src, dst = torch.where(copied, last, -1).int(), torch.where(copied, order[begin.clamp(max=refs.numel())], -1).int()
    # the cache's state
    refs.index_add_(0, last.clamp(min=0).long(), -copied.int())
    used = fresh & (at < need[:, None])
    refs.index_add_(0, step.clamp(min=0).flatten().long(), used.flatten().int())
    tables[rows] = torch.where(used, step, held)
    lens[rows] = new.int()
    s["free"].copy_(_pack(refs == 0))
    # the new tokens
    ends = counts.cumsum(0)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), ends])
    t = torch.arange(total, device="cuda")
    real = t < ends[-1]
    of = torch.searchsorted(ends, t, right=True).clamp(max=n - 1)
    positions = torch.where(real, old[of] + t - starts[of], 0)
    slots = torch.where(real, step[of, positions // page].long() * page + positions % page, -1)
    missing = (take.sum() - free.sum()).clamp(min=0).int().view(1)
    return [positions, slots, starts.int(), step, new.int(), src, dst, missing]


def plain_truncate(s):
    tables, lens, refs, page = s["tables"], s["lens"], s["refs"], s["page"]
    rows = s["seqs"].long()
    to = torch.minimum(s["back"], lens[rows])
    held = tables[rows]
    gone = torch.arange(tables.size(1), device="cuda") >= ((to + page - 1) // page)[:, None]
    refs.index_add_(0, held.clamp(min=0).flatten().long(), -(gone & (held >= 0)).flatten().int())
    tables[rows] = torch.where(gone, -1, held)
    lens[rows] = to
    s["free"].copy_(_pack(refs == 0))


def plain_prefixes(tables, lens, page):
    """Neighbours whose first pages are the same form a group; it shares the whole pages that all of them have."""
    n, width = tables.shape
    whole = torch.minimum(lens[1:], lens[:-1]) // page
    same = (tables[1:] == tables[:-1]) & (torch.arange(width, device="cuda") < whole[:, None])
    run = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), same.long().cumprod(dim=1).sum(dim=1)])
    group = (run == 0).long().cumsum(0) - 1
    groups = torch.full((n + 1,), n, dtype=torch.int32, device="cuda")
    groups.scatter_reduce_(0, group, torch.arange(n, dtype=torch.int32, device="cuda"), "amin")
    shared = torch.full((n,), 1 << 30, dtype=torch.int32, device="cuda")
    shared.scatter_reduce_(0, torch.where(run == 0, n - 1, group), torch.where(run == 0, 1 << 30, run * page).int(), "amin")
    # a group of one shares nothing
    return [groups, torch.where(groups[1:] - groups[:-1] > 1, shared, 0).int()]


def plain_tables(s):
    if s["forks"]:
        plain_fork(s["tables"], s["lens"], s["refs"], s["parents"], s["children"], s["page"])
    out = plain_extend(s)
    if s["forks"]:
        out += plain_prefixes(out[3], out[4], s["page"])
    plain_truncate(s)
    return out + [s["tables"], s["lens"], s["refs"], s["free"]]


def run_own(s):
    import jasper_amd

    if s["op"] == "shared":
        return list(jasper_amd.shared_attention(
            s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["groups"], s["shared"],
            k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True))
    if s["op"] == "tables":
        state = s["tables"], s["lens"], s["refs"], s["free"]
        if s["forks"]:
            jasper_amd.fork_tables(*state, s["parents"], s["children"], s["page"])
        out = list(jasper_amd.extend_tables(*state, s["seqs"], s["counts"], s["page"], s["total"]))
        if s["forks"]:
            out += jasper_amd.shared_prefixes(out[3], out[4], s["page"])
        jasper_amd.truncate_tables(*state, s["seqs"], s["back"], s["page"])
        return out + list(state)
    if s["op"] == "rotary":
        q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        out = jasper_amd.rotary(q, k, s["positions"], s["cos"], s["sin"], interleaved=s["interleaved"],
                                sections=s["sections"], cyclic=s["cyclic"])
        return list(out) + list(torch.autograd.grad(out, (q, k), (s["gq"], s["gk"])))
    q = jasper_amd.append_tokens(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["cos"], s["sin"], s["k_pages"],
                                 s["v_pages"], interleaved=s["interleaved"], k_scale=s["k_scale"],
                                 v_scale=s["v_scale"], sections=s["sections"], cyclic=s["cyclic"])
    return [q, s["k_pages"], s["v_pages"]]


def run(s):
    if own:
        return run_own(s)
    return {"shared": plain_shared, "tables": plain_tables, "rotary": plain_rotary, "append": plain_append}[s["op"]](s)


def work(case):
    page = case["page"] if "page" in case else 0
    if case["op"] == "tables":
        n = case["batch"] * (1 + case["forks"])
        tokens = sum(_spread(case, "new", n))
        olds = _spread(case, "old", case["batch"])
        kept = sum(-(-x // page) for x in olds) * (1 + case["forks"])
        given = -(-tokens // page) + case["forks"] * case["batch"]
        step = 4 * (kept + n * case["width"])  # read and written
        forked = 4 * 4 * kept * case["forks"] // (1 + case["forks"])  # entries and counts, read and written
        return {"bytes": 16 * tokens + step + forked + 4 * 4 * given + 6 * 4 * n + case["pages"] // 4, "flops": 0}
    dim, heads, hq = case["dim"], case["kv_heads"], case["q_heads"]
    if case["op"] == "shared":
        held = 1 if case["cache"] == "f8" else 2
        sizes, (shared, prompts) = _sizes(case), _prefixes(case)
        rest = sum(n * (p - x) for n, p, x in zip(sizes, prompts, shared)) + sum(_spread(case, "tail", case["batch"]))
        tokens = sum(shared) + rest
        seen = sum(n * x for n, x in zip(sizes, shared)) + rest
        return {"bytes": 2 * tokens * heads * dim * held + 4 * tokens // page + case["batch"] * hq * (2 * 2 * dim + 4),
                "flops": 4 * seen * hq * dim}
    n, pairs, axes = case["tokens"], sum(_sections(case)), len(_sections(case))
    indexes = 8 * n * axes
    if case["op"] == "rotary":
        values = n * (hq + heads) * dim
        return {"bytes": 2 * 2 * values * 2 + 2 * 4 * min(n, 1100) * pairs + indexes, "flops": 2 * 6 * n * (hq + heads) * pairs}
    held = 1 if case["cache"] == "f8" else 2
    size = n * dim * (2 * (2 * hq + 2 * heads) + 2 * heads * held)
    return {"bytes": size + 2 * 4 * min(n, 1100) * pairs + indexes + 8 * n, "flops": 6 * n * (hq + heads) * pairs}


# ---- 64 bits ----

def _exact_turn(x, s, sign):
    """The rotation as a product of complex numbers, an axis at a time."""
    axes = axis_of(s["sections"], s["cyclic"])
    rot = 2 * len(axes)
    x = x.double()
    part = x[..., :rot].unflatten(-1, (rot // 2, 2)) if s["interleaved"] else x[..., :rot].unflatten(-1, (2, rot // 2)).mT
    turn = torch.complex(s["cos"].double(), sign * s["sin"].double())
    angle = torch.empty((x.size(0), rot // 2), dtype=turn.dtype, device="cuda")
    for i, a in enumerate(axes):
        angle[:, i] = turn[:, i][s["positions"][a]]
    y = torch.view_as_real(torch.view_as_complex(part.contiguous()) * angle.unsqueeze(1))
    x = x.clone()
    x[..., :rot] = (y if s["interleaved"] else y.mT).flatten(-2)
    return x


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return [_exact_turn(s["q"], s, 1), _exact_turn(s["k"], s, 1), _exact_turn(s["gq"], s, -1),
                _exact_turn(s["gk"], s, -1)]
    if case["op"] == "append":
        stores = []
        for rows, scale in ((_exact_turn(s["k"], s, 1), s["k_scale"]), (s["v"].double(), s["v_scale"])):
            if scale is not None:
                rows = (rows / scale.double()[None, :, None]).clamp(-F8_MAX, F8_MAX)
            pages, heads, page, dim = s["k_pages"].shape
            store = torch.zeros((pages * page, heads, dim), dtype=torch.float64, device="cuda")
            store[s["slots"]] = rows
            stores.append(store.view(pages, page, heads, dim).transpose(1, 2).contiguous())
        return [_exact_turn(s["q"], s, 1)] + stores
    # every sequence by itself, over all of its own pages
    heads, dim, outs, logs = case["kv_heads"], case["dim"], [], []
    for i, n in enumerate(s["lengths"]):
        table = s["tables"][i, :-(-n // case["page"])].long()
        k, v = ((x.view(torch.uint8)[table].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[table])
                .transpose(0, 1).flatten(1, 2)[:, :n].double() for x in (s["k_pages"], s["v_pages"]))
        if s["k_scale"] is not None:
            k, v = k * s["k_scale"].double()[:, None, None], v * s["v_scale"].double()[:, None, None]
        score = torch.matmul(s["q"][i].double().view(heads, -1, dim), k.mT.contiguous()) * dim ** -0.5
        outs.append(torch.matmul(torch.softmax(score, dim=-1), v).view(-1, dim))
        logs.append(torch.logsumexp(score, dim=-1).view(-1))
    return [torch.stack(outs), torch.stack(logs)]
