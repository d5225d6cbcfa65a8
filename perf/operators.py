"""The key-value cache operators of jasper_amd, as cases that can be timed.

A case names an operator, its sizes and types:

  rotary     rotary(): positions turned into queries and keys, and the
             gradients back (a training step's two passes)
  append     append_tokens(): a serving step's new queries, keys and values,
             rotated, the keys and values written into the cache's pages
  pages      copy_pages(): pages of every layer copied (a fork) or moved with
             their table entries (compaction)
  decode     decode_attention(): one new token per sequence over its cache
  retrieved  retrieved_attention(): one new token over the first and last
             tokens and those an index returned

`plain_*` below are the operators in elementary torch operations, in 32 bits;
`exact` computes them in 64 bits. Data: normal keys and values, queries twice
as wide, so that a softmax over many tokens is neither flat nor one token.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn}
F8_MAX = 448.0


def listed():
    return [
        # A training batch of 4 sequences of 2048: rotary positions on 32
        # query and 8 key heads, forward and backward.
        {"name": "rotary-train", "op": "rotary", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "type": "bf16", "interleaved": False, "factor": 1.0},
        # A short batch of an odd length; neighbours are pairs, half of each
        # 96-value head is rotated, positions scaled down by 4.
        {"name": "rotary-partial", "op": "rotary", "tokens": 1021, "q_heads": 12, "kv_heads": 12, "dim": 96, "rot": 48,
         "type": "f16", "interleaved": True, "factor": 4.0},
        # One user's next token: a call's own latency.
        {"name": "append-token", "op": "append", "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "type": "bf16", "cache": "bf16", "page": 16, "interleaved": False},
        # A chunk of prompts, packed to an odd length, into a cache of 8 bits.
        {"name": "append-prompt", "op": "append", "tokens": 6007, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "type": "f16", "cache": "f8", "page": 32, "interleaved": False},
        # Two continuations of two answers: their last pages, in 32 layers.
        {"name": "pages-fork", "op": "pages", "layers": 32, "pages": 256, "moves": 4, "sequences": 0, "kv_heads": 8,
         "page": 16, "dim": 128, "cache": "bf16"},
        # A fragmented cache pulled together, its sequences' tables rewritten.
        {"name": "pages-compact", "op": "pages", "layers": 16, "pages": 2048, "moves": 513, "sequences": 64,
         "kv_heads": 8, "page": 16, "dim": 128, "cache": "f16"},
        # One short conversation: latency.
        {"name": "decode-one", "op": "decode", "batch": 1, "shortest": 700, "longest": 700, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "type": "f16", "cache": "f16", "page": 16, "window": 0},
        # A server's step: 48 sequences from a greeting to 8k tokens.
        {"name": "decode-batch", "op": "decode", "batch": 48, "shortest": 17, "longest": 8192, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "type": "bf16", "cache": "bf16", "page": 16, "window": 0},
        # Four long documents in a cache of 8 bits.
        {"name": "decode-long", "op": "decode", "batch": 4, "shortest": 131_000, "longest": 131_072, "q_heads": 64,
         "kv_heads": 8, "dim": 128, "type": "bf16", "cache": "f8", "page": 64, "window": 0},
        # A head of its own for every query, short heads, the last 1,000 tokens.
        {"name": "decode-window", "op": "decode", "batch": 17, "shortest": 1, "longest": 4096, "q_heads": 12,
         "kv_heads": 12, "dim": 64, "type": "f16", "cache": "f16", "page": 32, "window": 1000},
        # One user over 32k tokens, each query head with its own k = 100
        # neighbours among the keys.
        {"name": "retrieved-one", "op": "retrieved", "batch": 1, "shortest": 32_768, "longest": 32_768, "q_heads": 32,
         "kv_heads": 8, "lists": 32, "count": 100, "holes": 0, "first": 4, "last": 64, "dim": 128, "type": "f16",
         "cache": "f16", "page": 16},
        # A batch over up to 64k tokens, one list per key head, some of the
        # searches short of results.
        {"name": "retrieved-batch", "op": "retrieved", "batch": 24, "shortest": 20_000, "longest": 65_536,
         "q_heads": 32, "kv_heads": 8, "lists": 8, "count": 1000, "holes": 37, "first": 16, "last": 256, "dim": 128,
         "type": "bf16", "cache": "bf16", "page": 16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "pages", "decode", "retrieved"])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 10])
    c = {"op": op, "kv_heads": kv_heads, "dim": rng.choice([64, 80, 96, 128, 128, 256])}
    if op != "pages":
        c |= {"q_heads": kv_heads * rng.choice([1, 2, 3, 4, 8]), "type": rng.choice(["f16", "bf16"])}
    if op != "rotary":
        c["cache"] = rng.choice([c["type"] if op != "pages" else rng.choice(["f16", "bf16"])] * 2 + ["f8"])
        c["page"] = rng.choice([8, 16, 16, 32, 64])
    if op in ("rotary", "append"):
        c |= {"rot": c["dim"] // rng.choice([1, 1, 2]), "interleaved": rng.random() < 0.5}
    width = c["kv_heads"] * c["dim"]
    if op == "rotary":
        most = 8192 * 40 * 128 // (width + c["q_heads"] * c["dim"])
        c |= {"tokens": _log(rng, 1, min(16_384, most)), "factor": rng.choice([1.0, 1.0, 2.0, 8.0])}
    elif op == "append":
        c["tokens"] = _log(rng, 1, min(8192, 6007 * 48 * 128 // (2 * width + c["q_heads"] * c["dim"])))
    elif op == "pages":
        c |= {"layers": rng.choice([1, 2, 16, 32]), "sequences": rng.choice([0, 3, 64])}
        most = 16 * 513 * 16 * 8 * 128 // (c["layers"] * c["page"] * width)
        c["moves"] = _log(rng, 1, min(2000, most))
        c["pages"] = 4 * c["moves"] + rng.randrange(64)
    elif op == "decode":
        c["batch"] = _log(rng, 1, 128)
        most = 4 * 131_072 * 8 * 128 // (width * c["batch"]) // (1 if c["cache"] == "f8" else 2)
        c["longest"] = _log(rng, 1, min(200_000, most))
        c["shortest"] = rng.choice([c["longest"], max(1, c["longest"] // 7), 1])
        c["window"] = rng.choice([0, 0, 0, _log(rng, 1, 5000)])
    else:
        c["batch"] = _log(rng, 1, 32)
        most = 24 * 65_536 * 8 * 128 // (width * c["batch"])
        c["longest"] = _log(rng, 3000, min(150_000, most))
        c["shortest"] = rng.choice([c["longest"], c["longest"] // 3])
        c["lists"] = rng.choice([c["q_heads"], c["kv_heads"]])
        most = 24 * 8 * 1000 * 128 // (c["batch"] * c["lists"] * c["dim"])
        c["count"] = _log(rng, 1, max(1, min(most, 2000, c["shortest"] // 2)))
        c["holes"] = rng.choice([0, 0, c["count"] // 3])
        c |= {"first": rng.choice([0, 4, 16]), "last": rng.choice([0, 33, 256])}
    return c


def _lengths(case):
    """The sequences' lengths: evenly spread in their logarithm."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    if n == 1:
        return [hi]
    return [round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1))) for i in range(n)]


def _pages_of(case, lens):
    return [-(-n // case["page"]) for n in lens]


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


def _table(positions, rot, factor):
    """cos and sin of position / factor times 10000^(-2i / rot), [positions, rot / 2], made in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = (torch.arange(positions, dtype=torch.float64, device="cuda") / factor)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        dtype, n, hq = TYPES[case["type"]], case["tokens"], case["q_heads"]
        s["q"], s["gq"] = (_normal((n, hq, dim), dtype, gen) for _ in range(2))
        s["k"], s["gk"] = (_normal((n, heads, dim), dtype, gen) for _ in range(2))
        s["positions"] = torch.randint(0, 4096, (1,), device="cuda", generator=gen) + torch.arange(n, device="cuda") % 2048
        s["cos"], s["sin"] = _table(6144, case["rot"], case["factor"])
        return s
    if case["op"] == "append":
        dtype, n, hq = TYPES[case["type"]], case["tokens"], case["q_heads"]
        # the projection's output: queries, keys and values of a token side by side
        qkv = _normal((n, hq + 2 * heads, dim), dtype, gen)
        s["q"], s["k"], s["v"] = qkv.split([hq, heads, heads], dim=1)
        pages = -(-n // case["page"]) + 8
        s["k_pages"], s["v_pages"] = (torch.zeros((pages, heads, case["page"], dim), dtype=TYPES[case["cache"]],
                                                  device="cuda") for _ in range(2))
        start = torch.randint(0, 4096, (1,), device="cuda", generator=gen)
        s["positions"] = start + torch.arange(n, device="cuda")
        order = torch.randperm(pages, device="cuda", generator=gen)
        at = torch.arange(n, device="cuda")
        s["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        s["cos"], s["sin"] = _table(4096 + n, case["rot"], 1.0)
        s["k_scale"] = s["v_scale"] = None
        if case["cache"] == "f8":
            s["k_scale"], s["v_scale"] = (0.01 + 0.02 * torch.rand(heads, device="cuda", generator=gen)
                                          for _ in range(2))
        return s
    if case["op"] == "pages":
        shape = (case["layers"], case["pages"], heads, case["page"], dim)
        s["k_pages"], s["v_pages"] = (_normal(shape, TYPES[case["cache"]], gen) for _ in range(2))
        order = torch.randperm(case["pages"], device="cuda", generator=gen).int()
        s["src"], s["dst"] = order[:case["moves"]].clone(), order[case["moves"]:2 * case["moves"]].clone()
        s["tables"] = None
        if case["sequences"]:  # every page but the destinations has an owner
            kept = torch.cat([order[:case["moves"]], order[2 * case["moves"]:]])
            kept = kept[torch.randperm(kept.numel(), device="cuda", generator=gen)]
            wide = -(-kept.numel() // case["sequences"])
            s["tables"] = torch.full((case["sequences"] * wide,), -1, dtype=torch.int32, device="cuda")
            s["tables"][:kept.numel()] = kept
            s["tables"] = s["tables"].view(case["sequences"], wide)
        return s
    dtype, cache = TYPES[case["type"]], TYPES[case["cache"]]
    lens = _lengths(case)
    lens = [lens[i] for i in torch.randperm(len(lens), generator=torch.Generator().manual_seed(seed)).tolist()]
    count = _pages_of(case, lens)
    pages = sum(count) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).int()
    s["tables"] = torch.zeros((len(lens), max(count)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(count):
        s["tables"][i, :n] = order[at:at + n]
        at += n
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["q"] = _normal((len(lens), case["q_heads"], dim), dtype, gen, 2.0)
    s["k_scale"] = s["v_scale"] = None
    if case["cache"] == "f8":  # a value of deviation 1 is held as one of deviation 32
        s["k_scale"], s["v_scale"] = (0.02 + 0.02 * torch.rand(heads, device="cuda", generator=gen)
                                      for _ in range(2))
    wide = 32.0 if case["cache"] == "f8" else 1.0
    s["k_pages"], s["v_pages"] = (_normal((pages, heads, case["page"], dim), cache, gen, wide) for _ in range(2))
    if case["op"] == "retrieved":
        ids = torch.empty((len(lens), case["lists"], case["count"]), dtype=torch.int32, device="cuda")
        for i, n in enumerate(lens):
            ids[i] = torch.rand((case["lists"], n), device="cuda", generator=gen).topk(case["count"], dim=1).indices
        if case["holes"]:
            ids[::2, :, case["count"] - case["holes"]:] = -1
        s["ids"] = ids
    return s


# ---- the plain forms ----

def plain_rotary(x, positions, cos, sin, interleaved, back=False):
    """x [n, heads, dim] with its first 2 * cos.size(1) values of each head rotated; back: by the opposite angle."""
    c, t = cos[positions][:, None, :], sin[positions][:, None, :]
    if back:
        t = -t
    rot = 2 * cos.size(1)
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


def plain_append(s):
    _store(s["k_pages"], s["slots"], plain_rotary(s["k"], s["positions"], s["cos"], s["sin"], s["interleaved"]), s["k_scale"])
    _store(s["v_pages"], s["slots"], s["v"].float(), s["v_scale"])
    return plain_rotary(s["q"], s["positions"], s["cos"], s["sin"], s["interleaved"]).to(s["q"].dtype)


def plain_copy(s):
    kp, vp, src, dst = s["k_pages"], s["v_pages"], s["src"].long(), s["dst"].long()
    if kp.dtype == torch.float8_e4m3fn:
        kp, vp = kp.view(torch.uint8), vp.view(torch.uint8)
    kp[:, dst], vp[:, dst] = kp[:, src], vp[:, src]
    if s["tables"] is not None:
        to = torch.arange(kp.size(1), dtype=torch.int32, device="cuda")
        to[src] = s["dst"]
        s["tables"].copy_(torch.where(s["tables"] < 0, s["tables"], to[s["tables"].clamp(min=0).long()]))


def _attend(q, keys, values, valid, type_):
    """q [b, hq, d] over keys, values [b, h, t, d] (32 bits) where valid [b, h, t]; out and the scores' log of sums."""
    b, hq, d = q.shape
    h = keys.size(1)
    valid = valid[:, :, None, :]
    scores = torch.matmul(q.float().view(b, h, hq // h, d), keys.transpose(2, 3)) * d ** -0.5
    scores = torch.where(valid, scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    values = torch.where(valid.transpose(2, 3), values, 0.0)
    out = torch.matmul(p, values) / torch.where(total == 0, 1.0, total)
    return out.view(b, hq, d).to(type_), (top + torch.log(total)).view(b, hq)


def plain_decode(s):
    tables, lens, page = s["tables"].long(), s["lens"], s["page"]
    b, wide = tables.shape
    heads, dim = s["k_pages"].size(1), s["k_pages"].size(3)

    def rows(pages, scale):
        if pages.dtype == torch.float8_e4m3fn:
            x = pages.view(torch.uint8)[tables].view(torch.float8_e4m3fn)
        else:
            x = pages[tables]
        x = x.transpose(1, 2).reshape(b, heads, wide * page, dim).float()
        return x if scale is None else x.mul_(scale[None, :, None, None])

    at = torch.arange(wide * page, device="cuda")
    valid = at < lens[:, None]
    if s["window"]:
        valid &= at >= lens[:, None] - s["window"]
    valid = valid[:, None, :].expand(b, heads, wide * page)
    return _attend(s["q"], rows(s["k_pages"], s["k_scale"]), rows(s["v_pages"], s["v_scale"]), valid, s["q"].dtype)


def plain_retrieved(s):
    tables, lens, page, ids = s["tables"].long(), s["lens"][:, None, None], s["page"], s["ids"].long()
    b, lists, _ = ids.shape
    heads = s["k_pages"].size(1)
    first = torch.minimum(torch.full_like(lens, s["first"]), lens)
    last = torch.maximum(lens - s["last"], first)
    head = torch.arange(s["first"], device="cuda").expand(b, lists, -1)
    tail = torch.arange(s["last"], device="cuda") + last
    tail = tail.expand(b, lists, -1)
    at = torch.cat([head, tail, ids], dim=2)
    valid = torch.cat([head < first, tail < lens, (ids >= first) & (ids < last)], dim=2)
    at = torch.where(valid, at, 0)
    seq = torch.arange(b, device="cuda")[:, None, None]
    of = (torch.arange(lists, device="cuda") // (lists // heads))[None, :, None]
    pages, row = tables[seq, at // page], at % page

    def rows(store, scale):
        if store.dtype == torch.float8_e4m3fn:
            x = store.view(torch.uint8)[pages, of, row].view(torch.float8_e4m3fn).float()
        else:
            x = store[pages, of, row].float()
        return x if scale is None else x * scale[of][..., None]

    return _attend(s["q"], rows(s["k_pages"], s["k_scale"]), rows(s["v_pages"], s["v_scale"]), valid, s["q"].dtype)


def run_own(s):
    import jasper_amd

    if s["op"] == "rotary":
        q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        out = jasper_amd.rotary(q, k, s["positions"], s["cos"], s["sin"], interleaved=s["interleaved"])
        return list(out) + list(torch.autograd.grad(out, (q, k), (s["gq"], s["gk"])))
    if s["op"] == "append":
        q = jasper_amd.append_tokens(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["cos"], s["sin"],
                                     s["k_pages"], s["v_pages"], interleaved=s["interleaved"],
                                     k_scale=s["k_scale"], v_scale=s["v_scale"])
        return [q, s["k_pages"], s["v_pages"]]
    if s["op"] == "pages":
        jasper_amd.copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"], tables=s["tables"])
        return [s["k_pages"], s["v_pages"], s["tables"]]
    if s["op"] == "decode":
        return jasper_amd.decode_attention(
            s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], window=s["window"],
            k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True)
    return jasper_amd.retrieved_attention(
        s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["ids"], first=s["first"], last=s["last"],
        k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True)


def run(s):
    if own:
        return run_own(s)
    if s["op"] == "rotary":
        args = s["positions"], s["cos"], s["sin"], s["interleaved"]
        return [plain_rotary(s["q"], *args).to(s["q"].dtype), plain_rotary(s["k"], *args).to(s["k"].dtype),
                plain_rotary(s["gq"], *args, back=True).to(s["q"].dtype),
                plain_rotary(s["gk"], *args, back=True).to(s["k"].dtype)]
    if s["op"] == "append":
        return [plain_append(s), s["k_pages"], s["v_pages"]]
    if s["op"] == "pages":
        plain_copy(s)
        return [s["k_pages"], s["v_pages"], s["tables"]]
    return plain_decode(s) if s["op"] == "decode" else plain_retrieved(s)


def work(case):
    dim, heads = case["dim"], case["kv_heads"]
    if case["op"] == "rotary":
        values = case["tokens"] * (case["q_heads"] + heads) * dim
        table = 2 * min(case["tokens"], 2048) * case["rot"] // 2 * 4
        turned = case["tokens"] * (case["q_heads"] + heads) * case["rot"] // 2
        return {"bytes": 2 * 2 * values * 2 + table + 8 * case["tokens"], "flops": 2 * 6 * turned}
    held = 1 if case["cache"] == "f8" else 2
    if case["op"] == "append":
        n, hq = case["tokens"], case["q_heads"]
        size = n * dim * (2 * (2 * hq + 2 * heads) + 2 * heads * held) + n * (case["rot"] * 4 + 16)
        return {"bytes": size, "flops": 3 * n * (hq + heads) * case["rot"]}
    if case["op"] == "pages":
        size = 2 * 2 * case["layers"] * case["moves"] * heads * case["page"] * dim * held
        owned = case["pages"] - case["moves"] if case["sequences"] else 0
        return {"bytes": size + 2 * 4 * owned + 8 * case["moves"], "flops": 0}
    b, hq, lens = case["batch"], case["q_heads"], _lengths(case)
    ends = b * hq * (2 * 2 * dim + 4) + 4 * b
    if case["op"] == "decode":
        tokens = sum(min(n, case["window"] or n) for n in lens)
        return {"bytes": 2 * tokens * heads * dim * held + 4 * tokens // case["page"] + ends,
                "flops": 4 * tokens * hq * dim}
    found = case["count"] - case["holes"] / 2
    rows = sum(min(n, case["first"] + case["last"] + round(found * max(0, n - case["first"] - case["last"]) / n))
               for n in lens)
    return {"bytes": 2 * rows * case["lists"] * dim * held + 4 * b * case["lists"] * case["count"] + ends,
            "flops": 4 * rows * hq * dim}


# ---- 64 bits ----

def _exact_turn(x, positions, cos, sin, interleaved, sign):
    """The rotation as a product of complex numbers."""
    rot = 2 * cos.size(1)
    x = x.double()
    part = x[..., :rot].unflatten(-1, (rot // 2, 2)) if interleaved else x[..., :rot].unflatten(-1, (2, rot // 2)).mT
    turn = torch.complex(cos.double(), sign * sin.double())[positions].unsqueeze(1)
    y = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
    x = x.clone()
    x[..., :rot] = (y if interleaved else y.mT).flatten(-2)
    return x


def _exact_token(q, k, v, scale):
    """One sequence: q [h, g, d] over k, v [h, t, d]."""
    if k.size(1) == 0:
        return torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    score = torch.matmul(q, k.mT.contiguous()) * scale
    return torch.matmul(torch.softmax(score, dim=-1), v), torch.logsumexp(score, dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return None  # copies: nothing is computed
    if case["op"] == "rotary":
        args = s["positions"], s["cos"], s["sin"], case["interleaved"]
        return [_exact_turn(s["q"], *args, 1), _exact_turn(s["k"], *args, 1),
                _exact_turn(s["gq"], *args, -1), _exact_turn(s["gk"], *args, -1)]
    if case["op"] == "append":
        args = s["positions"], s["cos"], s["sin"], case["interleaved"], 1
        stores = []
        for rows, scale in ((_exact_turn(s["k"], *args), s["k_scale"]), (s["v"].double(), s["v_scale"])):
            if scale is not None:
                rows = rows / scale.double()[None, :, None]
            pages, heads, page, dim = s["k_pages"].shape
            store = torch.zeros((pages * page, heads, dim), dtype=torch.float64, device="cuda")
            store[s["slots"]] = rows.clamp(-F8_MAX, F8_MAX) if scale is not None else rows
            stores.append(store.view(pages, page, heads, dim).transpose(1, 2).contiguous())
        return [_exact_turn(s["q"], *args)] + stores
    b, hq, dim = s["q"].shape
    heads, outs, logs = case["kv_heads"], [], []
    for i, n in enumerate(s["lens"].tolist()):
        table = s["tables"][i, :-(-n // case["page"])].long()
        k, v = ((x.view(torch.uint8)[table].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[table])
                .transpose(0, 1).flatten(1, 2)[:, :n].double() for x in (s["k_pages"], s["v_pages"]))
        if s["k_scale"] is not None:
            k, v = k * s["k_scale"].double()[:, None, None], v * s["v_scale"].double()[:, None, None]
        q = s["q"][i].double()
        if case["op"] == "decode":
            begin = max(0, n - case["window"]) if case["window"] else 0
            o, l = _exact_token(q.view(heads, hq // heads, dim), k[:, begin:], v[:, begin:], dim ** -0.5)
            outs.append(o.reshape(hq, dim))
            logs.append(l.reshape(hq))
            continue
        lists = case["lists"]
        first, last = min(case["first"], n), max(n - case["last"], min(case["first"], n))
        always = list(range(first)) + list(range(last, n))
        q = q.view(lists, hq // lists, dim)
        for j in range(lists):
            at = s["ids"][i, j].long()
            at = torch.cat([torch.tensor(always, dtype=torch.int64, device="cuda"), at[(at >= first) & (at < last)]])
            h = j // (lists // heads)
            o, l = _exact_token(q[j][None], k[h][at][None], v[h][at][None], dim ** -0.5)
            outs.append(o.reshape(-1, dim))
            logs.append(l.reshape(-1))
    return [torch.cat(outs).view(b, hq, dim), torch.cat(logs).view(b, hq)]
