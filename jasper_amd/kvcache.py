"""A paged cache of a model's keys and values on the GPU, what fills it, and
the attention of a new token that reads all of it or what an index retrieved.

With a long context the keys of the tokens so far are rows like any others of
an index (`Graph`, `bruteforce_knn`): a new token's query heads search them by
inner product, and `retrieved_attention` attends to the tokens found. No
reference counterpart.

  rotary_table, rotary    rotary positions, with their gradient
  append_tokens           the same for a serving step, stored to the pages
  copy_pages              pages copied or moved, in all layers
  decode_attention        one new token per sequence over its whole cache
  retrieved_attention     over the first, the last and the retrieved tokens
  shared_attention        over the whole cache, where sequences share a prefix
  PagedCache              pages, sequences, forks and compaction put together
  extend_tables, truncate_tables, fork_tables
                          which sequence has which pages, kept on the GPU
  shared_prefixes         which sequences of a batch begin with the same pages
  GpuPagedCache           a PagedCache of which every step can be captured

Pages are [n_pages, kv_heads, page_size, dim] (with a leading layer dimension
where said) in float16, bfloat16 or float8_e4m3fn, any strides that keep a
row's dim values together and rows on 16 bytes. Calls run on the current
stream of the tensors' device, synchronize nothing and may be captured in a
graph (PagedCache's bookkeeping is on the host and is not captured,
GpuPagedCache's is). They take tensors with memory, and are not operators
registered with torch: torch.compile runs them as they are, between the graphs
before and after, and vmap, torch.func's grad and jvp, export and fake tensors
end in an error.
"""

from __future__ import annotations

import importlib.machinery
import importlib.util
import math
from collections.abc import Sequence

import numpy as np
import torch

_TYPES = (torch.float16, torch.bfloat16, torch.float8_e4m3fn)
_F8 = torch.float8_e4m3fn


_module = None


def _kv():
    """The module that takes tensors to the HIP library's calls (csrc/torch_kv.cpp)."""
    return _module or _load_kv()


def _load_kv():
    global _module
    from . import _load_lib, library_path
    _load_lib()
    path = library_path().parent / "_kv.so"
    if not path.exists():
        raise RuntimeError(f"{path} not found; build it with `python -m jasper_amd.build_lib` (there is no other way "
                           "to these operators)")
    loader = importlib.machinery.ExtensionFileLoader("jasper_amd._kv", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("jasper_amd._kv", loader))
    loader.exec_module(module)
    _module = module
    return module


# ---- rotary positions ----

def rotary_table(n_positions: int, rot_dim: int, base: float = 10000.0, scaling: str | None = None,
                 factor: float = 1.0, original: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device: str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """The tables (cos, sin) float32 [n_positions, rot_dim / 2] of rotary
    positions: position p turns pair i by p * base^(-2i / rot_dim).

    scaling stretches them to `factor` times the context a model was trained
    on: "linear" divides the positions; "ntk" raises the base so that the
    slowest pair is divided by factor and the fastest is kept; "yarn" (Peng et
    al. 2023) divides the pairs that turn less than beta_slow times within
    `original` positions, keeps those that turn more than beta_fast times,
    blends between, and scales the tables by 0.1 ln(factor) + 1. Angles are
    made in 64 bits: at position 100,000 a 32-bit angle is off by 0.004.
    """
    if n_positions < 0 or rot_dim <= 0 or rot_dim % 2:
        raise ValueError("n_positions must be at least 0 and rot_dim even and positive")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"Unknown scaling: {scaling!r}")
    if scaling is not None and factor < 1.0:
        raise ValueError("factor must be at least 1")
    pair = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    size = 1.0
    if scaling == "ntk" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = base ** (-pair / rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original is None or original <= 0:
            raise ValueError("yarn scaling needs the original context length")

        def at(turns):  # the pair that turns so many times within the original context
            return rot_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))

        low = max(0, math.floor(at(beta_fast)))
        # past the last pair where even that turns more often: the blend then ends there, undivided
        high = min(rot_dim - 1, math.ceil(at(beta_slow)))
        ramp = ((pair / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        size = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return (angle.cos() * size).float(), (angle.sin() * size).float()


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           interleaved: bool = False, sections: Sequence[int] | None = None, cyclic: bool = False):
    """(q, k) [..., heads, dim] (fp16 or bf16) with rotary positions: the
    first 2 * cos.size(1) values of every head are turned in pairs by the
    angles in row positions[...] of the tables (`rotary_table`), the rest is
    as it was. Pairs are (i, i + rot_dim / 2), or neighbours when interleaved.
    Differentiable in q and k, backward and forward (tables that require a
    gradient or carry a tangent are refused). k may be None. A position
    outside the tables gives NaN. Sums are in 32 bits, rounded once.

    sections: positions have up to four axes (time, height and width of an
    image's or a video's tokens), positions [axes, ...], and sections[a] pairs
    are turned by axis a's: axis after axis or, when cyclic, dealt to the axes
    in turn, each until it has its share (sections (2, 1, 1): axes 0 1 2 0).
    They are cos.size(1) in sum. Pair i reads column i of its axis's row, so
    tables put together from several (`torch.cat`) give each axis frequencies
    of its own.
    """
    return _kv().rotary(q, k, positions, cos, sin, interleaved, sections, cyclic)


# ---- the cache ----

def append_tokens(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor | None,
                  slots: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None, k_pages: torch.Tensor,
                  v_pages: torch.Tensor, interleaved: bool = False, k_scale: torch.Tensor | None = None,
                  v_scale: torch.Tensor | None = None, sections: Sequence[int] | None = None,
                  cyclic: bool = False) -> torch.Tensor | None:
    """Stores k (rotated as `rotary` does) and v [n, kv_heads, dim] to rows
    slots [n] of the pages (page * page_size + row; a slot outside the cache,
    such as -1, stores nothing) and returns q [n, heads, dim] rotated. q may
    be None; cos and sin None: nothing is rotated. float8_e4m3fn pages hold
    values divided by k_scale, v_scale [kv_heads] (float32, or None),
    rounded to nearest and saturated at +-448. No two tokens may have one
    slot. q, k and v may be slices of one projection's output. sections and
    cyclic: positions [axes, n] of several axes, as in `rotary`.
    """
    return _kv().append_tokens(q, k, v, positions, slots, cos, sin, k_pages, v_pages, interleaved, k_scale, v_scale,
                               sections, cyclic)


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               tables: torch.Tensor | None = None) -> None:
    """Copies pages src[i] to dst[i] (int32) of k_pages and v_pages, [n_pages,
    kv_heads, page_size, dim] or with a leading layer dimension, all layers in
    one launch. With `tables` (int32, any shape, contiguous) it moves them:
    entries equal to src[i] become dst[i], and no page may be listed in src
    twice. No page may be a source and a destination, or the destination of
    two. Pairs with an id outside the cache are skipped."""
    _kv().copy_pages(k_pages, v_pages, src, dst, tables)


# ---- attention of one new token ----

def decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                     lens: torch.Tensor, scale: float | None = None, window: int = 0,
                     k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                     max_len: int | None = None, return_lse: bool = False):
    """Attention of one new token per sequence over its cache: q [batch,
    heads, dim], token t of sequence b in row t % page_size of page tables[b,
    t // page_size] (int32), for t < lens[b] (int32), the last `window` of
    them (0: all). heads is a multiple of the cache's; consecutive query heads
    share a key head. scale defaults to dim ** -0.5.

    Returns out [batch, heads, dim] in q's type, and with return_lse the
    logarithm of the sum of exp(scores) in float32 [batch, heads]; a sequence
    without tokens gives 0 and -inf. Whatever the rows past a sequence's end
    hold is not seen, nor are tokens whose table entry is no page. A row of
    v_pages that is read and holds an infinity gives an infinity or NaN.
    max_len: no sequence is longer (default: what tables can hold); the work
    is laid out for it, and tokens past it are not read.
    """
    return _kv().decode_attention(q, k_pages, v_pages, tables, lens, scale, window, k_scale, v_scale, max_len, return_lse)


def retrieved_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                        lens: torch.Tensor, ids: torch.Tensor, first: int = 0, last: int = 0,
                        scale: float | None = None, k_scale: torch.Tensor | None = None,
                        v_scale: torch.Tensor | None = None, return_lse: bool = False):
    """decode_attention over a choice of tokens: the first `first`, the last
    `last`, and between them those in ids [batch, lists, count] (int32), as a
    search of the keys returned them, in any order. lists is the number of
    query heads (each has its own) or of key heads (shared). Ids outside
    [first, len - last), such as a search's -1, are left out: the first and
    last tokens are there already. An id listed twice counts twice."""
    return _kv().retrieved_attention(q, k_pages, v_pages, tables, lens, ids, first, last, scale, k_scale, v_scale,
                                     return_lse)


def shared_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                     lens: torch.Tensor, groups: torch.Tensor, shared: torch.Tensor, scale: float | None = None,
                     k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                     max_len: int | None = None, return_lse: bool = False):
    """decode_attention for a batch whose neighbours share their first tokens,
    which are then read once for all of them. Sequences groups[g] to
    groups[g + 1] - 1 (int32 [n_groups + 1], rising; n_groups at most batch)
    have their first shared[g] tokens (int32 [n_groups]) in common, in the same
    pages or in others with the same rows: they are read where the first of
    them has them. tables and lens are those of whole sequences, as for
    decode_attention, and `shared_prefixes` gives groups and shared for them.
    A sequence that is shorter than its group's prefix reads its own pages, and
    so does one that is in no group. Groups are best as large as they come:
    every group costs as much as a sequence, and 16 query heads of one key head
    fill a matrix instruction. Where decode_attention would read less than 20 to
    60 MB of pages again it is as fast or faster: with 8 key heads of 128 values
    in 16 bits up to about 5,000 tokens in common of two sequences, 2,000 of
    four, 1,000 of 16. Sums, weights and rounding are decode_attention's.
    """
    return _kv().shared_attention(q, k_pages, v_pages, tables, lens, groups, shared, scale, k_scale, v_scale, max_len,
                                  return_lse)


# ---- page tables on the GPU ----

def extend_tables(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, free: torch.Tensor,
                  seqs: torch.Tensor, counts: torch.Tensor, page_size: int, n_tokens: int, width: int | None = None):
    """Room for counts[i] more tokens of sequences seqs[i] (int32 [n]), decided
    on the GPU from its own state: tables [sequences, max_pages] (a sequence's
    pages in order, -1 behind them), lens [sequences], refs [n_pages] (how many
    sequences have a page) and free [ceil(n_pages / 32)] (bit p % 32 of word
    p / 32 where none has page p), all int32 and updated in place; at first -1,
    0, 0 and the bits of all pages. The lowest free pages go to the requests in
    order. One that grows inside a page which other sequences have too gets a
    page for a copy of it first; the last that has it keeps it.

    Returns positions and slots (int64 [n_tokens]; the tokens request after
    request, then position 0 and slot -1), starts (int32 [n + 1], where each
    request's begin), the sequences' tables [n, width] (default: max_pages) and
    lens [n], the pages to copy before tokens are stored, src and dst [n] (-1:
    none; `copy_pages` takes them), and missing [1]: 0, or the number of pages
    that are not there, or -1 where a request cannot be: a sequence listed
    twice, a count below 0, a sequence past width or max_pages, more than
    n_tokens tokens. Nothing has changed then, and the outputs are those of no
    new tokens. Ids outside the tables, such as -1, are left out. At most 65,535
    requests, and 2^18 sequences.
    """
    return _kv().extend_tables(tables, lens, refs, free, seqs, counts, page_size, n_tokens, width)


def truncate_tables(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, free: torch.Tensor,
                    seqs: torch.Tensor, to: torch.Tensor, page_size: int) -> None:
    """Cuts sequences seqs[i] back to to[i] tokens (int32 [n]; 0 gives one up, a
    number below 0 or past its length leaves it), and frees the pages that no
    sequence has any more. State as in `extend_tables`. Of a sequence listed
    twice the first counts; ids outside the tables are left out."""
    _kv().truncate_tables(tables, lens, refs, free, seqs, to, page_size)


def fork_tables(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, free: torch.Tensor, seqs: torch.Tensor,
                into: torch.Tensor, page_size: int) -> None:
    """Gives the sequences into[i], empty until now, the tokens of seqs[i]
    (int32 [n]), on the same pages. State as in `extend_tables`. A sequence may
    be forked several times. Pairs are left out whose ids are outside the
    tables, whose into is not empty, is listed before or stands in seqs too,
    and whose sequence stands in into too (of a pair with both ids inside):
    with seqs 0 1 and into 1 2 neither is made. Forks of forks take a call
    each."""
    _kv().fork_tables(tables, lens, refs, free, seqs, into, page_size)


def shared_prefixes(tables: torch.Tensor, lens: torch.Tensor, page_size: int, least: int = 1):
    """(groups, shared) int32 [batch + 1] and [batch], as shared_attention takes
    them, of a batch's tables [batch, pages] and lens [batch] (int32): a
    sequence is of its predecessor's group where both have at least `least`
    tokens in the same whole pages, and a group shares the whole pages that all
    of it have. Sequences with a prefix in common should be neighbours. Behind
    the last group, groups is batch and shared 0.

    Groups are of one level: where all sequences begin alike and some go on
    alike, one group shares what all have. With `least` past that there are
    smaller groups that share more, and each reads the common part for itself."""
    return _kv().shared_prefixes(tables, lens, page_size, least)


# ---- pages and sequences ----

class PageTable:
    """Which pages the sequences of a cache have: host bookkeeping, with the
    copies and table entries that follow from it for the GPU. Pages are
    counted by their owners; a sequence that is forked shares all of them, and
    has its last one copied when it grows while that page is shared."""

    def __init__(self, n_pages: int, page_size: int, max_sequences: int, max_pages: int):
        if min(n_pages, max_sequences, max_pages) < 1 or page_size < 1:
            raise ValueError("n_pages, page_size, max_sequences and max_pages must be at least 1")
        self.page_size = page_size
        self.pages = np.full((max_sequences, max_pages), -1, dtype=np.int32)
        self.lens = np.full(max_sequences, -1, dtype=np.int64)  # -1: no such sequence
        self.refs = np.zeros(n_pages, dtype=np.int32)
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def n_free(self) -> int:
        return len(self._free)

    def check(self, seqs) -> np.ndarray:
        seqs = np.atleast_1d(np.asarray(seqs, dtype=np.int64))
        if seqs.ndim != 1 or len(np.unique(seqs)) != len(seqs):
            raise ValueError("sequences must be a list without repeats")
        if ((seqs < 0) | (seqs >= len(self.lens))).any() or (self.lens[seqs] < 0).any():
            raise ValueError(f"no such sequence among {seqs.tolist()}")
        return seqs

    def _count(self, seq) -> int:
        return -(-int(self.lens[seq]) // self.page_size)

    def new(self) -> int:
        free = np.flatnonzero(self.lens < 0)
        if not len(free):
            raise RuntimeError(f"all {len(self.lens)} sequences are in use")
        self.lens[free[0]] = 0
        return int(free[0])

    def fork(self, seq: int) -> int:
        seq = int(self.check([seq])[0])
        other, n = self.new(), self._count(seq)
        self.lens[other] = self.lens[seq]
        self.pages[other, :n] = self.pages[seq, :n]
        np.add.at(self.refs, self.pages[seq, :n], 1)
        return other

    def free(self, seqs) -> None:
        for seq in self.check(seqs):
            mine = self.pages[seq, :self._count(seq)]
            self.refs[mine] -= 1
            self._free.extend(sorted((int(p) for p in mine if self.refs[p] == 0), reverse=True))
            self.lens[seq] = -1

    def extend(self, seqs, counts):
        """Room for counts[i] more tokens of seqs[i]. Returns (positions,
        slots) of the new tokens, sequence by sequence, the pages to copy
        first [(src, dst)] and the changed entries [(sequence, index, page)].
        Without enough pages nothing is changed."""
        seqs = self.check(seqs)
        counts = np.broadcast_to(np.asarray(counts, dtype=np.int64), seqs.shape)
        if (counts < 0).any():
            raise ValueError("counts must be at least 0")
        ps, old = self.page_size, self.lens[seqs]
        new = old + counts
        have, need = -(-old // ps), -(-new // ps)
        if len(seqs) and need.max() > self.pages.shape[1]:
            raise ValueError(f"a sequence of {int(new.max())} tokens is too large for a table of {self.pages.shape[1]} pages")
        tail = (counts > 0) & (old % ps != 0)
        last = self.pages[seqs, np.maximum(have - 1, 0)]
        shared, growing = np.unique(last[tail], return_counts=True)
        copies_needed = np.minimum(growing, self.refs[shared] - 1).sum()  # the last owner keeps the page
        if (need - have).sum() + copies_needed > len(self._free):
            raise RuntimeError(f"out of pages: {int((need - have).sum() + copies_needed)} needed, {len(self._free)} free")
        copies, changed = [], []
        for i in np.flatnonzero((need > have) | tail):
            seq = int(seqs[i])
            if tail[i] and self.refs[last[i]] > 1:
                page = self._free.pop()
                self.refs[last[i]] -= 1
                self.refs[page] = 1
                copies.append((int(last[i]), page))
                self.pages[seq, have[i] - 1] = page
                changed.append((seq, int(have[i]) - 1, page))
            for at in range(int(have[i]), int(need[i])):
                page = self._free.pop()
                self.refs[page] = 1
                self.pages[seq, at] = page
                changed.append((seq, at, page))
        self.lens[seqs] = new
        of = np.repeat(np.arange(len(seqs)), counts)
        starts = np.cumsum(counts) - counts
        positions = np.arange(int(counts.sum())) - np.repeat(starts - old, counts)
        slots = self.pages[seqs[of], positions // ps].astype(np.int64) * ps + positions % ps
        return positions, slots, copies, changed

    def compact(self):
        """(src, dst): the moves after which the pages in use come first."""
        used = np.flatnonzero(self.refs > 0)
        n = len(used)
        src = used[used >= n].astype(np.int32)
        dst = np.flatnonzero(self.refs[:n] == 0).astype(np.int32)
        to = np.arange(len(self.refs), dtype=np.int32)
        to[src] = dst
        self.pages = np.where(self.pages >= 0, to[self.pages], -1).astype(np.int32)
        self.refs[dst] = self.refs[src]
        self.refs[src] = 0
        self._free = list(range(len(self.refs) - 1, n - 1, -1))
        return src, dst


class Step:
    """The new tokens of some sequences (PagedCache.extend): where they go,
    and the sequences' tables and lengths with them. All layers use one."""

    def __init__(self, seqs, positions, slots, tables, lens, max_len, starts=None, missing=None):
        self.seqs, self.positions, self.slots = seqs, positions, slots
        self.tables, self.lens, self.max_len = tables, lens, max_len
        self.starts, self.missing = starts, missing  # GpuPagedCache's


class PagedCache:
    """The keys and values of all layers of a model in pages, for sequences
    that grow, are forked and freed.

    k_pages, v_pages [n_layers, n_pages, kv_heads, page_size, dim] and tables
    [max_sequences, max_pages] (int32) are device tensors that the functions
    above take layer by layer; who owns which page is kept on the host
    (PageTable), so that an exhausted cache raises where it is asked for more,
    before anything is changed. dtype float8_e4m3fn takes k_scale, v_scale
    [n_layers, kv_heads] (float32; None: 1).

        step = cache.extend(seqs, 1)
        for layer in range(n_layers):
            q = cache.append(layer, step, q, k, v, cos, sin)
            out = cache.decode(layer, step, q)
    """

    def __init__(self, n_pages: int, n_layers: int, kv_heads: int, dim: int, page_size: int = 16,
                 dtype: torch.dtype = torch.float16, max_sequences: int = 64, max_pages: int | None = None,
                 device: str = "cuda", k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        if dtype not in _TYPES:
            raise ValueError(f"dtype must be float16, bfloat16 or float8_e4m3fn, got {dtype}")
        if page_size < 8 or page_size > 256 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 8 to 256")
        if n_layers < 1 or kv_heads < 1 or dim < 1 or dim > 256 or dim % (16 if dtype == _F8 else 8):
            raise ValueError("n_layers and kv_heads must be at least 1, dim up to 256 and a multiple of 16 bytes")
        max_pages = n_pages if max_pages is None else max_pages
        self.table = PageTable(n_pages, page_size, max_sequences, max_pages)
        shape = (n_layers, n_pages, kv_heads, page_size, dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=device)
        self.v_pages = torch.empty(shape, dtype=dtype, device=device)
        self.tables = torch.full((max_sequences, max_pages), -1, dtype=torch.int32, device=device)
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t is not None and (dtype != _F8 or t.shape != (n_layers, kv_heads)):
                raise ValueError(f"{name} must be [{n_layers}, {kv_heads}] with float8_e4m3fn pages")
        place = self.k_pages.device
        self.k_scale, self.v_scale = (None if t is None else t.to(place, torch.float32).contiguous()
                                      for t in (k_scale, v_scale))

    def new(self) -> int:
        """An empty sequence."""
        return self.table.new()

    def length(self, seq: int) -> int:
        return int(self.table.lens[self.table.check([seq])[0]])

    @property
    def n_free(self) -> int:
        """Pages that no sequence has."""
        return self.table.n_free

    def free(self, seqs) -> None:
        """Gives back the sequences and the pages that only they have."""
        self.table.free(seqs)

    def fork(self, seq: int) -> int:
        """A sequence with the tokens of `seq`, sharing its pages."""
        other = self.table.fork(seq)
        self.tables[other].copy_(self.tables[int(seq)])
        return other

    def _upload(self, *arrays):
        """Host arrays as int64 device tensors, through pinned memory in one copy that is not waited for."""
        flat = [np.asarray(a, dtype=np.int64).reshape(-1) for a in arrays]
        host = torch.empty(sum(len(a) for a in flat), dtype=torch.int64, pin_memory=True)
        np.concatenate(flat, out=host.numpy())
        return host.to(self.k_pages.device, non_blocking=True).split([len(a) for a in flat])

    def _copy(self, src, dst, tables=None):
        copy_pages(self.k_pages, self.v_pages, src.int(), dst.int(), tables=tables)

    def extend(self, seqs, counts=1) -> Step:
        """Room for `counts` (one number, or one per sequence) new tokens of
        each of the sequences; pages that other sequences share are copied
        first. Raises RuntimeError, with nothing changed, when pages run out."""
        positions, slots, copies, changed = self.table.extend(seqs, counts)
        seqs = self.table.check(seqs)
        lens = self.table.lens[seqs]
        copies, changed = np.reshape(copies, (-1, 2)), np.reshape(changed, (-1, 3))
        parts = self._upload(seqs, lens, positions, slots, copies[:, 0], copies[:, 1], *changed.T)
        at, lens_gpu, positions, slots, src, dst, rows, cols, pages = parts
        if len(copies):
            self._copy(src, dst)
        if len(changed):
            self.tables[rows, cols] = pages.int()
        longest = int(lens.max()) if len(lens) else 0
        width = max(1, -(-longest // self.table.page_size))
        return Step(seqs, positions, slots, self.tables[:, :width].index_select(0, at), lens_gpu.int(), longest)

    def compact(self) -> int:
        """Moves the pages in use to the front, in all layers, and returns how
        many moved. Steps taken before are void."""
        src, dst = self.table.compact()
        if len(src):
            self._copy(*self._upload(src, dst), tables=self.tables)
        return len(src)

    def _layer(self, layer):
        scales = {"k_scale": None if self.k_scale is None else self.k_scale[layer],
                  "v_scale": None if self.v_scale is None else self.v_scale[layer]}
        return self.k_pages[layer], self.v_pages[layer], scales

    def append(self, layer: int, step: Step, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
               cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, interleaved: bool = False,
               positions: torch.Tensor | None = None, sections: Sequence[int] | None = None, cyclic: bool = False):
        """append_tokens for the step's tokens. positions: other ones than their places in the sequences, as with
        several axes."""
        k_pages, v_pages, scales = self._layer(layer)
        return append_tokens(q, k, v, step.positions if positions is None else positions, step.slots, cos, sin, k_pages,
                             v_pages, interleaved=interleaved, sections=sections, cyclic=cyclic, **scales)

    def decode(self, layer: int, step: Step, q: torch.Tensor, **options):
        """decode_attention for the step's sequences, q [sequences, heads, dim]."""
        k_pages, v_pages, scales = self._layer(layer)
        return decode_attention(q, k_pages, v_pages, step.tables, step.lens, max_len=step.max_len, **scales, **options)

    def retrieved(self, layer: int, step: Step, q: torch.Tensor, ids: torch.Tensor, first: int = 0, last: int = 0,
                  **options):
        """retrieved_attention for the step's sequences."""
        k_pages, v_pages, scales = self._layer(layer)
        return retrieved_attention(q, k_pages, v_pages, step.tables, step.lens, ids, first=first, last=last, **scales,
                                   **options)

    def prefixes(self, step: Step, least: int = 1):
        """shared_prefixes of the step's sequences, for `shared` in all layers. Forks should be neighbours in it."""
        return shared_prefixes(step.tables, step.lens, self.k_pages.size(3), least)

    def shared(self, layer: int, step: Step, q: torch.Tensor, prefixes, **options):
        """shared_attention for the step's sequences: decode, with what `prefixes` found in common read once."""
        k_pages, v_pages, scales = self._layer(layer)
        return shared_attention(q, k_pages, v_pages, step.tables, step.lens, *prefixes, max_len=step.max_len, **scales,
                                **options)

    def _own(self, seq: int):
        """A sequence's length and its pages."""
        n = self.length(seq)
        own, = self._upload(self.table.pages[seq, :-(-n // self.table.page_size)])
        return n, own

    def keys(self, layer: int, seq: int) -> torch.Tensor:
        """The keys of a sequence, [kv_heads, length, dim], contiguous float16 rows for an index (`Graph`,
        `bruteforce_knn`), whatever the pages' type: what they hold (times k_scale), rounded once; finite values past
        float16's range are its ends, +-65504."""
        n, own = self._own(seq)
        store = self.k_pages[layer]
        rows = store.view(torch.uint8)[own].view(store.dtype) if store.dtype == _F8 else store[own]
        heads, dim = store.size(1), store.size(3)
        rows = rows.transpose(0, 1).reshape(heads, -1, dim)[:, :n]
        if store.dtype != torch.float16:
            rows = rows.float()
            if self.k_scale is not None:
                rows = rows * self.k_scale[layer][:, None, None]
            most = torch.finfo(torch.float16).max
            rows = torch.where(rows.isfinite(), rows.clamp(-most, most), rows).to(torch.float16)
        return rows.contiguous()


class GpuPagedCache(PagedCache):
    """A PagedCache whose bookkeeping is on the GPU as well, so that a step --
    sequences that grow, are cut back, forked and given up, their tokens
    appended and attended to -- synchronizes nothing and can be captured in a
    graph and replayed.

    Sequences are rows 0 to max_sequences - 1 of the tables, all empty at
    first; which of them a program uses is its own affair. Where pages run out
    nothing is stored, and step.missing says so (extend_tables), to be read
    when it suits.

    max_pages (default: all n_pages), or max_len in `extend`, is the width of
    the tables that every step writes, and the lengths that `decode` and
    `shared` lay their workspaces out for and refuse when they are too large:
    give the longest that a sequence may become.

        step = cache.extend(seqs, counts, n_tokens)       # int32 tensors
        prefixes = cache.prefixes(step)
        for layer in range(n_layers):
            q = cache.append(layer, step, q, k, v, cos, sin)
            out = cache.shared(layer, step, q, prefixes)
        cache.truncate(seqs, accepted)
    """

    def __init__(self, n_pages: int, n_layers: int, kv_heads: int, dim: int, page_size: int = 16,
                 dtype: torch.dtype = torch.float16, max_sequences: int = 64, max_pages: int | None = None,
                 device: str = "cuda", k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        super().__init__(n_pages, n_layers, kv_heads, dim, page_size, dtype, max_sequences, max_pages, device, k_scale,
                         v_scale)
        del self.table  # nothing is kept on the host
        self.page_size, place = page_size, self.k_pages.device
        self.lens = torch.zeros(max_sequences, dtype=torch.int32, device=place)
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device=place)
        bits = np.packbits(np.arange(-(-n_pages // 32) * 32) < n_pages, bitorder="little").view(np.int32)
        self.free_bits = torch.from_numpy(bits).to(place)

    def _state(self):
        return self.tables, self.lens, self.refs, self.free_bits

    def new(self):
        raise NotImplementedError("sequences of a GpuPagedCache are the rows of its tables, empty until they are extended")

    def compact(self):
        raise NotImplementedError("a GpuPagedCache takes the lowest free pages and is not compacted")

    def length(self, seq: int) -> int:
        """Waits for the GPU."""
        if not 0 <= seq < self.lens.size(0):
            raise ValueError(f"no such sequence: {seq}")
        return int(self.lens[seq])

    @property
    def n_free(self) -> int:
        """Pages that no sequence has. Waits for the GPU."""
        return int((self.refs == 0).sum())

    def extend(self, seqs: torch.Tensor, counts: torch.Tensor, n_tokens: int, max_len: int | None = None) -> Step:
        """extend_tables, and the copies of pages that are shared no longer, in all layers. n_tokens: the counts' sum,
        or more (the rest are tokens without a slot). max_len: no sequence is longer than that now, in whole pages;
        where one would be, nothing is stored (missing -1)."""
        width = self.tables.size(1)
        longest = width * self.page_size
        if max_len is not None:
            if max_len < 0:
                raise ValueError("max_len must be at least 0")
            width = min(width, -(-max_len // self.page_size))
            longest = width * self.page_size  # what extend_tables lets a sequence have is attended to
        positions, slots, starts, tables, lens, src, dst, missing = extend_tables(
            *self._state(), seqs, counts, self.page_size, n_tokens, width)
        copy_pages(self.k_pages, self.v_pages, src, dst)
        return Step(seqs, positions, slots, tables, lens, longest, starts, missing)

    def truncate(self, seqs: torch.Tensor, to: torch.Tensor) -> None:
        """truncate_tables."""
        truncate_tables(*self._state(), seqs, to, self.page_size)

    def free(self, seqs: torch.Tensor) -> None:
        """Gives up the sequences, and the pages that only they have."""
        self.truncate(seqs, torch.zeros_like(seqs))

    def fork(self, seqs: torch.Tensor, into: torch.Tensor) -> None:
        """fork_tables."""
        fork_tables(*self._state(), seqs, into, self.page_size)

    def _own(self, seq: int):
        n = self.length(seq)
        return n, self.tables[seq, :-(-n // self.page_size)].long()
