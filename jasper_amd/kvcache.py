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
  PagedCache              pages, sequences, forks and compaction put together

Pages are [n_pages, kv_heads, page_size, dim] (with a leading layer dimension
where said) in float16, bfloat16 or float8_e4m3fn, any strides that keep a
row's dim values together and rows on 16 bytes. Calls run on the current
stream of the tensors' device, synchronize nothing and may be captured in a
graph (PagedCache's bookkeeping is on the host and is not captured).
"""

from __future__ import annotations

import ctypes
import functools
import math

import numpy as np
import torch

_TYPES = {torch.float16: 0, torch.bfloat16: 1}
_PAGE_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float8_e4m3fn: 2}

_i32, _i64, _ptr, _f64 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_double


class _Pages(ctypes.Structure):
    _fields_ = [("k", _ptr), ("v", _ptr), ("k_scale", _ptr), ("v_scale", _ptr),
                ("layer_stride", _i64), ("page_stride", _i64), ("head_stride", _i64), ("row_stride", _i64),
                ("layers", _i32), ("pages", _i32), ("heads", _i32), ("page_size", _i32), ("dim", _i32), ("type", _i32)]


class _Rows(ctypes.Structure):
    _fields_ = [("data", _ptr), ("stride", _i64), ("head_stride", _i64), ("heads", _i64)]


_SIGNATURES = {
    "jasperx_rotary": [_ptr, _ptr, _i32, _i64, _i64, _ptr, _i32, _ptr, _ptr, _i64, _i64, ctypes.c_uint32, _ptr, _ptr,
                       _ptr],
    "jasperx_append_tokens": [_ptr, _ptr, _ptr, _i32, _i64, _ptr, _ptr, _i32, _ptr, _ptr, _i64, _i64,
                              ctypes.c_uint32, _ptr, _ptr, _ptr],
    "jasperx_copy_pages": [_ptr, _ptr, _ptr, _i64, _ptr, _i64, _ptr],
    "jasperx_decode_attention": [_ptr, _i32, _i64, _ptr, _ptr, _i64, _i64, _ptr, _i64, _f64, _i64, _ptr, _ptr, _ptr,
                                 _i64, _ptr],
    "jasperx_retrieved_attention": [_ptr, _i32, _i64, _ptr, _ptr, _i64, _i64, _ptr, _ptr, _i64, _i64, _i64, _i64,
                                    _f64, _ptr, _ptr, _ptr, _i64, _ptr],
    "jasperx_attention_workspace": [_i64, _i64, _ptr, _i64, _i64],
}


@functools.lru_cache(maxsize=None)
def _fn(name):
    from . import _bind
    return _bind(name, _SIGNATURES[name])


def _call(name, device, *args):
    """The C call `name` on the device's current stream (its last argument)."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _fn(name)(*args, torch.cuda.current_stream(device).cuda_stream)
    return _fn(name)(*args, torch.cuda.current_stream(device).cuda_stream)


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _on_gpu(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}")


def _index(name, t, device):
    """An int32 or int64 tensor as a contiguous one."""
    if t.dtype != torch.int64 and t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _int32(name, t, ndim, device):
    if t.dtype != torch.int32 or t.ndim != ndim:
        raise ValueError(f"{name} must be a {ndim}D int32 tensor, got {t.ndim}D {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t


def _scales(name, t, heads, pages):
    if t is None:
        return None
    _need(pages.dtype == torch.float8_e4m3fn, f"{name} needs float8_e4m3fn pages")
    _need(t.dtype == torch.float32 and t.shape == (heads,) and t.is_contiguous() and t.device == pages.device,
          f"{name} must be a contiguous float32 [{heads}] tensor on the pages' device")
    return t.data_ptr()


def _pages(k_pages, v_pages, k_scale=None, v_scale=None, layers=False):
    """The C description of a pair of page tensors, checked."""
    if k_pages.dtype not in _PAGE_TYPES:
        raise ValueError(f"pages must be float16, bfloat16 or float8_e4m3fn, got {k_pages.dtype}")
    if (v_pages.dtype != k_pages.dtype or v_pages.shape != k_pages.shape or v_pages.device != k_pages.device
            or v_pages.stride() != k_pages.stride()):
        raise ValueError("k_pages and v_pages must have the same type, shape, strides and device")
    if not k_pages.is_cuda:
        raise ValueError("k_pages must be a CUDA tensor")
    shape, stride = k_pages.shape, k_pages.stride()
    if layers and len(shape) == 4:
        shape, stride = (1, *shape), (0, *stride)
    if len(shape) != (5 if layers else 4):
        raise ValueError(f"pages must be [{'layers, ' if layers else ''}n_pages, kv_heads, page_size, dim], got {k_pages.ndim}D")
    if not layers:
        shape, stride = (1, *shape), (0, *stride)
    if stride[4] != 1:
        raise ValueError("the last dimension of the pages must be contiguous")
    return _Pages(k_pages.data_ptr(), v_pages.data_ptr(), _scales("k_scale", k_scale, shape[2], k_pages),
                  _scales("v_scale", v_scale, shape[2], k_pages), stride[0], stride[1], stride[2], stride[3],
                  shape[0], shape[1], shape[2], shape[3], shape[4], _PAGE_TYPES[k_pages.dtype])


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
    _need(n_positions >= 0, "n_positions must be at least 0")
    _need(rot_dim > 0 and rot_dim % 2 == 0, "rot_dim must be even and positive")
    _need(scaling in (None, "linear", "ntk", "yarn"), f"Unknown scaling: {scaling!r}")
    _need(scaling is None or factor >= 1.0, "factor must be at least 1")
    pair = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    size = 1.0
    if scaling == "ntk" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = base ** (-pair / rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        _need(original is not None and original > 0, "yarn scaling needs the original context length")

        def at(turns):  # the pair that turns so many times within the original context
            return rot_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))

        low = max(0, math.floor(at(beta_fast)))
        high = min(rot_dim // 2 - 1, math.ceil(at(beta_slow)))
        ramp = ((pair / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        size = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return (angle.cos() * size).float(), (angle.sin() * size).float()


def _table(cos, sin, device):
    if cos is None and sin is None:
        return None, None, 0, 0
    _need(cos is not None and sin is not None, "cos and sin come together")
    if (cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.ndim != 2 or cos.shape != sin.shape
            or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous float32 [n_positions, rot_dim / 2] tensors")
    _on_gpu(device, cos=cos, sin=sin)
    return cos.data_ptr(), sin.data_ptr(), cos.size(0), 2 * cos.size(1)


def _heads(name, t, like):
    """[..., heads, dim] as rows [n, heads, dim] whose values are contiguous."""
    if t.ndim < 2:
        raise ValueError(f"{name} must be [..., heads, dim]")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[:-2] != like.shape[:-2]
                             or t.size(-1) != like.size(-1)):
        raise ValueError(f"{name} must match the other rows in type, device, leading sizes and dim")
    if t.ndim != 3:
        t = t.flatten(0, -3) if t.ndim > 3 else t[None]
    return t if t.stride(2) == 1 else t.contiguous()


def _rows(t):
    return _Rows(t.data_ptr(), t.stride(0), t.stride(1), t.size(1))


def _rotate(q, k, positions, cos, sin, interleaved, back):
    first = q if q is not None else k
    device = first.device
    n = math.prod(first.shape[:-2])
    dim = first.size(-1)
    c, s, table_rows, rot = _table(cos, sin, device)
    outs, rows = [], []
    for name, t in (("q", q), ("k", k)):
        if t is None:
            outs.append(None)
            rows.append(None)
            continue
        flat = _heads(name, t, first)
        rows.append((flat, _rows(flat)))
        outs.append(torch.empty(t.shape, dtype=t.dtype, device=device))
    if n:
        _call("jasperx_rotary", device, *(None if r is None else ctypes.byref(r[1]) for r in rows),
              _TYPES[first.dtype], n, dim, positions.data_ptr(), positions.element_size(), c, s, table_rows, rot,
              (1 if interleaved else 0) | (2 if back else 0), *(None if o is None else o.data_ptr() for o in outs))
    return outs


class _Rotary(torch.autograd.Function):
    """Linear in q and k: the gradient is the rotation by the opposite
    angles, which is differentiated the same way."""

    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, interleaved, back):
        ctx.save_for_backward(positions, cos, sin)
        ctx.flags = interleaved, back
        ctx.set_materialize_grads(False)
        return tuple(_rotate(q, k, positions, cos, sin, interleaved, back))

    @staticmethod
    def backward(ctx, gq, gk):
        gq = gq if ctx.needs_input_grad[0] else None
        gk = gk if ctx.needs_input_grad[1] else None
        if gq is None and gk is None:
            return (None,) * 7
        interleaved, back = ctx.flags
        out = _Rotary.apply(gq, gk, *ctx.saved_tensors, interleaved, not back)
        return (*out, None, None, None, None, None)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           interleaved: bool = False):
    """(q, k) [..., heads, dim] (fp16 or bf16) with rotary positions: the
    first 2 * cos.size(1) values of every head are turned in pairs by the
    angles in row positions[...] of the tables (`rotary_table`), the rest is
    as it was. Pairs are (i, i + rot_dim / 2), or neighbours when interleaved.
    Differentiable in q and k. k may be None. A position outside the tables
    gives NaN. Sums are in 32 bits, rounded once.
    """
    if q.dtype not in _TYPES:
        raise ValueError(f"q must be float16 or bfloat16, got {q.dtype}")
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor")
    if q.ndim < 2 or q.size(-1) % 2:
        raise ValueError("q must be [..., heads, dim] with an even dim")
    if k is not None:
        _heads("k", k, q)
    positions = _index("positions", positions, q.device)
    _need(positions.shape == q.shape[:-2], f"positions must be {list(q.shape[:-2])}, got {list(positions.shape)}")
    _need(cos is not None and sin is not None, "cos and sin are needed")
    _table(cos, sin, q.device)
    _need(2 * cos.size(1) <= q.size(-1), "the tables rotate more values than a head has")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, positions, cos, sin, bool(interleaved), False)
    return tuple(_rotate(q, k, positions, cos, sin, bool(interleaved), False))


# ---- the cache ----

def append_tokens(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor | None,
                  slots: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None, k_pages: torch.Tensor,
                  v_pages: torch.Tensor, interleaved: bool = False, k_scale: torch.Tensor | None = None,
                  v_scale: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores k (rotated as `rotary` does) and v [n, kv_heads, dim] to rows
    slots [n] of the pages (page * page_size + row; a slot outside the cache,
    such as -1, stores nothing) and returns q [n, heads, dim] rotated. q may
    be None; cos and sin None: nothing is rotated. float8_e4m3fn pages hold
    values divided by k_scale, v_scale [kv_heads] (float32, or None),
    rounded to nearest and saturated at +-448. No two tokens may have one
    slot. q, k and v may be slices of one projection's output.
    """
    p = _pages(k_pages, v_pages, k_scale, v_scale)
    device = k_pages.device
    if k.dtype not in _TYPES:
        raise ValueError(f"k must be float16 or bfloat16, got {k.dtype}")
    if k_pages.dtype != torch.float8_e4m3fn and k_pages.dtype != k.dtype:
        raise ValueError(f"pages must be {k.dtype} or float8_e4m3fn, got {k_pages.dtype}")
    _need(k.ndim == 3 and k.size(1) == p.heads and k.size(2) == p.dim, f"k must be [n, {p.heads}, {p.dim}]")
    _need(v.shape == k.shape, "v must have k's shape")
    _on_gpu(device, k=k)
    k, v = _heads("k", k, None), _heads("v", v, k)
    n = k.size(0)
    out = None
    if q is not None:
        _need(q.ndim == 3, "q must be [n, heads, dim]")
        q = _heads("q", q, k)
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad)):
        raise ValueError("append_tokens has no gradient: use rotary, or torch.no_grad()")
    slots = _index("slots", slots, device)
    _need(slots.shape == (n,), f"slots must be [{n}]")
    c, s, table_rows, rot = _table(cos, sin, device)
    _need(rot <= p.dim, "the tables rotate more values than a head has")
    at = None
    if rot:
        _need(positions is not None, "positions are needed with cos and sin")
        positions = _index("positions", positions, device)
        _need(positions.shape == (n,), f"positions must be [{n}]")
        if positions.dtype != slots.dtype:
            positions, slots = positions.long(), slots.long()
        at = positions.data_ptr()
    if n:
        _call("jasperx_append_tokens", device, None if q is None else ctypes.byref(_rows(q)), ctypes.byref(_rows(k)),
              ctypes.byref(_rows(v)), _TYPES[k.dtype], n, at, slots.data_ptr(), slots.element_size(), c, s,
              table_rows, rot, 1 if interleaved else 0, ctypes.byref(p), None if out is None else out.data_ptr())
    return out


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               tables: torch.Tensor | None = None) -> None:
    """Copies pages src[i] to dst[i] (int32) of k_pages and v_pages, [n_pages,
    kv_heads, page_size, dim] or with a leading layer dimension, all layers in
    one launch. With `tables` (int32, any shape, contiguous) it moves them:
    entries equal to src[i] become dst[i]. No page may be a source and a
    destination, or the destination of two. Pairs with an id outside the
    cache are skipped."""
    p = _pages(k_pages, v_pages, layers=True)
    device = k_pages.device
    src, dst = _int32("src", src, 1, device), _int32("dst", dst, 1, device)
    _need(src.shape == dst.shape, "src and dst must have the same length")
    entries = 0
    if tables is not None:
        _need(tables.dtype == torch.int32 and tables.is_contiguous() and tables.device == device,
              "tables must be a contiguous int32 tensor on the pages' device")
        entries = tables.numel()
    src, dst = src.contiguous(), dst.contiguous()
    if src.numel():
        _call("jasperx_copy_pages", device, ctypes.byref(p), src.data_ptr(), dst.data_ptr(), src.numel(),
              tables.data_ptr() if entries else None, entries)


# ---- attention of one new token ----

@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device, batch, q_heads, heads, page_size, dim, type_, max_tokens, lists):
    p = _Pages(None, None, None, None, 0, 0, 0, dim, 1, 0, heads, page_size, dim, type_)
    with torch.cuda.device(device):
        return _fn("jasperx_attention_workspace")(batch, q_heads, ctypes.byref(p), max_tokens, lists)


def _attention_args(q, p, k_pages, tables, lens):
    device = k_pages.device
    if q.dtype not in _TYPES or (k_pages.dtype != torch.float8_e4m3fn and k_pages.dtype != q.dtype):
        raise ValueError(f"q must be float16 or bfloat16 and the pages of its type or float8_e4m3fn, got {q.dtype} "
                         f"and {k_pages.dtype}")
    _need(q.ndim == 3 and q.size(2) == p.dim, f"q must be [batch, heads, {p.dim}]")
    if q.device != device:
        raise ValueError(f"q must be on {device}, got {q.device}")
    _need(q.size(1) > 0 and q.size(1) % p.heads == 0, f"q's heads must be a multiple of the cache's {p.heads}")
    if torch.is_grad_enabled() and q.requires_grad:
        raise ValueError("attention over the cache has no gradient: use torch.no_grad()")
    b = q.size(0)
    _int32("tables", tables, 2, device)
    _need(tables.size(0) == b and (tables.size(1) <= 1 or tables.stride(1) == 1),
          f"tables must be [{b}, pages] with contiguous rows")
    _int32("lens", lens, 1, device)
    _need(lens.size(0) == b, f"lens must be [{b}]")
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    return q, tables, lens if lens.is_contiguous() else lens.contiguous(), device


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
    hold is not seen. max_len: no sequence is longer (default: what tables can
    hold); the work is laid out for it, and tokens past it are not read.
    """
    p = _pages(k_pages, v_pages, k_scale, v_scale)
    q, tables, lens, device = _attention_args(q, p, k_pages, tables, lens)
    _need(window >= 0, "window must be at least 0")
    b, heads, dim = q.shape
    capacity = tables.size(1) * p.page_size
    max_len = capacity if max_len is None else min(int(max_len), capacity)
    _need(max_len >= 0, "max_len must be at least 0")
    out = torch.empty((b, heads, dim), dtype=q.dtype, device=device)
    lse = torch.empty((b, heads), dtype=torch.float32, device=device) if return_lse else None
    if b:
        size = _workspace_bytes(device, b, heads, p.heads, p.page_size, dim, p.type,
                                min(max_len, window) if window else max_len, 0)
        scratch = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _call("jasperx_decode_attention", device, ctypes.byref(_rows(q)), _TYPES[q.dtype], b, ctypes.byref(p),
              tables.data_ptr(), tables.stride(0), tables.size(1), lens.data_ptr(), max_len,
              dim ** -0.5 if scale is None else scale, window, out.data_ptr(),
              lse.data_ptr() if return_lse else None, scratch.data_ptr() if size else None, size)
    return (out, lse) if return_lse else out


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
    p = _pages(k_pages, v_pages, k_scale, v_scale)
    q, tables, lens, device = _attention_args(q, p, k_pages, tables, lens)
    b, heads, dim = q.shape
    _int32("ids", ids, 3, device)
    lists, count = ids.size(1), ids.size(2)
    _need(ids.size(0) == b and lists in (heads, p.heads), f"ids must be [{b}, {heads} or {p.heads}, count]")
    _need(first >= 0 and last >= 0, "first and last must be at least 0")
    if not ids.is_contiguous():
        ids = ids.contiguous()
    out = torch.empty((b, heads, dim), dtype=q.dtype, device=device)
    lse = torch.empty((b, heads), dtype=torch.float32, device=device) if return_lse else None
    if b:
        size = _workspace_bytes(device, b, heads, p.heads, p.page_size, dim, p.type, first + last + count, lists)
        scratch = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _call("jasperx_retrieved_attention", device, ctypes.byref(_rows(q)), _TYPES[q.dtype], b, ctypes.byref(p),
              tables.data_ptr(), tables.stride(0), tables.size(1), lens.data_ptr(), ids.data_ptr(), lists, count,
              first, last, dim ** -0.5 if scale is None else scale, out.data_ptr(),
              lse.data_ptr() if return_lse else None, scratch.data_ptr() if size else None, size)
    return (out, lse) if return_lse else out
