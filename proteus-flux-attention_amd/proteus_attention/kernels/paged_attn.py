"""Paged key-value cache and the attention of one new token over it.

:func:`aspa_sparse_attention` and the layer take whole sequences.  A program
that generates holds the keys and values of what it has read and written, and
asks for one token's attention at a time:

* :func:`new_kv_pages` -- a pool of pages, in the values' type or in 8 bits;
* :func:`write_kv_pages` -- new tokens into their sequences' pages, quantised as
  they are written;
* :func:`read_kv_pages` -- a range of every sequence back out of its pages;
* :func:`paged_attention` -- one new token a sequence over its cache, over a
  window of it, or over listed pages of it;
* :func:`select_kv_pages` -- the pages whose keys promise the largest scores;
* :func:`paged_sparse_attention` -- attention over those.

A block table ``(B, P)`` int32 names each sequence's pages in the order of its
positions; entries that name no page (-1) hold no keys.  ``lengths``,
``starts`` and ``counts`` are ``(B,)`` int32 on the device and are never copied
to the host, so every call can be captured in a HIP graph.  Like the rest of
the package this is the inference path: tensors that require a gradient raise
``NotImplementedError``.  The reference has no counterpart.
"""
from __future__ import annotations

import functools
import math
import struct
from typing import NamedTuple, Optional, Tuple

import torch

from .. import _hip
from .sparse_attn import _size_out

HEAD_DIMS = (16, 32, 64, 128)
PAGE_SIZES = (16, 32, 64, 128, 256)

_VALUE_TAG = {torch.float32: _hip.PFA_F32, torch.bfloat16: _hip.PFA_BF16, torch.float16: _hip.PFA_F16}
_CELL_TAG = {**_VALUE_TAG, torch.int8: _hip.PFA_I8, torch.float8_e4m3fn: _hip.PFA_E4M3}
_EIGHT_BITS = (torch.int8, torch.float8_e4m3fn)
# Pages of a table or list, sequences: the library takes them in 32 bits and has limits
# of its own below these, by the page size and the rows.
_MOST = 1 << 30


class KVPages(NamedTuple):
    """A pool of pages.  ``k``, ``v``: ``(pages, kv_heads, page_size,
    head_dim)`` cells, f32, bf16, f16, int8 or float8_e4m3fn (a stride between
    pages is fine, the inner dimensions are dense).  ``k_scale``, ``v_scale``:
    ``(pages, kv_heads, page_size)`` f32 for 8-bit cells.  ``k_bounds``: the
    least and the largest stored key of every channel, ``(pages, kv_heads, 2,
    head_dim)`` in the cells' type, f32 for 8-bit cells; needed for selection
    alone."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None
    k_bounds: Optional[torch.Tensor] = None


def new_kv_pages(num_pages: int, kv_heads: int, page_size: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, bounds: bool = False, device="cuda") -> KVPages:
    """A pool of zeros; ``bounds`` adds the key bounds that selection reads."""

    if dtype not in _CELL_TAG:
        raise ValueError(f"unsupported cell dtype {dtype}")
    if head_dim not in HEAD_DIMS or page_size not in PAGE_SIZES:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} and page_size one of {PAGE_SIZES}")
    if num_pages < 1 or kv_heads < 1:
        raise ValueError("a pool needs pages and heads")
    shape = (num_pages, kv_heads, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    scales = (None, None)
    if dtype in _EIGHT_BITS:
        scales = tuple(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
    kb = None
    if bounds:
        kb = torch.zeros(num_pages, kv_heads, 2, head_dim, device=device,
                         dtype=torch.float32 if dtype in _EIGHT_BITS else dtype)
    return KVPages(k, v, *scales, kb)


# pfa_kv_pages, pfa_tensor4 and pfa_paged_query of include/pfa_hip.h
_POOL = struct.Struct("PPPPPqqiiiii4x")
_TENSOR4 = struct.Struct("Pqqq")
_QUERY = struct.Struct(_POOL.format + _TENSOR4.format + "PqPPiiii")


def _dense(t: torch.Tensor, shape: Tuple[int, ...], dtype: torch.dtype, name: str) -> int:
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    return t.data_ptr()


def _pool(pages: KVPages) -> tuple:
    """The fields of pfa_kv_pages; the last five are pages, heads, page size, head
    dim and the cells' tag."""

    k, v, k_scale, v_scale, bounds = pages
    dtype, shape = k.dtype, k.shape
    tag = _CELL_TAG.get(dtype)
    if tag is None or v.dtype != dtype:
        raise ValueError(f"k and v pages must share one of {tuple(_CELL_TAG)} (got {dtype}, {v.dtype})")
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("k and v pages must be (pages, kv_heads, page_size, head_dim) tensors of one shape")
    N, H, ps, D = shape
    if D not in HEAD_DIMS or ps not in PAGE_SIZES:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} and page_size one of {PAGE_SIZES} (got {D}, {ps})")
    if N == 0 or H == 0:
        raise ValueError("an empty pool")
    ks, vs = k.stride(), v.stride()
    dense = (ps * D, D, 1)
    if ks[1:] != dense or vs[1:] != dense:
        for s in (ks, vs):
            if s[2:] != dense[1:] or (H > 1 and s[1] != dense[0]):
                raise ValueError("a page's heads, slots and channels must be dense")
    a = c = b = 0
    bound_dtype = dtype
    if dtype in _EIGHT_BITS:
        if k_scale is None or v_scale is None:
            raise ValueError("8-bit pages need k_scale and v_scale")
        rows = shape[:3]
        a = _dense(k_scale, rows, torch.float32, "k_scale")
        c = _dense(v_scale, rows, torch.float32, "v_scale")
        bound_dtype = torch.float32
    if bounds is not None:
        b = _dense(bounds, (N, H, 2, D), bound_dtype, "k_bounds")
    if (k.requires_grad or v.requires_grad or (b and bounds.requires_grad)
            or (a and (k_scale.requires_grad or v_scale.requires_grad))) and torch.is_grad_enabled():
        raise NotImplementedError("pages have no backward pass: call it under torch.no_grad()")
    return k.data_ptr(), v.data_ptr(), a, c, b, ks[0], vs[0], N, H, ps, D, tag


def _table(block_table: torch.Tensor, B: int) -> torch.Tensor:
    shape = block_table.shape
    if len(shape) != 2 or shape[0] != B or block_table.dtype != torch.int32:
        raise ValueError(f"block_table must be a ({B}, P) int32 tensor")
    if B > _MOST or shape[1] > _MOST:
        raise ValueError(f"a block table of up to {_MOST} sequences and pages (got {tuple(shape)})")
    return block_table if block_table.stride(1) == 1 or shape[1] <= 1 else block_table.contiguous()


def _per_sequence(t: torch.Tensor, B: int, name: str) -> torch.Tensor:
    if t.shape != (B,) or t.dtype != torch.int32:
        raise ValueError(f"{name} must be a ({B},) int32 tensor")
    return t if t.is_contiguous() else t.contiguous()


def _device(what: str, *tensors: Optional[torch.Tensor]) -> int:
    """The index of the one device that all tensors are on."""

    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0):
            _hip.require_device(*tensors, what=what)
    return index


def _call(index: int, name: str, fn, *args) -> None:
    """fn(*args, stream) on a device's current stream, the device the current one
    for the call where it is not."""

    now = torch._C._cuda_getDevice()
    if now != index:
        with torch.cuda.device(index):
            return _call(index, name, fn, *args)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if _hip.TIMER.enabled:
        with _hip.TIMER.timed(name):
            rc = fn(*args, stream)
    else:
        rc = fn(*args, stream)
    if rc:
        _hip.check(rc, fn.__name__)


@functools.lru_cache(maxsize=256)
def _attend_bytes(*sizes: int) -> int:
    """Workspace of one-token attention: B, query heads, kv heads, page size,
    head dim, cell tag, the table's pages, listed pages or -1."""

    return _size_out(_hip.lib().pfa_paged_attn_workspace_size, *sizes)


@functools.lru_cache(maxsize=256)
def _select_bytes(*sizes: int) -> int:
    """Workspace of selection: B, kv heads, head dim, the table's pages."""

    return _size_out(_hip.lib().pfa_kv_pages_select_workspace_size, *sizes)


@functools.lru_cache(maxsize=256)
def _sparse_bytes(*sizes: int) -> int:
    """Workspace of both: as of attention, with the pages to choose."""

    return _size_out(_hip.lib().pfa_paged_sparse_attn_workspace_size, *sizes)


def _scratch(nbytes: int, device: torch.device) -> Tuple[Optional[torch.Tensor], Optional[int], int]:
    """A workspace of the call's own, from torch's allocator on the current
    stream, its address and size."""

    if nbytes == 0:
        return None, None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), nbytes


def write_kv_pages(pages: KVPages, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, starts: torch.Tensor,
                   *, counts: Optional[torch.Tensor] = None) -> None:
    """New tokens ``k``, ``v`` ``(B, n, kv_heads, head_dim)`` into the pages of
    their sequences: token i of sequence b, for i < ``counts[b]`` (all n
    without ``counts``), goes to position ``starts[b] + i``.  Positions below
    zero, behind the table's last page or without a page are left out.

    Values have the pages' type, or f32, bf16 or f16 for 8-bit pages: a row is
    divided by ``scale = max(absmax / top, 1e-6)`` (top 127 for int8, 448 for
    e4m3) and rounded to nearest even.  A row with a value that is not finite
    gets scale NaN, and reads back as NaN.  The pages' key bounds, where the
    pool has them, follow: they start anew with a page's first slot, so a page
    is written from there on.

    Two sequences of one call must not write to one page.
    """

    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or v.shape != shape or v.dtype != dtype:
        raise ValueError("k and v must be (B, n, kv_heads, head_dim) tensors of one shape and dtype")
    B, n, H, D = shape
    pool = _pool(pages)
    pool_heads, pool_dim = pool[8], pool[10]
    if H != pool_heads or D != pool_dim:
        raise ValueError(f"k and v have {H} heads of {D}, the pages {pool_heads} of {pool_dim}")
    tag, cells = _VALUE_TAG.get(dtype), pages[0].dtype
    if tag is None or (cells != dtype and cells not in _EIGHT_BITS):
        raise ValueError(f"values of {dtype} for pages of {cells}")
    table, starts = _table(block_table, B), _per_sequence(starts, B, "starts")
    if counts is not None:
        counts = _per_sequence(counts, B, "counts")
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError("write_kv_pages has no backward pass: call it under torch.no_grad()")
    index = _device("write_kv_pages", k, v, *pages, table, starts, counts)
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[3] != 1:
        v = v.contiguous()
        vs = v.stride()
    _call(index, "kv_pages_write", _hip.lib().pfa_kv_pages_write, _POOL.pack(*pool),
          _TENSOR4.pack(k.data_ptr(), ks[0], ks[2], ks[1]), _TENSOR4.pack(v.data_ptr(), vs[0], vs[2], vs[1]), tag, B, n,
          table.data_ptr(), table.stride(0), table.shape[1], starts.data_ptr(),
          None if counts is None else counts.data_ptr())


def read_kv_pages(pages: KVPages, block_table: torch.Tensor, starts: torch.Tensor, counts: Optional[torch.Tensor],
                  n: int, *, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Positions ``starts[b] .. starts[b] + counts[b] - 1`` (``counts`` None:
    n of them) of every sequence: k and v ``(B, n, kv_heads, head_dim)`` in
    ``dtype`` (default: the pages' type, f32 for 8-bit pages).  Rows
    i >= ``counts[b]``, and those without a page, are zero."""

    pool = _pool(pages)
    H, D = pool[8], pool[10]
    B, n = block_table.shape[0] if block_table.dim() else 0, int(n)
    table, starts = _table(block_table, B), _per_sequence(starts, B, "starts")
    if counts is not None:
        counts = _per_sequence(counts, B, "counts")
    if n < 0:
        raise ValueError("n must not be negative")
    if dtype is None:
        dtype = torch.float32 if pages[0].dtype in _EIGHT_BITS else pages[0].dtype
    tag = _VALUE_TAG.get(dtype)
    if tag is None:
        raise ValueError(f"unsupported value dtype {dtype}")
    index = _device("read_kv_pages", *pages, table, starts, counts)
    device = table.device
    k = torch.empty((B, n, H, D), dtype=dtype, device=device)
    v = torch.empty((B, n, H, D), dtype=dtype, device=device)
    _call(index, "kv_pages_read", _hip.lib().pfa_kv_pages_read, _POOL.pack(*pool), B, n, table.data_ptr(), table.stride(0),
          table.shape[1], starts.data_ptr(), None if counts is None else counts.data_ptr(), k.data_ptr(), v.data_ptr(),
          tag)
    return k, v


def _query(what: str, q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor,
           starts: Optional[torch.Tensor], selected: Optional[torch.Tensor] = None) -> tuple:
    """The arguments that selection and attention share, checked: packed for the
    library, (B, heads, kv_heads, page size, head dim, cell tag, the table's pages),
    the device's index, q, and what must stay referenced until the call is made."""

    shape, dtype = q.shape, q.dtype
    if len(shape) != 3:
        raise ValueError("q must be a (B, heads, head_dim) tensor: one new token a sequence")
    B, H, D = shape
    pool = _pool(pages)
    _, _, _, _, _, _, _, _, Hkv, ps, pool_dim, cell_tag = pool
    if D != pool_dim or H == 0 or H % Hkv:
        raise ValueError(f"q has {H} heads of {D}, the pages {Hkv} of {pool_dim}")
    tag, cells = _VALUE_TAG.get(dtype), pages[0].dtype
    if tag is None or (cells != dtype and cells not in _EIGHT_BITS):
        raise ValueError(f"queries of {dtype} for pages of {cells}")
    table, lengths = _table(block_table, B), _per_sequence(lengths, B, "lengths")
    P, starts_ptr = table.shape[1], 0
    if starts is not None:
        starts = _per_sequence(starts, B, "starts")
        starts_ptr = starts.data_ptr()
    if q.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{what} has no backward pass: call it under torch.no_grad()")
    index = _device(what, q, *pages, table, lengths, starts, selected)
    s = q.stride()
    if s[2] != 1:
        q = q.contiguous()
        s = q.stride()
    packed = _QUERY.pack(*pool, q.data_ptr(), s[0], s[1], 0, table.data_ptr(), table.stride(0), lengths.data_ptr(),
                         starts_ptr, P, B, H, tag)
    return packed, (B, H, Hkv, ps, D, cell_tag, P), index, q, (table, lengths, starts)


def _output(q: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _scale(scale: Optional[float]) -> Optional[float]:
    if scale is None:
        return None
    scale = float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    return scale


def paged_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, *,
                    starts: Optional[torch.Tensor] = None, selected: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one new token a sequence, ``q`` ``(B, heads, head_dim)``,
    over positions ``starts[b] .. lengths[b] - 1`` of its cache (``starts``
    None: from 0).  ``heads`` is a multiple of the pages' kv_heads, each of
    which serves as many query heads in a row.  With ``selected`` ``(B,
    kv_heads, S)`` int32 only positions in those entries of the sequence's
    table row count: entries outside of the row are left out, one listed twice
    counts twice.  ``scale`` defaults to 1 / sqrt(head_dim).

    Returns ``(B, heads, head_dim)`` in q's type; scores, weights and sums are
    f32, rounded once at the end.  A row that sees no key, or
    none with a score above -inf, is zero.  What stands in slots that no
    sequence sees has no effect, whatever it is; a value that is seen and not
    finite leaves its channel not finite (inf or NaN) in a row that sees another
    score than -inf, a score that is NaN or +inf its row NaN.
    """

    if selected is not None and (selected.dim() != 3 or selected.dtype != torch.int32 or selected.shape[2] > _MOST):
        raise ValueError(f"selected must be a (B, kv_heads, S) int32 tensor of up to {_MOST} entries a list")
    scale = _scale(scale)
    packed, sizes, index, q, keep = _query("paged_attention", q, pages, block_table, lengths, starts, selected)
    S, selected_ptr = -1, None
    if selected is not None:
        if selected.shape[:2] != (sizes[0], sizes[2]):
            raise ValueError("selected must be a (B, kv_heads, S) int32 tensor")
        selected = selected.contiguous()
        S, selected_ptr = selected.shape[2], selected.data_ptr()
    ws, ws_ptr, ws_bytes = _scratch(_attend_bytes(*sizes, S), q.device)
    out = _output(q)
    _call(index, "paged_attn_fwd", _hip.lib().pfa_paged_attn_fwd, packed, selected_ptr, max(S, 0), S,
          1.0 / math.sqrt(sizes[4]) if scale is None else scale, out.data_ptr(), ws_ptr, ws_bytes)
    return out


def _counted(pages: KVPages, count: int, first: int, last: int) -> Tuple[int, int, int]:
    count, first, last = int(count), int(first), int(last)
    if pages[4] is None:
        raise ValueError("selection needs pages with k_bounds")
    if not 1 <= count <= _MOST or first < 0 or last < 0 or first + last > count:
        raise ValueError(f"count must be positive, at most {_MOST}, and hold the first and last pages")
    return count, first, last


def select_kv_pages(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, count: int, *,
                    first: int = 1, last: int = 1, starts: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The ``count`` pages of each sequence and key-value head whose keys can
    score highest: ``(B, kv_heads, count)`` int32, entries of the sequence's
    table row in ascending order, -1 behind the last.

    A page's score is the largest, over the query heads that share the
    key-value head, of ``sum_d q_d * (max_d if q_d > 0 else min_d)`` with the
    bounds of its keys, an upper bound of every ``q . k`` in it; summed in 64
    bits, held in 32, NaN below everything.  The ``first`` first and ``last``
    last pages that hold a position to attend to are always taken; then the
    better score wins, ties the lower entry.
    """

    count, first, last = _counted(pages, count, first, last)
    packed, (B, _, Hkv, _, D, _, P), index, q, keep = _query("select_kv_pages", q, pages, block_table, lengths, starts)
    ws, ws_ptr, ws_bytes = _scratch(_select_bytes(B, Hkv, D, P), q.device)
    chosen = torch.empty((B, Hkv, count), dtype=torch.int32, device=q.device)
    _call(index, "kv_pages_select", _hip.lib().pfa_kv_pages_select, packed, count, first, last, chosen.data_ptr(), ws_ptr,
          ws_bytes)
    return chosen


def paged_sparse_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor,
                           count: int, *, first: int = 1, last: int = 1, starts: Optional[torch.Tensor] = None,
                           scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`paged_attention` over the pages that :func:`select_kv_pages`
    chooses.  Returns the output and the chosen entries."""

    count, first, last = _counted(pages, count, first, last)
    scale = _scale(scale)
    packed, sizes, index, q, keep = _query("paged_sparse_attention", q, pages, block_table, lengths, starts)
    ws, ws_ptr, ws_bytes = _scratch(_sparse_bytes(*sizes, count), q.device)
    out = _output(q)
    chosen = torch.empty((sizes[0], sizes[2], count), dtype=torch.int32, device=q.device)
    _call(index, "paged_sparse_attn_fwd", _hip.lib().pfa_paged_sparse_attn_fwd, packed, count, first, last,
          1.0 / math.sqrt(sizes[4]) if scale is None else scale, chosen.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes)
    return out, chosen


__all__ = [
    "KVPages",
    "new_kv_pages",
    "write_kv_pages",
    "read_kv_pages",
    "select_kv_pages",
    "paged_attention",
    "paged_sparse_attention",
]
