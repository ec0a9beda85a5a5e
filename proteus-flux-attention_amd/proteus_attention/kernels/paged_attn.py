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

import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch

from .. import _hip
from .sparse_attn import _workspace

HEAD_DIMS = (16, 32, 64, 128)
PAGE_SIZES = (16, 32, 64, 128, 256)

_VALUE_TAG = {torch.float32: _hip.PFA_F32, torch.bfloat16: _hip.PFA_BF16, torch.float16: _hip.PFA_F16}
_CELL_TAG = {**_VALUE_TAG, torch.int8: _hip.PFA_I8, torch.float8_e4m3fn: _hip.PFA_E4M3}
_EIGHT_BITS = (torch.int8, torch.float8_e4m3fn)


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


def _dense(t: torch.Tensor, shape: Tuple[int, ...], dtype: torch.dtype, name: str) -> int:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}")
    return t.data_ptr()


def _pool(pages: KVPages) -> "_hip.KVPagesC":
    k, v, k_scale, v_scale, bounds = pages
    dtype = k.dtype
    tag = _CELL_TAG.get(dtype)
    if tag is None or v.dtype != dtype:
        raise ValueError(f"k and v pages must share one of {tuple(_CELL_TAG)} (got {dtype}, {v.dtype})")
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError("k and v pages must be (pages, kv_heads, page_size, head_dim) tensors of one shape")
    N, H, ps, D = shape = tuple(k.shape)
    if D not in HEAD_DIMS or ps not in PAGE_SIZES:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} and page_size one of {PAGE_SIZES} (got {D}, {ps})")
    if N == 0 or H == 0:
        raise ValueError("an empty pool")
    for t in (k, v):
        s = t.stride()
        if s[3] != 1 or s[2] != D or (H > 1 and s[1] != ps * D):
            raise ValueError("a page's heads, slots and channels must be dense")
    ks = vs = kb = None
    if dtype in _EIGHT_BITS:
        if k_scale is None or v_scale is None:
            raise ValueError("8-bit pages need k_scale and v_scale")
        ks = _dense(k_scale, shape[:3], torch.float32, "k_scale")
        vs = _dense(v_scale, shape[:3], torch.float32, "v_scale")
    if bounds is not None:
        kb = _dense(bounds, (N, H, 2, D), torch.float32 if dtype in _EIGHT_BITS else dtype, "k_bounds")
    return _hip.KVPagesC(k.data_ptr(), v.data_ptr(), ks, vs, kb, k.stride(0), v.stride(0), N, H, ps, D, tag)


def _table(block_table: torch.Tensor) -> torch.Tensor:
    if block_table.dim() != 2 or block_table.dtype != torch.int32:
        raise ValueError("block_table must be a (B, P) int32 tensor")
    return block_table if block_table.stride(1) == 1 or block_table.shape[1] <= 1 else block_table.contiguous()


def _per_sequence(t: Optional[torch.Tensor], B: int, name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != B or t.dtype != torch.int32:
        raise ValueError(f"{name} must be a ({B},) int32 tensor")
    return t if t.is_contiguous() else t.contiguous()


def _inference(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} has no backward pass: call it under torch.no_grad()")


class _OnDevice:
    """Makes a tensor's device the current one for a call, where it is not."""

    __slots__ = ("index", "before")

    def __init__(self, device: torch.device) -> None:
        self.index = device.index

    def __enter__(self):
        now = torch.cuda.current_device()
        self.before = -1 if now == self.index else now
        if self.before >= 0:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.before >= 0:
            torch.cuda.set_device(self.before)
        return False


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
    pool has them, follow: they start anew with a page's first slot.

    Two sequences of one call must not write to one page.
    """

    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k and v must be (B, n, kv_heads, head_dim) tensors of one shape and dtype")
    B, n, H, D = k.shape
    pool = _pool(pages)
    if H != pool.kv_heads or D != pool.head_dim:
        raise ValueError(f"k and v have {H} heads of {D}, the pages {pool.kv_heads} of {pool.head_dim}")
    tag = _VALUE_TAG.get(k.dtype)
    if tag is None or (pages.k.dtype not in _EIGHT_BITS and pages.k.dtype != k.dtype):
        raise ValueError(f"values of {k.dtype} for pages of {pages.k.dtype}")
    table = _table(block_table)
    starts, counts = _per_sequence(starts, B, "starts"), _per_sequence(counts, B, "counts")
    if starts is None or table.shape[0] != B:
        raise ValueError("block_table and starts need one row per sequence")
    _inference("write_kv_pages", k, v)
    device = _hip.require_device(*pages, k, v, table, starts, counts, what="write_kv_pages")
    if k.stride(3) != 1:
        k = k.contiguous()
    if v.stride(3) != 1:
        v = v.contiguous()
    with _OnDevice(device), _hip.TIMER.timed("kv_pages_write"):
        rc = _hip.lib().pfa_kv_pages_write(
            pool, _hip.Tensor4(k.data_ptr(), k.stride(0), k.stride(2), k.stride(1)),
            _hip.Tensor4(v.data_ptr(), v.stride(0), v.stride(2), v.stride(1)), tag, B, n, table.data_ptr(),
            table.stride(0), table.shape[1], starts.data_ptr(), _hip.ptr(counts), _hip.stream_ptr(device))
    _hip.check(rc, "pfa_kv_pages_write")


def read_kv_pages(pages: KVPages, block_table: torch.Tensor, starts: torch.Tensor, counts: Optional[torch.Tensor],
                  n: int, *, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Positions ``starts[b] .. starts[b] + counts[b] - 1`` (``counts`` None:
    n of them) of every sequence: k and v ``(B, n, kv_heads, head_dim)`` in
    ``dtype`` (default: the pages' type, f32 for 8-bit pages).  Rows
    i >= ``counts[b]``, and those without a page, are zero."""

    pool = _pool(pages)
    table = _table(block_table)
    B, n = table.shape[0], int(n)
    starts, counts = _per_sequence(starts, B, "starts"), _per_sequence(counts, B, "counts")
    if starts is None:
        raise ValueError("starts needs one entry per sequence")
    if n < 0:
        raise ValueError("n must not be negative")
    if dtype is None:
        dtype = torch.float32 if pages.k.dtype in _EIGHT_BITS else pages.k.dtype
    tag = _VALUE_TAG.get(dtype)
    if tag is None:
        raise ValueError(f"unsupported value dtype {dtype}")
    device = _hip.require_device(*pages, table, starts, counts, what="read_kv_pages")
    k, v = (torch.empty(B, n, pool.kv_heads, pool.head_dim, dtype=dtype, device=device) for _ in range(2))
    with _OnDevice(device), _hip.TIMER.timed("kv_pages_read"):
        rc = _hip.lib().pfa_kv_pages_read(pool, B, n, table.data_ptr(), table.stride(0), table.shape[1],
                                          starts.data_ptr(), _hip.ptr(counts), k.data_ptr(), v.data_ptr(), tag,
                                          _hip.stream_ptr(device))
    _hip.check(rc, "pfa_kv_pages_read")
    return k, v


class _Query(NamedTuple):
    """The checked arguments that selection and attention share."""

    pool: "_hip.KVPagesC"
    q: torch.Tensor
    q4: "_hip.Tensor4"
    tag: int
    table: torch.Tensor
    lengths: torch.Tensor
    starts: Optional[torch.Tensor]
    device: torch.device


def _query(what: str, q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor,
           starts: Optional[torch.Tensor], selected: Optional[torch.Tensor] = None) -> _Query:
    if q.dim() != 3:
        raise ValueError("q must be a (B, heads, head_dim) tensor: one new token a sequence")
    B, H, D = q.shape
    pool = _pool(pages)
    if D != pool.head_dim or H == 0 or H % pool.kv_heads:
        raise ValueError(f"q has {H} heads of {D}, the pages {pool.kv_heads} of {pool.head_dim}")
    tag = _VALUE_TAG.get(q.dtype)
    if tag is None or (pages.k.dtype not in _EIGHT_BITS and pages.k.dtype != q.dtype):
        raise ValueError(f"queries of {q.dtype} for pages of {pages.k.dtype}")
    table = _table(block_table)
    lengths, starts = _per_sequence(lengths, B, "lengths"), _per_sequence(starts, B, "starts")
    if lengths is None or table.shape[0] != B:
        raise ValueError("block_table and lengths need one row per sequence")
    _inference(what, q)
    device = _hip.require_device(q, *pages, table, lengths, starts, selected, what=what)
    if q.stride(2) != 1:
        q = q.contiguous()
    return _Query(pool, q, _hip.Tensor4(q.data_ptr(), q.stride(0), q.stride(1), 0), tag, table, lengths, starts, device)


def _scale(scale: Optional[float], D: int) -> float:
    if scale is None:
        return 1.0 / math.sqrt(D)
    scale = float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    return scale


def _attend(a: _Query, selected: Optional[torch.Tensor], scale: float) -> torch.Tensor:
    B, H, D = a.q.shape
    lib = _hip.lib()
    size = ctypes.c_size_t(0)
    P, S = a.table.shape[1], -1 if selected is None else selected.shape[2]
    _hip.check(lib.pfa_paged_attn_workspace_size(B, H, a.pool, P, S, ctypes.byref(size)),
               "pfa_paged_attn_workspace_size")
    ws = _workspace(size.value, a.device)
    out = torch.empty(B, H, D, dtype=a.q.dtype, device=a.device)
    with _OnDevice(a.device), _hip.TIMER.timed("paged_attn_fwd"):
        rc = lib.pfa_paged_attn_fwd(a.q4, a.tag, B, H, a.pool, a.table.data_ptr(), a.table.stride(0), P,
                                    a.lengths.data_ptr(), _hip.ptr(a.starts), _hip.ptr(selected), S, scale,
                                    out.data_ptr(), ws.data_ptr(), ws.numel(), _hip.stream_ptr(a.device))
    _hip.check(rc, "pfa_paged_attn_fwd")
    return out


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

    Returns ``(B, heads, head_dim)`` in q's type.  A row that sees no key, or
    none with a score above -inf, is zero.
    """

    a = _query("paged_attention", q, pages, block_table, lengths, starts, selected)
    if selected is not None:
        if selected.dim() != 3 or selected.shape[:2] != (q.shape[0], a.pool.kv_heads) or selected.dtype != torch.int32:
            raise ValueError("selected must be a (B, kv_heads, S) int32 tensor")
        selected = selected.contiguous()
    return _attend(a, selected, _scale(scale, q.shape[2]))


def _select(a: _Query, pages: KVPages, count: int, first: int, last: int) -> torch.Tensor:
    B, H, _ = a.q.shape
    count, first, last = int(count), int(first), int(last)
    if pages.k_bounds is None:
        raise ValueError("selection needs pages with k_bounds")
    if count < 1 or first < 0 or last < 0 or first + last > count:
        raise ValueError("count must be positive and hold the first and last pages")
    lib = _hip.lib()
    size = ctypes.c_size_t(0)
    P = a.table.shape[1]
    _hip.check(lib.pfa_kv_pages_select_workspace_size(B, a.pool.kv_heads, P, ctypes.byref(size)),
               "pfa_kv_pages_select_workspace_size")
    ws = _workspace(size.value, a.device)
    chosen = torch.empty(B, a.pool.kv_heads, count, dtype=torch.int32, device=a.device)
    with _OnDevice(a.device), _hip.TIMER.timed("kv_pages_select"):
        rc = lib.pfa_kv_pages_select(a.q4, a.tag, B, H, a.pool, a.table.data_ptr(), a.table.stride(0), P,
                                     a.lengths.data_ptr(), _hip.ptr(a.starts), count, first, last, chosen.data_ptr(),
                                     ws.data_ptr(), ws.numel(), _hip.stream_ptr(a.device))
    _hip.check(rc, "pfa_kv_pages_select")
    return chosen


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

    return _select(_query("select_kv_pages", q, pages, block_table, lengths, starts), pages, count, first, last)


def paged_sparse_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor,
                           count: int, *, first: int = 1, last: int = 1, starts: Optional[torch.Tensor] = None,
                           scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`paged_attention` over the pages that :func:`select_kv_pages`
    chooses.  Returns the output and the chosen entries."""

    a = _query("paged_sparse_attention", q, pages, block_table, lengths, starts)
    sc = _scale(scale, q.shape[2])
    chosen = _select(a, pages, count, first, last)
    return _attend(a, chosen, sc), chosen


__all__ = [
    "KVPages",
    "new_kv_pages",
    "write_kv_pages",
    "read_kv_pages",
    "select_kv_pages",
    "paged_attention",
    "paged_sparse_attention",
]
