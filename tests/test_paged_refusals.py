"""Refusals of the paged cache's calls, on the CPU: argument errors come before
the device is looked at, and none of them reaches a kernel."""
from __future__ import annotations

import ctypes
import math
import struct

import pytest
import torch

from proteus_attention import (KVPages, _hip, new_kv_pages, paged_attention, paged_sparse_attention, read_kv_pages,
                               select_kv_pages, write_kv_pages)


def _new(**kw):
    args = dict(num_pages=4, kv_heads=2, page_size=16, head_dim=32, dtype=torch.float32, bounds=True, device="cpu")
    args.update(kw)
    return new_kv_pages(**args)


TABLE = torch.zeros(1, 2, dtype=torch.int32)
ONE = torch.ones(1, dtype=torch.int32)
Q = torch.zeros(1, 4, 32)
KV = torch.zeros(1, 3, 2, 32)


def test_cpu_tensors_fail_loudly():
    p = _new()
    for call in (lambda: write_kv_pages(p, KV, KV, TABLE, ONE), lambda: read_kv_pages(p, TABLE, ONE, None, 3),
                 lambda: paged_attention(Q, p, TABLE, ONE), lambda: select_kv_pages(Q, p, TABLE, ONE, 2),
                 lambda: paged_sparse_attention(Q, p, TABLE, ONE, 2)):
        with pytest.raises(_hip.HipLibraryError):
            call()


@pytest.mark.parametrize("kw", [dict(head_dim=48), dict(page_size=24), dict(page_size=512), dict(num_pages=0),
                                dict(kv_heads=0), dict(dtype=torch.float64)], ids=str)
def test_pools_that_are_not_made(kw):
    with pytest.raises(ValueError):
        _new(**kw)


def test_pools_that_do_not_fit():
    p = _new()
    bad = [
        p._replace(v=p.v[:3]),
        p._replace(v=p.v.bfloat16()),
        p._replace(k=p.k.transpose(1, 2), v=p.v.transpose(1, 2)),
        p._replace(k=p.k.double(), v=p.v.double()),
        p._replace(k=p.k[:0], v=p.v[:0]),
        p._replace(k=p.k.to(torch.int8), v=p.v.to(torch.int8)),  # no scales
        p._replace(k_bounds=p.k_bounds.bfloat16()),
        p._replace(k_bounds=p.k_bounds[:, :1]),
        p._replace(k=p.k[..., :31], v=p.v[..., :31]),
        _new(dtype=torch.int8)._replace(k_scale=torch.zeros(4, 2, 15)),
        _new(dtype=torch.int8)._replace(v_scale=torch.zeros(4, 2, 16).double()),
    ]
    for pages in bad:
        with pytest.raises(ValueError):
            paged_attention(Q, pages, TABLE, ONE)


@pytest.mark.parametrize("call", [
    lambda p: write_kv_pages(p, KV, KV[:, :2], TABLE, ONE),
    lambda p: write_kv_pages(p, KV, KV.bfloat16(), TABLE, ONE),
    lambda p: write_kv_pages(p, KV.bfloat16(), KV.bfloat16(), TABLE, ONE),
    lambda p: write_kv_pages(p, KV[:, :, :1], KV[:, :, :1], TABLE, ONE),
    lambda p: write_kv_pages(p, KV, KV, TABLE.long(), ONE),
    lambda p: write_kv_pages(p, KV, KV, TABLE, ONE.long()),
    lambda p: write_kv_pages(p, KV, KV, TABLE, torch.ones(2, dtype=torch.int32)),
    lambda p: write_kv_pages(p, KV, KV, TABLE, ONE, counts=ONE.float()),
    lambda p: write_kv_pages(p, KV, KV, TABLE.repeat(2, 1), ONE),
    lambda p: read_kv_pages(p, TABLE, ONE, None, -1),
    lambda p: read_kv_pages(p, TABLE, ONE, None, 3, dtype=torch.int8),
    lambda p: read_kv_pages(p, TABLE[0], ONE, None, 3),
    lambda p: paged_attention(Q[0], p, TABLE, ONE),
    lambda p: paged_attention(Q[:, :3], p, TABLE, ONE),
    lambda p: paged_attention(Q[:, :0], p, TABLE, ONE),
    lambda p: paged_attention(Q[..., :16], p, TABLE, ONE),
    lambda p: paged_attention(Q.half(), p, TABLE, ONE),
    lambda p: paged_attention(Q, p, TABLE, ONE, scale=0.0),
    lambda p: paged_attention(Q, p, TABLE, ONE, scale=math.inf),
    lambda p: paged_attention(Q, p, TABLE, ONE, starts=ONE.long()),
    lambda p: paged_sparse_attention(Q, p, TABLE, ONE, 0),
    lambda p: paged_sparse_attention(Q, p, TABLE, ONE, 3, first=2, last=2),
    lambda p: paged_sparse_attention(Q, p, TABLE, ONE, 3, first=-1),
    lambda p: select_kv_pages(Q, p._replace(k_bounds=None), TABLE, ONE, 3),
])
def test_arguments_that_do_not_fit(call):
    with pytest.raises(ValueError):
        call(_new())


def test_no_backward():
    for call in (lambda: paged_attention(Q.clone().requires_grad_(), _new(), TABLE, ONE),
                 lambda: write_kv_pages(_new(), KV.clone().requires_grad_(), KV, TABLE, ONE)):
        with pytest.raises(NotImplementedError):
            call()


@pytest.mark.parametrize("name", ["k", "v", "k_bounds"])
def test_no_backward_of_pools(name):
    p = _new()
    p = p._replace(**{name: getattr(p, name).clone().requires_grad_()})
    for call in (lambda: write_kv_pages(p, KV, KV, TABLE, ONE), lambda: read_kv_pages(p, TABLE, ONE, None, 3),
                 lambda: paged_attention(Q, p, TABLE, ONE), lambda: select_kv_pages(Q, p, TABLE, ONE, 2),
                 lambda: paged_sparse_attention(Q, p, TABLE, ONE, 2)):
        with pytest.raises(NotImplementedError):
            call()
        with torch.no_grad(), pytest.raises(_hip.HipLibraryError):  # then only the device is wrong
            call()


WIDE = 2 ** 32 + 1  # 1 in the library's 32-bit arguments


def _wide(*shape):
    return torch.empty(shape, dtype=torch.int32, device="meta")  # no memory behind it


@pytest.mark.parametrize("call", [
    lambda p: select_kv_pages(Q, p, TABLE, ONE, WIDE),
    lambda p: paged_sparse_attention(Q, p, TABLE, ONE, WIDE),
    lambda p: paged_attention(Q, p, TABLE, ONE, selected=_wide(1, 2, WIDE)),
    lambda p: paged_attention(Q, p, _wide(1, WIDE), ONE),
    lambda p: read_kv_pages(p, _wide(1, WIDE), ONE, None, 3),
    lambda p: read_kv_pages(p, _wide(WIDE, 1), _wide(WIDE), None, 3),
    lambda p: write_kv_pages(p, KV, KV, _wide(1, WIDE), ONE),
])
def test_sizes_that_pass_32_bits(call):
    with pytest.raises(ValueError):
        call(_new())


_POOL, _TENSOR4, _QUERY = "PPPPPqqiiiii4x", "Pqqq", "PqPPiiii"  # include/pfa_hip.h


def _fields(**kw):
    a = dict(k=256, v=256, k_scale=0, v_scale=0, k_bounds=0, k_page=2 * 16 * 32, v_page=2 * 16 * 32, n_pages=4,
             kv_heads=2, page_size=16, head_dim=32, dtype=_hip.PFA_F32)
    a.update(kw)
    return list(a.values())


def _c_pool(**kw):
    return struct.pack(_POOL, *_fields(**kw))


def _c_query(pool=None, q=256, table=256, lengths=256, P=2, B=1, H=2, tag=_hip.PFA_F32):
    return struct.pack(_POOL + _TENSOR4 + _QUERY, *_fields(**(pool or {})), q, 64, 32, 0, table, P, lengths, 0, P, B, H, tag)


def test_c_entries_refuse_before_any_launch():
    lib = _hip.lib()
    t4 = struct.pack(_TENSOR4, 256, 64, 32, 32)
    p = ctypes.c_void_p(256)  # never dereferenced

    def attend(pool=None, n=-1, out=p, selected=None, stride=0, scale=0.5, **kw):
        return lib.pfa_paged_attn_fwd(_c_query(pool, **kw), selected, stride, n, scale, out, p, 1 << 40, None)

    def select(count, first, last, pool=None, ws=1 << 40, **kw):
        return lib.pfa_kv_pages_select(_c_query(pool, **kw), count, first, last, p, p, ws, None)

    def sparse(count, first, last, scale=0.5, chosen=p, out=p, ws=1 << 40, pool=None, **kw):
        return lib.pfa_paged_sparse_attn_fwd(_c_query(pool or dict(k_bounds=256), **kw), count, first, last, scale, chosen,
                                             out, p, ws, None)

    bad = [sparse(2, 1, 1, pool=dict(head_dim=32)), sparse(0, 0, 0), sparse(2, 2, 1), sparse(2, 1, 1, scale=0.0),
           sparse(2, 1, 1, scale=math.nan), sparse(2, 1, 1, chosen=None), sparse(2, 1, 1, out=None), sparse(2, 1, 1, H=3),
           lib.pfa_paged_sparse_attn_fwd(None, 2, 1, 1, 0.5, p, p, p, 0, None),
           attend(dict(head_dim=48)), attend(dict(page_size=48)), attend(dict(n_pages=0)), attend(dict(dtype=9)),
           attend(dict(dtype=_hip.PFA_I8)), attend(dict(k=264)), attend(dict(k_page=100)), attend(dict(kv_heads=0)),
           attend(B=-1), attend(B=70000), attend(H=3), attend(H=0), attend(tag=_hip.PFA_BF16), attend(tag=_hip.PFA_I8),
           attend(P=1 << 28), attend(P=-1), attend(n=2), attend(n=2, selected=p, stride=1),
           attend(n=1 << 28, selected=p, stride=1 << 28), attend(out=None), attend(lengths=0), attend(q=0),
           attend(table=0), attend(scale=0.0), attend(scale=math.inf), attend(scale=math.nan), attend(scale=-1.0),
           attend(B=60000, H=60),
           lib.pfa_paged_attn_fwd(None, None, 0, -1, 0.5, p, p, 0, None),
           select(2, 1, 1), select(2, 2, 1, dict(k_bounds=256)), select(0, 0, 0, dict(k_bounds=256)),
           select(2, -1, 1, dict(k_bounds=256)), lib.pfa_kv_pages_select(None, 2, 1, 1, p, p, 0, None),
           lib.pfa_kv_pages_read(_c_pool(), 1, -1, p, 2, 2, p, p, p, p, 0, None),
           lib.pfa_kv_pages_read(_c_pool(), 1, 5, p, 2, 2, p, p, p, p, _hip.PFA_I8, None),
           lib.pfa_kv_pages_read(None, 1, 5, p, 2, 2, p, p, p, p, 0, None),
           lib.pfa_kv_pages_write(_c_pool(), t4, t4, _hip.PFA_F16, 1, 3, p, 2, 2, p, p, None),
           lib.pfa_kv_pages_write(_c_pool(), t4, t4, _hip.PFA_F32, 1, 3, p, 2, 2, None, p, None),
           lib.pfa_kv_pages_write(_c_pool(), None, t4, _hip.PFA_F32, 1, 3, p, 2, 2, p, p, None)]
    assert bad == [-1] * len(bad)
    # workspaces: too small, or not aligned
    assert select(2, 1, 1, dict(k_bounds=256), P=600, ws=4) == -3
    assert sparse(2, 1, 1, P=600, ws=4) == -3 and sparse(2, 1, 1, B=0) == 0
    assert lib.pfa_paged_attn_fwd(_c_query(P=6000), None, 0, -1, 0.5, p, p, 4, None) == -3
    assert lib.pfa_paged_attn_fwd(_c_query(P=6000), None, 0, -1, 0.5, p, ctypes.c_void_p(264), 1 << 40, None) == -3
    size = ctypes.c_size_t(0)
    sizes = [(1, 4, 2, 16, 32, _hip.PFA_F32, 100, -1), (1, 3, 2, 16, 32, 0, 100, -1), (1, 4, 2, 24, 32, 0, 100, -1),
             (1, 4, 2, 16, 48, 0, 100, -1), (1, 4, 2, 16, 32, 7, 100, -1), (-1, 4, 2, 16, 32, 0, 100, -1)]
    assert [lib.pfa_paged_attn_workspace_size(*x, ctypes.byref(size)) for x in sizes] == [0] + [-1] * 5
    # nothing to do: no launch, no error
    assert attend(B=0) == 0
    assert lib.pfa_kv_pages_write(_c_pool(), t4, t4, 0, 1, 0, p, 2, 2, p, p, None) == 0
    assert lib.pfa_kv_pages_read(_c_pool(), 0, 5, p, 2, 2, p, p, p, p, 0, None) == 0


def test_select_reference_is_an_upper_bound():
    """The oracle's scores bound every q . k of their page (64 bits)."""
    import paged_reference as R

    g = torch.Generator().manual_seed(0)
    pool = R.make_pool(6, 2, 16, 32, torch.bfloat16, g, bounds=True)
    q = torch.randn(4, 32, generator=g).double()
    for page in range(6):
        for h in range(2):
            k = pool["k"][page, h].double()
            lo, hi = pool["k_bounds"][page, h].double()
            bound = (q * torch.where(q > 0, hi, lo)).sum(-1)
            assert bool((q @ k.T <= bound[:, None] + 1e-9).all())
