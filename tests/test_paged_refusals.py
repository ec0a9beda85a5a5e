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


def _c_pool(**kw):
    a = dict(k=256, v=256, k_scale=None, v_scale=None, k_bounds=None, k_page=2 * 16 * 32, v_page=2 * 16 * 32, n_pages=4,
             kv_heads=2, page_size=16, head_dim=32, dtype=_hip.PFA_F32)
    a.update(kw)
    return struct.pack("PPPPPqqiiiii4x", *(x or 0 for x in a.values()))


def test_c_entries_refuse_before_any_launch():
    lib = _hip.lib()
    t4 = struct.pack("Pqqq", 256, 64, 32, 32)
    p = ctypes.c_void_p(256)  # never dereferenced

    def attend(pool, q=t4, tag=_hip.PFA_F32, B=1, H=2, P=2, n=-1, out=p, lengths=p):
        return lib.pfa_paged_attn_fwd(q, tag, B, H, pool, p, P, P, lengths, None, None, max(n, 0), n, 0.5, out, p, 1 << 40, None)

    bad = [attend(_c_pool(head_dim=48)), attend(_c_pool(page_size=48)), attend(_c_pool(n_pages=0)),
           attend(_c_pool(dtype=9)), attend(_c_pool(dtype=_hip.PFA_I8)), attend(_c_pool(k=264)),
           attend(_c_pool(k_page=100)), attend(_c_pool(), B=-1), attend(_c_pool(), B=70000), attend(_c_pool(), H=3),
           attend(_c_pool(), H=0), attend(_c_pool(), tag=_hip.PFA_BF16), attend(_c_pool(), P=1 << 28),
           attend(_c_pool(), n=2), attend(_c_pool(), out=None), attend(_c_pool(), lengths=None),
           lib.pfa_kv_pages_select(t4, 0, 1, 2, _c_pool(), p, 2, 2, p, None, 2, 1, 1, p, p, 1 << 40, None),
           lib.pfa_kv_pages_select(t4, 0, 1, 2, _c_pool(k_bounds=256), p, 2, 2, p, None, 2, 2, 1, p, p, 1 << 40, None),
           lib.pfa_kv_pages_read(_c_pool(), 1, -1, p, 2, 2, p, p, p, p, 0, None),
           lib.pfa_kv_pages_read(_c_pool(), 1, 5, p, 2, 2, p, p, p, p, _hip.PFA_I8, None),
           lib.pfa_kv_pages_write(_c_pool(), t4, t4, _hip.PFA_F16, 1, 3, p, 2, 2, p, p, None),
           lib.pfa_kv_pages_write(_c_pool(), t4, t4, _hip.PFA_F32, 1, 3, p, 2, 2, None, p, None)]
    assert bad == [-1] * len(bad)
    rc = lib.pfa_kv_pages_select(t4, 0, 1, 2, _c_pool(k_bounds=256), p, 600, 600, p, None, 2, 1, 1, p, p, 4, None)
    assert rc == -3
    size = ctypes.c_size_t(0)
    sizes = [(1, 4, 2, 16, 32, _hip.PFA_F32, 100, -1), (1, 3, 2, 16, 32, 0, 100, -1), (1, 4, 2, 24, 32, 0, 100, -1),
             (1, 4, 2, 16, 48, 0, 100, -1), (1, 4, 2, 16, 32, 7, 100, -1), (-1, 4, 2, 16, 32, 0, 100, -1)]
    assert [lib.pfa_paged_attn_workspace_size(*x, ctypes.byref(size)) for x in sizes] == [0] + [-1] * 5
    # nothing to do: no launch, no error
    assert attend(_c_pool(), B=0) == 0
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
