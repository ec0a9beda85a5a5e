"""Refusals of 4-bit pools, of key weights and of eviction, on the CPU: argument errors
come before the device is looked at, and none of them reaches a kernel."""
from __future__ import annotations

import ctypes
import math
import struct

import pytest
import torch

from proteus_attention import (_hip, evict_kv_tokens, new_kv_pages, paged_attention, paged_sparse_attention, read_kv_pages,
                               select_kv_pages, select_kv_tokens, write_kv_pages)

FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _new(**kw):
    args = dict(num_pages=6, kv_heads=2, page_size=16, head_dim=64, dtype=FP4, bounds=True, device="cpu")
    args.update(kw)
    return new_kv_pages(**args)


TABLE = torch.zeros(1, 2, dtype=torch.int32)
INTO = torch.ones(1, 2, dtype=torch.int32)
ONE = torch.ones(1, dtype=torch.int32)
Q = torch.zeros(1, 4, 64)
KV = torch.zeros(1, 3, 2, 64)
W = torch.zeros(1, 2, 32)


def test_shapes_of_4_bit_pools():
    for D, scales in ((16, 1), (32, 1), (64, 2), (128, 4)):
        p = _new(head_dim=D)
        assert p.k.dtype == p.v.dtype == FP4 and p.k.shape == p.v.shape == (6, 2, 16, D // 2)
        assert p.k_scale.dtype == E8M0 and p.k_scale.shape == p.v_scale.shape == (6, 2, 16, scales)
        assert p.k_bounds.dtype == torch.bfloat16 and p.k_bounds.shape == (6, 2, 2, D)


def test_pools_that_do_not_fit():
    p = _new()
    raw = p.k.view(torch.uint8)
    bad = [p._replace(k_scale=None), p._replace(v_scale=None), p._replace(k_scale=p.k_scale.view(torch.uint8)),
           p._replace(k_scale=p.k_scale[..., :1]), p._replace(v_scale=torch.zeros(6, 2, 16)),
           p._replace(k_bounds=p.k_bounds.float()), p._replace(k=raw, v=raw), p._replace(v=p.v[:3]),
           p._replace(k=p.k.transpose(1, 2), v=p.v.transpose(1, 2)),
           p._replace(k=p.k[..., :16], v=p.v[..., :16])]
    for pages in bad:
        with pytest.raises(ValueError):
            paged_attention(Q, pages, TABLE, ONE)


def test_cpu_tensors_fail_loudly():
    p = _new()
    for call in (lambda: write_kv_pages(p, KV.half(), KV.half(), TABLE, ONE), lambda: read_kv_pages(p, TABLE, ONE, None, 3),
                 lambda: paged_attention(Q.bfloat16(), p, TABLE, ONE), lambda: select_kv_pages(Q, p, TABLE, ONE, 2),
                 lambda: paged_sparse_attention(Q, p, TABLE, ONE, 2), lambda: select_kv_tokens(W, ONE, 3),
                 lambda: paged_attention(Q, p, TABLE, ONE, key_weights=W),
                 lambda: evict_kv_tokens(p, W, TABLE, ONE, 3, INTO)):
        with pytest.raises(_hip.HipLibraryError):
            call()


@pytest.mark.parametrize("call", [
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=W[..., :31]),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=W[:, :1]),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=W[0]),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=W.double()),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=W.repeat(2, 1, 1)),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=W[:, :1].expand(1, 2, 32)),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=torch.zeros(1, 2, 1).expand(1, 2, 32)),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=torch.zeros(1, 32, 2).transpose(1, 2)),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=torch.zeros(40).as_strided((1, 2, 32), (64, 8, 1))),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=W, selected=torch.zeros(1, 2, 1, dtype=torch.int32)),
    lambda p: paged_attention(Q, p, TABLE, ONE, key_weights=W, scale=0.0),
    lambda p: evict_kv_tokens(p, W, TABLE, ONE, 0, INTO),
    lambda p: evict_kv_tokens(p, W, TABLE, ONE, 3, INTO, first=2, last=2),
    lambda p: evict_kv_tokens(p, W, TABLE, ONE, 3, INTO, last=-1),
    lambda p: evict_kv_tokens(p, W, TABLE, ONE, 3, INTO.long()),
    lambda p: evict_kv_tokens(p, W, TABLE, ONE, 3, INTO[0]),
    lambda p: evict_kv_tokens(p, W, TABLE, ONE, 3, TABLE),
    lambda p: evict_kv_tokens(p, W, TABLE, ONE.long(), 3, INTO),
    lambda p: evict_kv_tokens(p, W[:, :1], TABLE, ONE, 3, INTO),
    lambda p: evict_kv_tokens(p, W.half(), TABLE, ONE, 3, INTO),
    lambda p: evict_kv_tokens(p._replace(k_scale=None), W, TABLE, ONE, 3, INTO),
    lambda p: select_kv_tokens(W, ONE, 3, first=3),
    lambda p: select_kv_tokens(W, ONE, 2 ** 32 + 1),
    lambda p: select_kv_tokens(W[0], ONE, 3),
    lambda p: select_kv_tokens(W[:, :0], ONE, 3),
    lambda p: select_kv_tokens(W, torch.ones(2, dtype=torch.int32), 3),
    lambda p: select_kv_tokens(torch.empty(1, 2, 2 ** 31, device="meta"), ONE, 3),
])
def test_arguments_that_do_not_fit(call):
    with pytest.raises(ValueError):
        call(_new())


def test_no_backward():
    w = W.clone().requires_grad_()
    for call in (lambda: paged_attention(Q, _new(), TABLE, ONE, key_weights=w), lambda: select_kv_tokens(w, ONE, 3),
                 lambda: paged_attention(Q.clone().requires_grad_(), _new(), TABLE, ONE, key_weights=W),
                 lambda: evict_kv_tokens(_new(), w, TABLE, ONE, 3, INTO)):
        with pytest.raises(NotImplementedError):
            call()


_POOL, _TENSOR4, _QUERY = "PPPPPqqiiiii4x", "Pqqq", "PqPPiiii"  # include/pfa_hip.h


def _fields(**kw):
    a = dict(k=256, v=256, k_scale=256, v_scale=256, k_bounds=0, k_page=2 * 16 * 32, v_page=2 * 16 * 32, n_pages=4,
             kv_heads=2, page_size=16, head_dim=64, dtype=_hip.PFA_E2M1)
    a.update(kw)
    return list(a.values())


def test_c_entries_refuse_before_any_launch():
    lib = _hip.lib()
    p = ctypes.c_void_p(256)  # never dereferenced

    def query(P=2, B=1, H=2, **kw):
        return struct.pack(_POOL + _TENSOR4 + _QUERY, *_fields(**kw), 256, 128, 64, 0, 256, P, 256, 0, P, B, H, 0)

    def weigh(w=p, n=32, scale=0.5, out=p, ws=p, size=1 << 40, **kw):
        return lib.pfa_paged_weigh_attn_fwd(query(**kw), w, 64, 32, n, scale, out, ws, size, None)

    def evict(w=256, n=32, B=1, table=256, P=2, lengths=256, count=3, first=1, last=1, into=256, P2=2, kept=256, fresh=256,
              ws=256, size=1 << 40, **kw):
        return lib.pfa_kv_tokens_evict(struct.pack(_POOL + "PqqqPPPqqPPPqiiiiii", *_fields(**kw), w, 64, 32, n, table, into,
                                                   lengths, P, P2, kept, fresh, ws, size, P, P2, B, count, first, last), None)

    def select(w=p, n=32, B=1, H=2, lengths=p, count=3, first=1, last=1, kept=p, ws=p, size=1 << 40):
        return lib.pfa_kv_tokens_select(w, 64, 32, n, B, H, lengths, count, first, last, kept, ws, size, None)

    bad = [weigh(w=None), weigh(w=ctypes.c_void_p(258)), weigh(n=31), weigh(scale=0.0), weigh(scale=math.nan), weigh(out=None),
           weigh(H=3), weigh(k_scale=0), weigh(k_page=2 * 16 * 32 - 16), weigh(v_page=2 * 16 * 32 + 8), weigh(k=264),
           weigh(B=-1), weigh(head_dim=48), lib.pfa_paged_weigh_attn_fwd(None, p, 64, 32, 32, 0.5, p, p, 1 << 40, None),
           lib.pfa_kv_tokens_evict(None, None), evict(w=0), evict(w=257), evict(n=-1), evict(n=(1 << 30) + 1), evict(B=-1), evict(table=0),
           evict(P=-1), evict(lengths=0), evict(count=0), evict(count=1), evict(first=3), evict(last=-1), evict(into=0),
           evict(P2=-1), evict(P2=1 << 28), evict(kept=0), evict(fresh=0), evict(v_scale=0), evict(dtype=6),
           select(w=None), select(n=-1), select(B=70000), select(B=60000, H=60), select(H=0), select(lengths=None),
           select(count=0), select(count=-3, first=0, last=0), select(kept=None), select(last=3)]
    assert bad == [-1] * len(bad)
    assert weigh(size=8) == -3 and weigh(ws=ctypes.c_void_p(264)) == -3 and weigh(ws=None) == -3
    long = dict(n=70000, P=4400)
    assert [evict(ws=0, **long), evict(ws=264, **long), evict(size=4096, **long)] == [-3] * 3
    assert [select(n=70000, ws=None), select(n=70000, ws=ctypes.c_void_p(264)), select(n=70000, size=4096)] == [-3] * 3
    size = ctypes.c_size_t(0)
    assert lib.pfa_kv_tokens_workspace_size(3, 8, 65536, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.pfa_kv_tokens_workspace_size(3, 8, 65537, ctypes.byref(size)) == 0 and size.value >= 3 * 8 * 2 * 8192
    assert lib.pfa_kv_tokens_workspace_size(0, 8, 1 << 30, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.pfa_kv_tokens_workspace_size(1, 8, (1 << 30) + 1, ctypes.byref(size)) == -1
    assert lib.pfa_kv_tokens_workspace_size(60000, 60, 9, ctypes.byref(size)) == -1
    assert lib.pfa_paged_weigh_attn_workspace_size(1, 4, 2, 16, 64, _hip.PFA_E2M1, 100, ctypes.byref(size)) == 0
    assert size.value >= 4 * 4 * 1600
    assert lib.pfa_paged_weigh_attn_workspace_size(1, 3, 2, 16, 64, _hip.PFA_E2M1, 100, ctypes.byref(size)) == -1
    # nothing to do: no launch, no error
    assert weigh(B=0) == 0 and evict(B=0) == 0 and select(B=0) == 0
