"""Rotary positions at the ends of what the call allows, on the GPU against 64 bits on
the CPU."""
from __future__ import annotations

import pytest
import torch

from test_gpu_rotary import DEV, holds

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [(1 << 24) - 1, (1 << 24) + 3])
def test_more_workgroups_than_a_grid_has(n):
    """A workgroup a token of 257 heads: from 2^24 tokens on, more threads than one grid."""
    from proteus_attention import apply_rotary, new_rotary_positions

    H, D = 257, 3
    rotary = new_rotary_positions(2, device=DEV)
    g = torch.Generator().manual_seed(n)
    far = torch.zeros(1, n, H, D, dtype=torch.float16, device=DEV)
    first = torch.tensor([-12345], dtype=torch.int32)
    some = torch.tensor([0, 1, 70001, (1 << 24) - 3, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, (1 << 24) + 1, n - 2, n - 1])
    some = some[some < n].unique()
    x = torch.randn(1, len(some), H, D, generator=g).half()
    far[:, some.to(DEV)] = x.to(DEV)
    got, _ = apply_rotary(far, None, first.to(DEV), rotary, inplace=True)
    assert got is far and holds(far[:, some.to(DEV)], x, first.long()[:, None] + some, rotary)
    far[:, some.to(DEV)] = 0.0
    assert not bool(far.any())  # the others are turned zeros


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_single_tokens_of_a_projection(dt, interleaved):
    """(B, heads, head_dim) as slices, written over or not, positions (B,) or (B, 1)."""
    from proteus_attention import apply_rotary, new_rotary_positions

    g = torch.Generator().manual_seed(3)
    B, H, Hk, D = 5, 6, 2, 64
    rotary = new_rotary_positions(48, interleaved=interleaved, magnitude=0.75, device=DEV)
    qkv, pos = torch.randn(B, H + 2 * Hk, D, generator=g).to(dt), torch.randint(-9, 9999, (B,), generator=g, dtype=torch.int32)
    d = qkv.to(DEV)
    q, k = apply_rotary(d[:, :H], d[:, H:H + Hk], pos.to(DEV), rotary)
    assert torch.equal(d.cpu(), qkv) and q.is_contiguous() and k.shape == (B, Hk, D)
    assert holds(q[:, None], qkv[:, None, :H], pos[:, None], rotary) and holds(k[:, None], qkv[:, None, H:H + Hk], pos[:, None], rotary)
    apply_rotary(d[:, :H], d[:, H:H + Hk], pos[:, None].to(DEV), rotary, inplace=True)
    assert torch.equal(d[:, :H], q) and torch.equal(d[:, H:H + Hk], k) and torch.equal(d[:, H + Hk:].cpu(), qkv[:, H + Hk:])
    odd = torch.zeros(B, H, D + 3, dtype=dt, device=DEV)[..., 3:].copy_(qkv[:, :H])
    apply_rotary(odd, None, pos.to(DEV), rotary, inplace=True)
    assert torch.equal(odd, q)
