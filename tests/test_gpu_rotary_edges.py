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
