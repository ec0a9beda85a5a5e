"""Page selection where scores underflow to zeros of either sign."""
from __future__ import annotations

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("P", [40, 400, 1500, 17000])
@pytest.mark.parametrize("H", [1, 2])
def test_zeros_of_either_sign_are_equal(P, H):
    """A sum of -1e-60 is held as -0 in 32 bits, one of 1e-60 as +0: a tie, and the
    lower entry's.  Rows of one launch, of several, and in rounds."""
    from proteus_attention import KVPages, select_kv_pages

    D, ps = 16, 16
    k = torch.zeros(4, H, ps, D)
    bounds = torch.zeros(4, H, 2, D)
    bounds[0, ..., 0] = -1e-30  # -0 for q = 1e-30
    bounds[1, ..., 0] = 1e-30  # +0
    bounds[2, ..., 0] = -1.0  # below zero in 32 bits
    bounds[3, ..., 0] = 0.0
    q = torch.zeros(1, 2 * H, D)
    q[..., 0] = 1e-30
    g = torch.Generator().manual_seed(P)
    table = torch.randint(0, 4, (1, P), generator=g, dtype=torch.int32)
    pool = dict(k=k, v=k.clone(), k_bounds=bounds)
    pages = KVPages(**{m: t.to(DEV) for m, t in pool.items()})
    n = torch.tensor([P * ps], dtype=torch.int32)
    for count, first, last in ((1, 0, 0), (P // 4, 0, 1), (P - 3, 0, 0)):
        want = R.select(q, pool, table, n, None, count, first, last)
        got = select_kv_pages(q.to(DEV), pages, table.to(DEV), n.to(DEV), count, first=first, last=last).cpu()
        assert torch.equal(got, want), count
