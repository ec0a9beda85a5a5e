"""One-token attention's 16-bit results against 32-bit arithmetic: how many are not
the 64-bit result rounded once.  A rounding hides the error of the sums before it
from any norm, but not the results that the error makes fall on its other side."""
from __future__ import annotations

import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _gathered(pool, m, table):
    """(B, Hkv, P * page, D) f32 or f64."""
    x = pool[m].to(DEV)
    x = x.float() if m + "_scale" not in pool else x.float() * pool[m + "_scale"].to(DEV)[..., None]
    return x[table.long()].transpose(1, 2).flatten(2, 3)


@pytest.mark.parametrize("pair", [p for p in R.PAIRS if p[0] != torch.float32], ids=R.pair_id)
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("form", ["whole", "shared"])
def test_no_further_from_64_bits_than_32_bits(pair, D, form):
    """Against elementary torch operations in f32 on the same device, which hold
    probabilities in 24 bits.  n results on the other side of a rounding scatter by
    sqrt(n) on each side of the comparison: four sigma and a few."""
    from proteus_attention import KVPages, paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(31)
    # 512 pairs and more of up to 16 tiles, a workgroup each; 248 of 24 or 47, shared out
    B, H, G, ps, n = (64, 8, 512 // D, 32, 512) if form == "whole" else (31, 8, 16, 32, 1500)
    P = -(-n // ps)
    pool = R.make_pool(B * P, H, ps, D, cell, g)
    table = torch.randperm(B * P, generator=g).view(B, P).to(torch.int32).to(DEV)
    lengths = torch.randint(n // 2, n + 1, (B,), generator=g).to(torch.int32).to(DEV)
    q = torch.randn(B, H * G, D, generator=g).to(dt).to(DEV)
    got = paged_attention(q, KVPages(**{m: t.to(DEV) for m, t in pool.items()}), table, lengths)
    seen = (torch.arange(P * ps, device=DEV) < lengths[:, None])[:, None, None]
    k, v = _gathered(pool, "k", table), _gathered(pool, "v", table)

    def plain(k, v):
        qq = q.to(k.dtype).view(B, H, G, D)
        s = torch.matmul(qq, k.transpose(2, 3).contiguous()) / math.sqrt(D)
        s = s.masked_fill(~seen, -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        return (torch.matmul(e, v) / e.sum(-1, keepdim=True)).view(B, H * G, D)

    near = plain(k, v).to(dt)
    want = plain(k.double(), v.double()).to(dt)
    n_near, n_got = int((near != want).sum()), int((got != want).sum())
    assert n_got <= n_near + 4 * math.sqrt(2 * n_near) + 8, (n_near, n_got, want.numel())
