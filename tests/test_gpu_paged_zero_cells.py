"""Cells of zeros: the sign that a division leaves."""
from __future__ import annotations

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("D", [16, 128])
def test_zeros_keep_their_sign(dt, D):
    """e4m3 has zeros of both signs: -0, and values that round to it, are 0x80."""
    from proteus_attention import new_kv_pages, write_kv_pages

    g = torch.Generator().manual_seed(D)
    x = torch.randn(1, 20, 2, D, generator=g)
    x[:, ::2, :, ::3] = -0.0
    x[:, 1::2, :, ::5] *= 1e-5
    x[:, 7] = -0.0
    x[:, 8] = 0.0
    x = x.to(dt)
    pages = new_kv_pages(2, 2, 16, D, dtype=torch.float8_e4m3fn, device=DEV)
    write_kv_pages(pages, x.to(DEV), x.neg().to(DEV), torch.tensor([[0, 1]], dtype=torch.int32, device=DEV),
                   torch.zeros(1, dtype=torch.int32, device=DEV))
    for got, new in ((pages.k, x), (pages.v, x.neg())):
        rows = got.cpu().view(torch.uint8).transpose(1, 2).reshape(1, 32, 2, D)[:, :20]
        assert torch.equal(rows, R.quantise(new, torch.float8_e4m3fn)[0].view(torch.uint8))
