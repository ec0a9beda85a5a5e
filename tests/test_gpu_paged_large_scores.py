"""One-token attention at scores so large that the rounding of a score is more than
a power of two: the largest weight of a row is one, and nothing overflows."""
from __future__ import annotations

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _attend(q, k, v, scale):
    """q (heads, D) over one sequence's keys and values (n, D) of one head, in pages
    of 16."""
    from proteus_attention import KVPages, paged_attention

    n, D = k.shape
    P = -(-n // 16)
    pool = torch.zeros(2, P * 16, D, dtype=k.dtype)
    pool[0, :n], pool[1, :n] = k, v
    pages = KVPages(*pool.view(2, P, 1, 16, D).to(DEV))
    table = torch.arange(P, dtype=torch.int32, device=DEV)[None]
    return paged_attention(q[None].to(DEV), pages, table, torch.tensor([n], dtype=torch.int32, device=DEV),
                           scale=scale)[0].cpu()


# values of q and k: f16 scores up to the type's end, the others' far beyond
LARGE = {torch.float16: [30.0, 200.0, 2000.0, 3000.0, 4000.0, 20000.0, 65504.0],
         torch.bfloat16: [3000.0, 1e6, 3e8, 1e12, 1e16], torch.float32: [3000.0, 1.1e6, 3.3e8, 1.7e12, 1e16]}


@pytest.mark.parametrize("dt", list(LARGE), ids=str)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 4])
def test_keys_alike(dt, D, n):
    """All keys the same: the mean of the values, whatever the score; of one
    key, its value to the bit.  Four: three sums and a division, 5 f32 roundings of
    at most 4 in size, and the result's own."""
    g = torch.Generator().manual_seed(D)
    v = torch.randn(n, D, generator=g).to(dt)
    for x in LARGE[dt]:
        for scale in (None, 0.3, 1.7):
            q = torch.full((5, D), x).to(dt)
            got = _attend(q, q[:1].expand(n, D), v, scale)
            want = v.double().mean(0)
            if n == 1:
                assert torch.equal(got, v.expand(5, D)), (x, scale)
            else:
                err = (got.double() - want).abs()
                assert bool((err <= R.HALF[dt] * want.abs() + 5 * 4 * 2.0 ** -24).all()), (x, scale)


@pytest.mark.parametrize("dt", list(LARGE), ids=str)
@pytest.mark.parametrize("D", [16, 64, 128])
def test_keys_nearly_alike(dt, D):
    """Scores that f32 holds exactly, 2^22 and a few in size: their differences alone
    decide.  A weight's error: the exponent, of up to 8 * 0.5 * log2(e) = 5.8, has
    three roundings (scale and its product with log2(e), the product) of 2^-24 each,
    times ln 2: 12.1 * 2^-24; its exponential 2 * 2^-24, sums of 40 weights 40 * 2^-24
    at the most, in the numerator and in the denominator, and one division: below
    110 * 2^-24 of sum p |v|."""
    g = torch.Generator().manual_seed(D + 1)
    n = 40
    q = torch.zeros(3, D)
    q[:, 0], q[:, 1] = 2048.0, 1.0
    k = torch.zeros(n, D)
    k[:, 0], k[:, 1] = 2048.0, torch.randint(0, 9, (n,), generator=g).float()
    q, k, v = q.to(dt), k.to(dt), torch.randn(n, D, generator=g).to(dt)
    p = torch.softmax(q.double() @ k.double().T * 0.5, -1)
    want = p @ v.double()
    got = _attend(q, k, v, 0.5).double()
    assert bool(((got - want).abs() <= R.HALF[dt] * want.abs() + 110 * 2.0 ** -24 * (p @ v.double().abs())).all())
