"""Key weights and evictions at the ends of what their calls allow, on the GPU against
plain torch on the CPU."""
from __future__ import annotations

import pytest
import torch

import four_bits_reference as F
import paged_reference as R
from test_gpu_key_weights import DEV, _bytes, _i32, _pages, _plain, _pool, _values, choose, holds, moved, weights

pytestmark = pytest.mark.gpu

# what sees nothing: at the length, behind it, and the last starts of 32 bits, from which
# a workgroup's 1,024 positions leave them
NOTHING = [0, 1, 2 ** 31 - 1, 2 ** 31 - 4, 2 ** 31 - 1020, 2 ** 31 - 1024, 2 ** 31 - 1025, 2 ** 30]


@pytest.mark.parametrize("pair", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.int8), (torch.float16, F.FP4)],
                         ids=R.pair_id)
@pytest.mark.parametrize("longest", [300, 4500])  # a workgroup a pair, and rows shared out
@pytest.mark.parametrize("G", [1, 4, 18])
def test_starts_that_see_nothing(pair, longest, G):
    """Beside rows that see keys: output rows of zeros, weights that keep their bits."""
    from proteus_attention import paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(G)
    H, D, ps = 2, 64, 16
    lengths = [longest, 40] + [min(longest, 90 + 7 * i) for i in range(len(NOTHING))] + [33, 33, 10 ** 9]
    starts = [3, -2 ** 31] + [n if n > 1 else lengths[2 + i] + n for i, n in enumerate(NOTHING)] + [32, 33, 2 ** 31 - 2]
    N = sum(-(-min(n, longest) // ps) for n in lengths) + 1
    table = R.make_table([min(n, longest) for n in lengths], ps, N, g)
    pool = _pool(cell, N, H, ps, D, g)
    q = torch.randn(len(lengths), H * G, D, generator=g).to(dt)
    ref = weights(q, _plain(cell, pool), table, lengths, starts)
    before = torch.rand(len(lengths), H, table.shape[1] * ps, generator=g)
    w, wide = before.to(DEV), torch.zeros(*before.shape[:2], before.shape[2] + 1, device=DEV)[..., 1:].copy_(before)
    args, kw = (q.to(DEV), _pages(cell, pool), table.to(DEV), _i32(lengths).to(DEV)), dict(starts=_i32(starts).to(DEV))
    out = paged_attention(*args, key_weights=w, **kw)
    assert torch.equal(out, paged_attention(*args, key_weights=wide, **kw)) and torch.equal(out, paged_attention(*args, **kw))
    blind = [b for b, (s, n) in enumerate(zip(starts, lengths)) if s >= min(n, table.shape[1] * ps)]
    assert len(blind) == len(NOTHING) + 2 and not out[blind].any() and bool(out[[0, 1, -3]].any(-1).all())
    assert torch.equal(w[blind].cpu(), before[blind]) and torch.equal(w, wide)
    assert holds(w.cpu(), before, ref, G, D, longest)


def test_eviction_from_no_pages_into_none():
    from proteus_attention import evict_kv_tokens, new_kv_pages

    pages = new_kv_pages(4, 2, 16, 32, bounds=True, device=DEV)
    none, w = torch.zeros(2, 0, dtype=torch.int32, device=DEV), torch.ones(2, 2, 40, device=DEV)
    kept, fresh = evict_kv_tokens(pages, w, none, _i32([5, 0]).to(DEV), 9, none)
    assert kept.shape == (2, 2, 9) and bool((kept == -1).all()) and fresh.shape == w.shape and not fresh.any()
    assert not any(t.any() for t in pages if t is not None)


def evicts(cell, pool, table, into, w, lengths, count, first, last, before=None):
    """evict_kv_tokens against choose() and moved(), bit for bit; NaN as NaN.  `before`: the
    device's weights, in a layout of their own."""
    from proteus_attention import evict_kv_tokens

    N, ps = pool["k"].shape[0], pool["k"].shape[2]
    B, _, T = w.shape
    have = torch.zeros(B, T, dtype=torch.bool)
    for b in range(B):
        for p in range(min(T, table.shape[1] * ps)):
            have[b, p] = R.page_of(table, b, p // ps, N) >= 0
    held = [min(max(int(n), 0), table.shape[1] * ps) for n in lengths]
    kept = choose(w, held, count, first, last, have)
    want, fresh = moved(_bytes(cell, pool), kept, w, table, into, _values(cell))
    pages = _pages(cell, pool)
    before = w.to(DEV) if before is None else before
    got, after = evict_kv_tokens(pages, before, table.to(DEV), _i32(lengths).to(DEV), count, into.to(DEV), first=first,
                                 last=last)
    assert torch.equal(got.cpu(), kept)
    assert torch.equal(after.cpu().view(torch.int32), fresh.view(torch.int32))  # NaN move with their bits
    assert torch.equal(before.cpu().view(torch.int32), w.view(torch.int32))
    for m in want:
        x, y = getattr(pages, m), want[m]
        x = x.view(torch.uint8).cpu() if y.dtype == torch.uint8 else x.cpu()
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num()), m
    return kept


@pytest.mark.parametrize("shape", [(2, 3, 16384), (2, 3, 16385), (1, 2, 1 << 20), (64, 2, 20001)], ids=str)
def test_weights_far_wider_than_the_table(shape):
    """What is behind the kept weights is zero, in one launch and in two."""
    B, H, T = shape
    g = torch.Generator().manual_seed(T)
    ps, D, count = 16, 16, 40
    lengths = [(90, 1000, 5)[b % 3] for b in range(B)]
    P = 64
    N = B * P + B * 3
    both = torch.randperm(N, generator=g).to(torch.int32)
    table, into = both[:B * P].view(B, P).clone(), both[B * P:].view(B, 3).clone()
    table[0, 1] = -1
    pool = _pool(torch.bfloat16, N, H, ps, D, g)
    w = torch.rand(B, H, T, generator=g) + 1.0
    evicts(torch.bfloat16, pool, table, into, w, lengths, count, 1, 3)
