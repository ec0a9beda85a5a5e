"""Key weights and evictions at the ends of what their calls allow, on the GPU against
plain torch on the CPU."""
from __future__ import annotations

import math

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


def _odd_rows(w):
    """w on the device, rows off a 16-byte line and heads apart by a stride of their own."""
    B, H, T = w.shape
    return torch.zeros(H, B, T + 2, device=DEV).transpose(0, 1)[..., 1:T + 1].copy_(w)


@pytest.mark.parametrize("cell", [torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn, F.FP4], ids=str)
@pytest.mark.parametrize("kind", ["one launch", "two", "bounds"])
@pytest.mark.parametrize("more", [5, -7, 0])
def test_weights_that_the_table_does_not_fit(cell, kind, more):
    """Weights of more positions than the table has, and of fewer, with lengths beyond
    them: what has no weight is not kept, and `last` counts from the last that has one."""
    g = torch.Generator().manual_seed(17)
    ps, D, H = 16, 32, 2
    count = 70 if kind != "two" else 1100
    lengths = [10 ** 9, 200, 37] if kind != "two" else [10 ** 9, 1500, 300]
    P = 25 if kind != "two" else 110
    pages = -(-count // ps)
    N = 3 * (P + pages)
    both = torch.randperm(N, generator=g).to(torch.int32)
    table, into = both[:3 * P].view(3, P).clone(), both[3 * P:].view(3, pages).clone()
    table[0, 2], table[1, P - 1], table[2, 1], into[1, 1] = -1, -1, N, -1
    pool = _pool(cell, N, H, ps, D, g, bounds=kind == "bounds")
    T = P * ps + more
    w = torch.rand(3, H, T, generator=g)
    w[:, :, 3::7] = 0.25
    w[0, 0, 40:60], w[1, 1, ::3], w[0, 1, -1], w[2] = math.nan, math.nan, math.inf, -w[2]
    for last in (0, 9):
        for before in (None, _odd_rows(w)):
            kept = evicts(cell, pool, table, into, w, lengths, count, 2, last, before)
            assert int(kept.max()) < min(T, P * ps)
            if last and more < 0:  # the last of the clamped length
                assert kept[0, 0, -1] == T - 1 and (kept[0, 0, -last:] >= T - last).all()


@pytest.mark.parametrize("more", [0, 5, -7])
def test_long_weights_that_the_table_does_not_fit(more):
    """Rows that are cut in slices, with pages that are gone."""
    g = torch.Generator().manual_seed(23)
    ps, D, H, P, count = 256, 16, 2, 275, 700
    pages = 3
    N = P + pages + 1
    both = torch.randperm(N, generator=g).to(torch.int32)
    table, into = both[:P].view(1, P).clone(), both[P:P + pages].view(1, pages)
    table[0, 40], table[0, 3] = -1, N
    pool = _pool(torch.bfloat16, N, H, ps, D, g, bounds=True)
    T = P * ps + more
    w = torch.rand(1, H, T, generator=g)
    w[0, 0, 9000:9500], w[0, 1, ::2], w[0, 0, 70001] = math.nan, 0.75, -1.0
    for before in (None, _odd_rows(w)):
        evicts(torch.bfloat16, pool, table, into, w, [2 ** 31 - 1], count, 4, 11, before)


@pytest.mark.parametrize("cell", [torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn, F.FP4], ids=str)
def test_keys_that_are_not_numbers_move_with_their_bounds(cell):
    g = torch.Generator().manual_seed(29)
    ps, D, H, N = 16, 64, 2, 8
    pool = _pool(cell, N, H, ps, D, g, bounds=True)
    table, into = _i32([[3, 0, 6]]), _i32([[1, 5]])
    if cell == F.FP4:
        pool["k_scale"][3, 0, 2, 1] = pool["v_scale"][6, 1, 3, 0] = 255
    elif cell in R.TOP:
        pool["k_scale"][3, 0, 2] = pool["v_scale"][6, 1, 3] = math.nan
    else:
        pool["k"][3, 0, 2, 7], pool["v"][6, 1, 3, 0], pool["k"][6, 0, 1, 9] = math.nan, math.nan, -math.inf
    w = torch.rand(1, H, 3 * ps, generator=g)
    w[0, 0, 2], w[0, 0, 2 * ps + 1] = 9.0, 8.0  # kept, in the first fresh page and the second
    kept = evicts(cell, pool, table, into, w, [40], 20, 0, 3)
    assert 2 in kept[0, 0].tolist()


@pytest.mark.parametrize("cell", [torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn, F.FP4], ids=str)
@pytest.mark.parametrize("bounds", [False, True])
def test_pools_and_tables_with_strides(cell, bounds):
    """k and v side by side in one tensor, tables that are columns of a wider one: the bits
    of dense ones, and nothing else written."""
    from proteus_attention import evict_kv_tokens, paged_attention

    g = torch.Generator().manual_seed(31)
    ps, D, H, N, count = 16, 32, 2, 40, 37
    pool = _pool(cell, N, H, ps, D, g, bounds=bounds)
    both = torch.randperm(N, generator=g).to(torch.int32).view(2, 20).to(DEV)
    table, into, lengths = both[:, 2:14], both[:, 15:18], _i32([190, 77]).to(DEV)
    q = torch.randn(2, 3 * H, D, generator=g).to(torch.bfloat16 if cell in (torch.int8, torch.float8_e4m3fn, F.FP4) else cell)
    dense, apart = _pages(cell, pool), _pages(cell, pool)
    byte = torch.uint8 if cell == F.FP4 else cell
    wide = torch.stack([apart.k.view(byte).view(torch.uint8), torch.full_like(apart.k.view(byte).view(torch.uint8), 99),
                        apart.v.view(byte).view(torch.uint8)], 1).contiguous()
    apart = apart._replace(k=wide[:, 0].view(byte).view(cell), v=wide[:, 2].view(byte).view(cell))
    assert apart.k.stride(0) == 3 * dense.k.stride(0)
    got = []
    for pages, t, into_ in ((dense, table.contiguous(), into.contiguous()), (apart, table, into)):
        w = torch.zeros(2, H, 12 * ps, device=DEV)
        out = paged_attention(q.to(DEV), pages, t, lengths, key_weights=w)
        got.append([out, w, *evict_kv_tokens(pages, w, t, lengths, count, into_, last=5)])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and bool((got[0][2] >= 0).all())
    for a, b in zip(dense, apart):
        if a is not None:
            a, b = (x.view(torch.uint8) if x.dtype in (F.FP4, F.E8M0) else x for x in (a, b))
            assert torch.equal(a.cpu(), b.cpu())
    assert bool((wide[:, 1] == 99).all())


@pytest.mark.parametrize("pair", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, F.FP4)], ids=R.pair_id)
@pytest.mark.parametrize("G", [2, 17])
def test_weights_of_many_sequences(pair, G):
    """More sequences than a workgroup has threads, rows of a key to rows shared out."""
    from proteus_attention import paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(37)
    B, H, D, ps, N, T = 600, 1, 32, 16, 320, 4096
    lengths = [int(n) for n in torch.exp(torch.rand(B, generator=g) * math.log(300)).int()]
    lengths[7], lengths[300], lengths[599], lengths[11] = T, T - 1, 3000, 0
    table = torch.randint(0, N, (B, T // ps), generator=g, dtype=torch.int32)
    pool = _pool(cell, N, H, ps, D, g)
    q = torch.randn(B, H * G, D, generator=g).to(dt)
    before = torch.rand(B, H, T, generator=g)
    w = before.to(DEV)
    args = (q.to(DEV), _pages(cell, pool), table.to(DEV), _i32(lengths).to(DEV))
    assert torch.equal(paged_attention(*args, key_weights=w), paged_attention(*args))
    assert holds(w.cpu(), before, weights(q, _plain(cell, pool), table, lengths), G, D, T)


@pytest.mark.parametrize("lengths", [[200, 90], [6000, 90]], ids=str)
def test_scores_of_plus_infinity(lengths):
    """One in a row of a group's: its output and the weights of the keys it sees are NaN,
    wherever the row is cut; the other key-value head's are as they were."""
    from proteus_attention import KVPages, paged_attention

    g = torch.Generator().manual_seed(41)
    ps, D, H, N = 16, 32, 2, sum(-(-n // 16) for n in lengths) + 1
    k, v = (torch.randn(N, H, ps, D, generator=g) for _ in range(2))
    table = R.make_table(lengths, ps, N, g)
    k[int(table[0, 5]), 1, 3, 2] = math.inf
    q = torch.rand(2, 2 * H, D, generator=g) + 0.5
    w, clean = (torch.zeros(2, H, table.shape[1] * ps, device=DEV) for _ in range(2))
    rest = (table.to(DEV), _i32(lengths).to(DEV))
    out = paged_attention(q.to(DEV), KVPages(k.to(DEV), v.to(DEV)), *rest, key_weights=w)
    same = paged_attention(q.to(DEV), KVPages(k.nan_to_num(posinf=0.0).to(DEV), v.to(DEV)), *rest, key_weights=clean)
    assert out[0, 2:].isnan().all() and w[0, 1, :lengths[0]].isnan().all() and not w[0, 1, lengths[0]:].any()
    assert torch.equal(out[0, :2], same[0, :2]) and torch.equal(out[1], same[1])
    assert torch.equal(w[0, 0], clean[0, 0]) and torch.equal(w[1], clean[1])


def test_more_kept_than_there_are():
    g = torch.Generator().manual_seed(43)
    for count, bounds in ((900, False), (1500, False), (900, True)):
        pool = _pool(torch.bfloat16, 120, 2, 16, 32, g, bounds=bounds)
        table, into = _i32([[3, 1, 2]]), torch.arange(10, 10 + -(-count // 16), dtype=torch.int32)[None]
        evicts(torch.bfloat16, pool, table, into, torch.rand(1, 2, 48, generator=g), [41], count, 300, 500)
