"""Pages of 4 bits on the GPU against plain torch on the CPU: cells, scales, bounds
and chosen pages bit for bit, attention within the bound of
paged_reference.attend_error (cells and scales are exact in bf16, so that nothing but
what that bound counts is rounded)."""
from __future__ import annotations

import math

import pytest
import torch

import four_bits_reference as F
import paged_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DIMS = [16, 32, 64, 128]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _same(a, b):
    a, b = a.cpu().float(), b.float()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())


def _agree(pages, pool):
    got = F.raw(pages)
    return all(torch.equal(got[m], pool[m]) for m in ("k", "v", "k_scale", "v_scale")) and \
        ("k_bounds" not in pool or _same(got["k_bounds"], pool["k_bounds"]))


WRITES = [
    # B, H, ps, starts, counts, n
    (1, 1, 16, [0], [1], 1),
    (3, 2, 16, [0, 15, 16], [1, 1, 1], 1),
    (2, 3, 32, [5, 31], [70, 0], 70),
    (4, 1, 64, [0, 1, 63, 200], [64, 65, 1, 130], 130),
    (2, 5, 256, [250, 0], [300, 257], 300),
    (2, 2, 128, [-3, 100], [9, 40], 50),
]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("D", DIMS)
def test_write_and_read(dt, D):
    from proteus_attention import read_kv_pages, write_kv_pages

    g = torch.Generator().manual_seed(D)
    for B, H, ps, starts, counts, n in WRITES:
        ends = [max(s + c, 0) for s, c in zip(starts, counts)]
        N = sum(-(-e // ps) for e in ends) + 2
        table = R.make_table(ends, ps, N, g)
        if B == 4:
            table[1, 0] = -1
            table[3, 1] = N + 7
        pool = F.make_pool(N, H, ps, D, g, bounds=True)
        wide = torch.randn(B, n, 3, H, D + (4 if B == 3 else 0), generator=g).to(dt)[..., :D]
        # sizes from nothing to the type's large ones, and zeros
        wide *= torch.exp2(torch.randint(-24, 13, (B, n, 3, H, 1), generator=g).float()).to(dt)
        k, v = wide[:, :, 1], wide[:, :, 2]
        if n > 1:
            k[0, 0, 0] = 0.0
        want = F.write(pool, k, v, table, starts, counts)
        pages = F.pages(pool, DEV)
        wd = wide.to(DEV) if B != 3 else torch.empty(B, n, 3, H, D + 4, dtype=dt, device=DEV)[..., :D].copy_(wide)
        args = (table.to(DEV), _i32(starts).to(DEV))
        write_kv_pages(pages, wd[:, :, 1], wd[:, :, 2], *args, counts=_i32(counts).to(DEV))
        assert _agree(pages, want), (B, ps)
        for out in (None, torch.bfloat16, torch.float32, torch.float16):
            kd, vd = read_kv_pages(pages, *args, _i32(counts).to(DEV), n, dtype=out)
            rk, rv = R.read(F.as_values(want), table, starts, counts, n, kd.dtype)
            assert kd.dtype == (out or torch.float32) and _same(kd, rk) and _same(vd, rv), (out, B, ps)


def test_every_border_between_cells():
    """Values on, just below and just above every tie, at both ends of the scales'
    range and where the largest of a group decides the scale."""
    from proteus_attention import new_kv_pages, read_kv_pages, write_kv_pages

    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0]
    near = torch.tensor([[x * (1 + d * 2.0 ** -23) for x in ties] for d in (-1, 0, 1)], dtype=torch.float64)
    rows = torch.cat([torch.cat([near[i], -near[i]]) for i in range(3)]).view(3, 32)
    rows = torch.cat([rows, rows.clamp(-6, 6)])
    sizes = torch.tensor([-140.0, -60.0, -21.0, -20.0, -19.0, 0.0, 14.0, 100.0, 124.0, 125.0], dtype=torch.float64)
    x = (rows * torch.exp2(sizes)[:, None, None]).flatten(0, 1).float()
    big = torch.finfo(torch.float32).max
    x = torch.cat([x, torch.full((1, 32), big), torch.full((1, 32), -0.0), torch.full((1, 32), 2.0 ** -149)])
    n = x.shape[0]
    pages = new_kv_pages(n // 16 + 1, 1, 16, 32, dtype=F.FP4, device=DEV)
    pool = F.raw(pages)
    table = torch.arange(n // 16 + 1, dtype=torch.int32)[None]
    k = x[None, :, None]
    want = F.write(pool, k, -k, table, [0], [n])
    zero = _i32([0]).to(DEV)
    write_kv_pages(pages, k.to(DEV), -k.to(DEV), table.to(DEV), zero)
    assert _agree(pages, want)
    kd, vd = read_kv_pages(pages, table.to(DEV), zero, None, n)
    assert bool(torch.isfinite(kd).all()) and torch.equal(kd, -vd)


@pytest.mark.parametrize("D", DIMS)
def test_groups_that_are_not_finite(D):
    from proteus_attention import paged_attention, read_kv_pages, write_kv_pages

    g = torch.Generator().manual_seed(1)
    pool = F.make_pool(2, 2, 16, D, g, bounds=True)
    k, v = torch.randn(1, 3, 2, D, generator=g), torch.randn(1, 3, 2, D, generator=g)
    k[0, 1, 0, 5], v[0, 2, 1, D - 1] = math.nan, -math.inf
    table, zero = _i32([[1, 0]]), _i32([0])
    want = F.write(pool, k, v, table, [0], [3])
    pages = F.pages(pool, DEV)
    write_kv_pages(pages, k.to(DEV), v.to(DEV), table.to(DEV), zero.to(DEV))
    assert _agree(pages, want)
    kd, vd = (x.cpu() for x in read_kv_pages(pages, table.to(DEV), zero.to(DEV), None, 3))
    w = F.group(D)
    assert torch.isnan(kd[0, 1, 0, :w]).all() and torch.isnan(vd[0, 2, 1, D - w:]).all()
    assert int(torch.isnan(kd).sum()) == w and int(torch.isnan(vd).sum()) == w
    # a key that is not a number makes its row so, a value its channels
    out = paged_attention(torch.randn(1, 4, D, generator=g).to(DEV), pages, table.to(DEV), _i32([3]).to(DEV)).cpu()
    assert torch.isnan(out[0, :2]).all() and torch.isnan(out[0, 2:, D - w:]).all()
    assert torch.isfinite(out[0, 2:, :D - w]).all()


def test_tokens_one_by_one_leave_what_one_call_leaves():
    from proteus_attention import new_kv_pages, write_kv_pages

    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(2, 37, 3, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    table = _i32([[4, 1, 2], [0, 5, 3]]).to(DEV)
    a, b = (new_kv_pages(6, 3, 16, 64, dtype=F.FP4, bounds=True, device=DEV) for _ in range(2))
    write_kv_pages(a, k, v, table, _i32([0, 3]).to(DEV))
    for i in range(37):
        write_kv_pages(b, k[:, i:i + 1], v[:, i:i + 1], table, _i32([i, 3 + i]).to(DEV))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


ATTENDS = [
    # H, G, ps, lengths
    (1, 1, 16, [1]),
    (2, 1, 16, [0, 1, 15, 16, 17, 33]),
    (3, 4, 64, [64, 65, 63, 300]),
    (1, 5, 32, [31, 1000]),
    (2, 16, 128, [129, 700]),
    (1, 20, 256, [513, 5]),
]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("D", DIMS)
def test_attention(dt, D):
    from proteus_attention import paged_attention

    g = torch.Generator().manual_seed(D + 1)
    for H, G, ps, lengths in ATTENDS:
        N = sum(-(-n // ps) for n in lengths) + 1
        pool, table = F.make_pool(N, H, ps, D, g), R.make_table(lengths, ps, N, g)
        q = torch.randn(len(lengths), H * G, D + 3, generator=g).to(dt)[..., :D]
        ref = R.attend(q, F.as_values(pool), table, lengths)
        qd = torch.empty(len(lengths), H * G, D + 3, dtype=dt, device=DEV)[..., :D].copy_(q)
        got = paged_attention(qd, F.pages(pool, DEV), table.to(DEV), _i32(lengths).to(DEV)).cpu()
        assert got.dtype == dt and R.attend_error(got, ref, dt, max(lengths)) <= 1, (H, G, ps)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("D", DIMS)
def test_nothing_of_what_is_not_seen(dt, D):
    """NaN scales in every slot that no sequence holds or sees, pages that are gone,
    windows that start inside a page, rows that see nothing, a stride between pages."""
    from proteus_attention import KVPages, paged_attention

    g = torch.Generator().manual_seed(3)
    for ps, H, G in ((32, 2, 3), (16, 1, 1), (128, 2, 2)):
        lengths = [5 * ps + 7, 3 * ps, 1, 0, 4 * ps + 1, 2 * ps]
        starts = [ps + 3, 0, 0, 0, 4 * ps + 1, -5]
        N = sum(-(-n // ps) for n in lengths) + 2
        table = R.make_table(lengths, ps, N, g)
        table[0, 3], table[1, 0], table[5, 1] = -1, N, -2 ** 31
        clean, pool = F.make_pool(N, H, ps, D, g), F.make_pool(N, H, ps, D, g, garbage=True)
        for b, (s, n) in enumerate(zip(starts, lengths)):
            for p in range(table.shape[1]):
                page, a, z = R.page_of(table, b, p, N), max(s - p * ps, 0), min(n - p * ps, ps)
                if page >= 0 and a < z:
                    for m in clean:
                        pool[m][page, :, a:z] = clean[m][page, :, a:z]
        q = torch.randn(len(lengths), H * G, D, generator=g).to(dt)
        ref = R.attend(q, F.as_values(clean), table, lengths, starts)
        side = torch.stack([pool["k"], pool["v"]], 1).to(DEV).view(F.FP4)
        pages = KVPages(side[:, 0], side[:, 1], pool["k_scale"].to(DEV).view(F.E8M0), pool["v_scale"].to(DEV).view(F.E8M0))
        got = paged_attention(q.to(DEV), pages, table.to(DEV), _i32(lengths).to(DEV), starts=_i32(starts).to(DEV)).cpu()
        assert R.attend_error(got, ref, dt, max(lengths)) <= 1, ps
        assert not got[3:5].any()


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_long_and_ragged(dt):
    from proteus_attention import paged_attention

    for lengths, H, G, ps, D in (([40001], 1, 2, 32, 64), ([0, 30011, 1, 5000, 17, 0, 999], 2, 1, 64, 32),
                                 ([7] * 300 + [9001], 1, 1, 16, 16), ([12345, 3], 2, 17, 16, 128)):
        g = torch.Generator().manual_seed(5)
        N = sum(-(-n // ps) for n in lengths)
        pool, table = F.make_pool(N, H, ps, D, g), R.make_table(lengths, ps, N, g, extra=40)
        q = (2.0 * torch.randn(len(lengths), H * G, D, generator=g)).to(dt)
        ref = R.attend(q, F.as_values(pool), table, lengths)
        args = (q.to(DEV), F.pages(pool, DEV), table.to(DEV), _i32(lengths).to(DEV))
        got = paged_attention(*args)
        assert R.attend_error(got.cpu(), ref, dt, max(lengths)) <= 1, (max(lengths), H)
        assert torch.equal(got, paged_attention(*args))


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("D", DIMS)
def test_selection_and_sparse_attention(dt, D):
    from proteus_attention import paged_attention, paged_sparse_attention, select_kv_pages

    g = torch.Generator().manual_seed(6)
    for H, G, ps, lengths, starts, count, first, last in (
            (2, 1, 16, [700, 0, 1, 16, 33], None, 6, 1, 1), (1, 16, 32, [1000, 40], [100, 39], 9, 2, 3),
            (2, 17, 16, [300, 90], None, 4, 0, 1), (3, 2, 64, [64, 3], [0, 7], 50, 1, 1),
            (1, 2, 16, [9000, 100], [33, 0], 70, 0, 0), (1, 1, 256, [700], None, 2, 1, 1)):
        N = sum(-(-n // ps) for n in lengths) + 1
        pool, table = F.make_pool(N, H, ps, D, g, bounds=True), R.make_table(lengths, ps, N, g)
        if H == 2:
            table[0, 3] = -1
        plain = F.as_values(pool)
        q = torch.randn(len(lengths), H * G, D, generator=g).to(dt)
        args = (q.to(DEV), F.pages(pool, DEV), table.to(DEV), _i32(lengths).to(DEV))
        kw = dict(starts=None if starts is None else _i32(starts).to(DEV))
        out, chosen = paged_sparse_attention(*args, count, first=first, last=last, scale=0.15, **kw)
        want = R.select(q, plain, table, lengths, starts, count, first, last)
        assert torch.equal(chosen.cpu(), want), (H, G, ps)
        assert torch.equal(select_kv_pages(*args, count, first=first, last=last, **kw).cpu(), want)
        ref = R.attend(q, plain, table, lengths, starts, want, scale=0.15)
        assert R.attend_error(out.cpu(), ref, dt, count * ps) <= 1, (H, G, ps)
        out = paged_attention(*args, selected=chosen, scale=0.15, **kw)
        assert R.attend_error(out.cpu(), ref, dt, count * ps) <= 1, (H, G, ps)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_prompt_then_tokens(dt):
    """Queries and keys turned by their positions, keys and values into pages of 4 bits,
    attention over all of the cache and over selected pages: a prompt, then tokens."""
    from proteus_attention import (apply_rotary, new_kv_pages, new_rotary_positions, paged_attention,
                                   paged_sparse_attention, write_kv_pages)

    g = torch.Generator().manual_seed(7)
    B, H, G, D, ps, n = 2, 2, 2, 64, 16, 150
    rotary = new_rotary_positions(D, scaling="yarn", factor=4.0, trained=64, device=DEV)
    pages = new_kv_pages(30, H, ps, D, dtype=F.FP4, bounds=True, device=DEV)
    pool = F.raw(pages)
    table = R.make_table([240, 200], ps, 30, g)
    lengths, counts = [0, 0], [150, 77]
    for step in range(4):
        q, k, v = (torch.randn(B, n, h, D, generator=g).to(dt).to(DEV) for h in (H * G, H, H))
        at = _i32(lengths).to(DEV)
        q, k = apply_rotary(q, k, at, rotary)
        write_kv_pages(pages, k, v, table.to(DEV), at, counts=_i32(counts).to(DEV))
        pool = F.write(pool, k.cpu(), v.cpu(), table, lengths, counts)
        assert _agree(pages, pool)
        lengths = [a + c for a, c in zip(lengths, counts)]
        q = torch.stack([q[b, c - 1] for b, c in enumerate(counts)])
        plain = F.as_values(pool)
        args = (q, pages, table.to(DEV), _i32(lengths).to(DEV))
        assert R.attend_error(paged_attention(*args).cpu(), R.attend(q.cpu(), plain, table, lengths), dt, 200) <= 1
        got, chosen = paged_sparse_attention(*args, 4)
        want = R.select(q.cpu(), plain, table, lengths, None, 4, 1, 1)
        assert torch.equal(chosen.cpu(), want)
        assert R.attend_error(got.cpu(), R.attend(q.cpu(), plain, table, lengths, None, want), dt, 64) <= 1
        n, counts = 1, [1, 1]


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes: rows of its last pages."""
    from proteus_attention import KVPages, paged_attention, read_kv_pages, write_kv_pages

    H, ps, D = 8, 256, 128
    N = (1 << 32) // (H * ps * D // 2) + 40
    k, v = (torch.empty(N, H, ps, D // 2, dtype=torch.uint8, device=DEV).view(F.FP4) for _ in range(2))
    scales = [torch.empty(N, H, ps, 4, dtype=torch.uint8, device=DEV).view(F.E8M0) for _ in range(2)]
    pages = KVPages(k, v, *scales, torch.empty(N, H, 2, D, dtype=torch.bfloat16, device=DEV))
    g = torch.Generator().manual_seed(10)
    table, zero = _i32([[N - 1, 3], [N - 20, N - 2]]), _i32([0, 0]).to(DEV)
    kn, vn = (torch.randn(2, 300, H, D, generator=g) for _ in range(2))
    write_kv_pages(pages, kn.to(DEV), vn.to(DEV), table.to(DEV), zero)
    rk, rv = (F.values(F.pack(c), s) for c, s in (F.quantise(kn), F.quantise(vn)))
    kd, vd = read_kv_pages(pages, table.to(DEV), zero, None, 300)
    assert torch.equal(kd.cpu(), rk) and torch.equal(vd.cpu(), rv)
    q = torch.randn(2, H, D, generator=g)
    out = paged_attention(q.to(DEV), pages, table.to(DEV), _i32([300, 300]).to(DEV))
    # the same rows as a small pool's
    small = {m: x.new_zeros(4, H, ps, D) for m, x in (("k", rk), ("v", rv))}
    for b in range(2):
        for m, x in (("k", rk), ("v", rv)):
            small[m][2 * b] = x[b, :ps].transpose(0, 1)
            small[m][2 * b + 1, :, :300 - ps] = x[b, ps:].transpose(0, 1)
    ref = R.attend(q, small, _i32([[0, 1], [2, 3]]), [300, 300])
    assert R.attend_error(out.cpu(), ref, torch.float32, 300) <= 1
