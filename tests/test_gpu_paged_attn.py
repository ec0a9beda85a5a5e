"""Paged key-value cache and one-token attention on the GPU against plain
torch on the CPU: cells, scales, bounds and chosen pages bit for bit, attention
within the bound of paged_reference.attend_error."""
from __future__ import annotations

import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _pages(pool, dev=DEV):
    from proteus_attention import KVPages

    return KVPages(**{m: t.to(dev) for m, t in pool.items()})


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _same(a, b):
    """Bit for bit, NaN alike; a zero's sign in bounds is free."""
    a, b = a.cpu().float(), b.float()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())


# ---------------------------------------------------------------------------
# writing and reading
# ---------------------------------------------------------------------------

WRITES = [
    # B, H, ps, starts, counts, n
    (1, 1, 16, [0], [1], 1),
    (3, 2, 16, [0, 15, 16], [1, 1, 1], 1),
    (2, 3, 32, [5, 31], [70, 0], 70),
    (4, 1, 64, [0, 1, 63, 200], [64, 65, 1, 130], 130),
    (2, 5, 256, [250, 0], [300, 257], 300),
    (2, 2, 128, [-3, 100], [9, 40], 50),  # positions below zero; fewer than n
]


@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_write_and_read(pair, D):
    from proteus_attention import read_kv_pages, write_kv_pages

    dt, cell = pair
    g = torch.Generator().manual_seed(D)
    for B, H, ps, starts, counts, n in WRITES:
        ends = [max(s + c, 0) for s, c in zip(starts, counts)]
        N = sum(-(-e // ps) for e in ends) + 2
        table = R.make_table(ends, ps, N, g)
        if B == 4:
            table[1, 0] = -1  # a page that is gone
            table[3, 1] = N + 7  # and one that no pool has
        pool = R.make_pool(N, H, ps, D, cell, g, bounds=True)
        # slices of a projection's output, and rows that start off an 8-element line
        wide = torch.randn(B, n, 3, H, D + (4 if B == 3 else 0), generator=g).to(dt)[..., :D]
        k, v = wide[:, :, 1], wide[:, :, 2]
        if n > 1:
            k[0, 0, 0] = 0.0  # the scale's floor
        want = R.write(pool, k, v, table, _i32(starts), _i32(counts))
        pages = _pages(pool)
        wd = wide.to(DEV) if B != 3 else torch.empty(B, n, 3, H, D + 4, dtype=dt, device=DEV)[..., :D].copy_(wide)
        args = (table.to(DEV), _i32(starts).to(DEV))
        write_kv_pages(pages, wd[:, :, 1], wd[:, :, 2], *args, counts=_i32(counts).to(DEV))
        for m in want:
            assert _same(getattr(pages, m), want[m]), (m, B, ps)
        for out in (None, torch.bfloat16, torch.float32, torch.float16):
            kd, vd = read_kv_pages(pages, *args, _i32(counts).to(DEV), n, dtype=out)
            rk, rv = R.read(want, table, starts, counts, n, kd.dtype)
            assert _same(kd, rk) and _same(vd, rv), (out, B, ps)


@pytest.mark.parametrize("cell", [torch.int8, torch.float8_e4m3fn], ids=str)
def test_rows_that_are_not_finite(cell):
    from proteus_attention import read_kv_pages, write_kv_pages

    g = torch.Generator().manual_seed(1)
    pool = R.make_pool(2, 2, 16, 32, cell, g, bounds=True)
    k, v = torch.randn(1, 3, 2, 32, generator=g), torch.randn(1, 3, 2, 32, generator=g)
    k[0, 1, 0, 5], v[0, 2, 1, 31] = math.nan, -math.inf
    table, zero = _i32([[1, 0]]), _i32([0])
    want = R.write(pool, k, v, table, zero, _i32([3]))
    pages = _pages(pool)
    write_kv_pages(pages, k.to(DEV), v.to(DEV), table.to(DEV), zero.to(DEV))
    for m in want:
        assert _same(getattr(pages, m), want[m]), m
    kd, vd = read_kv_pages(pages, table.to(DEV), zero.to(DEV), None, 3)
    assert torch.isnan(kd[0, 1, 0]).all() and torch.isnan(vd[0, 2, 1]).all()
    assert torch.isfinite(kd[0, 1, 1]).all() and torch.isfinite(vd[0, 2, 0]).all()


def test_tokens_one_by_one_leave_what_one_call_leaves():
    from proteus_attention import new_kv_pages, write_kv_pages

    for dt, cell in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.int8)):
        g = torch.Generator().manual_seed(2)
        k, v = (torch.randn(2, 37, 3, 64, generator=g).to(dt).to(DEV) for _ in range(2))
        table = _i32([[4, 1, 2], [0, 5, 3]]).to(DEV)
        a, b = (new_kv_pages(6, 3, 16, 64, dtype=cell, bounds=True, device=DEV) for _ in range(2))
        write_kv_pages(a, k, v, table, _i32([0, 3]).to(DEV))
        for i in range(37):
            write_kv_pages(b, k[:, i:i + 1], v[:, i:i + 1], table, _i32([i, 3 + i]).to(DEV))
        for x, y in zip(a, b):
            # the second sequence's first page joins the zeros of the new pool in both
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

ATTENDS = [
    # H, G, ps, lengths
    (1, 1, 16, [1]),
    (2, 1, 16, [0, 1, 15, 16, 17, 33]),
    (3, 4, 64, [64, 65, 63, 300]),
    (1, 5, 32, [31, 1000]),
    (2, 16, 128, [129, 700]),
    (1, 20, 256, [513, 5]),  # more heads than a tile has rows
]


@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_attention(pair, D):
    from proteus_attention import paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(D + 1)
    for H, G, ps, lengths in ATTENDS:
        B = len(lengths)
        N = sum(-(-n // ps) for n in lengths) + 1
        pool = R.make_pool(N, H, ps, D, cell, g)
        table = R.make_table(lengths, ps, N, g)
        q = torch.randn(B, H * G, D + 3, generator=g).to(dt)[..., :D]
        ref = R.attend(q, pool, table, lengths)
        qd = torch.empty(B, H * G, D + 3, dtype=dt, device=DEV)[..., :D].copy_(q)
        got = paged_attention(qd, _pages(pool), table.to(DEV), _i32(lengths).to(DEV)).cpu()
        assert got.dtype == dt and R.attend_error(got, ref, dt, max(lengths)) <= 1, (H, G, ps)


@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
def test_nothing_of_what_is_not_seen(pair):
    """NaN and infinities in every slot that no sequence holds or sees, pages
    that are gone in the middle, windows that start inside a page, rows that see
    nothing; a pool with k and v side by side."""
    from proteus_attention import KVPages, paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(3)
    for D, ps, H, G in ((64, 32, 2, 3), (128, 16, 1, 1), (16, 128, 2, 2)):
        lengths = [5 * ps + 7, 3 * ps, 1, 0, 4 * ps + 1, 2 * ps]
        starts = [ps + 3, 0, 0, 0, 4 * ps + 1, -5]
        N = sum(-(-n // ps) for n in lengths) + 2
        table = R.make_table(lengths, ps, N, g)
        table[0, 3], table[1, 0], table[5, 1] = -1, N, -2 ** 31
        clean = R.make_pool(N, H, ps, D, cell, g)
        pool = R.make_pool(N, H, ps, D, cell, g, garbage=True)
        for b, (s, n) in enumerate(zip(starts, lengths)):
            for p in range(table.shape[1]):
                page = R.page_of(table, b, p, N)
                a, z = max(s - p * ps, 0), min(n - p * ps, ps)
                if page >= 0 and a < z:
                    for m in clean:
                        src = clean[m].view(torch.uint8) if clean[m].element_size() == 1 else clean[m]
                        dst = pool[m].view(torch.uint8) if pool[m].element_size() == 1 else pool[m]
                        dst[page, :, a:z] = src[page, :, a:z]
        q = torch.randn(len(lengths), H * G, D, generator=g).to(dt)
        ref = R.attend(q, clean, table, lengths, starts)
        side = torch.stack([pool["k"].view(torch.uint8), pool["v"].view(torch.uint8)], 1).to(DEV).view(cell)
        pages = KVPages(k=side[:, 0], v=side[:, 1],
                        **{m: t.to(DEV) for m, t in pool.items() if m not in ("k", "v")})
        got = paged_attention(q.to(DEV), pages, table.to(DEV), _i32(lengths).to(DEV), starts=_i32(starts).to(DEV))
        assert R.attend_error(got.cpu(), ref, dt, max(lengths)) <= 1, (D, ps)
        assert torch.equal(got[3:5].cpu(), torch.zeros_like(got[3:5].cpu()))


@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("ps", [16, 64, 256])
def test_listed_pages(pair, ps):
    from proteus_attention import paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(4)
    H, G, D, lengths = 2, 3, 64, [9 * ps + 5, 2 * ps, ps - 3, 0]
    N = sum(-(-n // ps) for n in lengths)
    pool, table = R.make_pool(N, H, ps, D, cell, g), R.make_table(lengths, ps, N, g)
    selected = _i32([[[0, 9, 4, -1, 4], [3, 2, 1, 8, 7]], [[1, 0, 2, 99, -7], [-1, -1, -1, -1, -1]],
                     [[0, 0, 0, 1, 2], [0, -1, -1, -1, -1]], [[0, 1, 2, 3, 4]] * 2])
    q = torch.randn(4, H * G, D, generator=g).to(dt)
    starts = [5, 0, 2, 0]
    for sel in (selected, selected[..., :1], selected[..., :0], selected.repeat(1, 1, 30)):
        ref = R.attend(q, pool, table, lengths, starts, sel, scale=0.2)
        got = paged_attention(q.to(DEV), _pages(pool), table.to(DEV), _i32(lengths).to(DEV),
                              starts=_i32(starts).to(DEV), selected=sel.to(DEV), scale=0.2)
        assert R.attend_error(got.cpu(), ref, dt, 5 * ps) <= 1, tuple(sel.shape)


@pytest.mark.parametrize("pair", [R.PAIRS[0], R.PAIRS[1], R.PAIRS[4], R.PAIRS[8]], ids=R.pair_id)
def test_long_and_ragged(pair):
    """Sequences from nothing to tens of thousands of tokens in one call, and
    one alone: lengths that end anywhere in a split."""
    from proteus_attention import paged_attention

    dt, cell = pair
    for lengths, H, G, ps, D in (([40001], 1, 2, 32, 64), ([0, 30011, 1, 5000, 17, 0, 999], 2, 1, 64, 32),
                                 ([7] * 300 + [9001], 1, 1, 16, 16), ([12345, 3], 2, 17, 16, 128)):
        g = torch.Generator().manual_seed(5)
        N = sum(-(-n // ps) for n in lengths)
        pool, table = R.make_pool(N, H, ps, D, cell, g), R.make_table(lengths, ps, N, g, extra=40)
        q = (2.0 * torch.randn(len(lengths), H * G, D, generator=g)).to(dt)
        ref = R.attend(q, pool, table, lengths)
        args = (q.to(DEV), _pages(pool), table.to(DEV), _i32(lengths).to(DEV))
        got = paged_attention(*args)
        assert R.attend_error(got.cpu(), ref, dt, max(lengths)) <= 1, (max(lengths), H)
        assert torch.equal(got, paged_attention(*args))  # the same bits every time


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("D", [16, 128])
def test_selection(pair, D):
    from proteus_attention import select_kv_pages

    dt, cell = pair
    g = torch.Generator().manual_seed(6)
    for H, G, ps, lengths, starts in ((1, 1, 16, [1, 160, 161, 0], None), (2, 4, 16, [4000, 900], [0, 333]),
                                      (3, 5, 64, [5000, 64, 640], [70, 64, 9]), (1, 17, 32, [1200], None),
                                      (1, 3, 16, [20011, 9000, 8193], [37, 0, 8192])):
        N = sum(-(-n // ps) for n in lengths) + 1
        pool = R.make_pool(N, H, ps, D, cell, g, bounds=True)
        table = R.make_table(lengths, ps, N, g)
        if len(lengths) == 2:
            table[0, 40] = -1
            pool["k_bounds"][table[0, 7].item(), 0, 0, 3] = math.nan  # a page whose bound is not a number
            pool["k_bounds"][table[0, 9].item(), 1] = pool["k_bounds"][table[0, 99].item(), 1]  # and a tie
        q = torch.randn(len(lengths), H * G, D, generator=g).to(dt)
        st = None if starts is None else _i32(starts).to(DEV)
        for count, first, last in ((1, 0, 1), (5, 1, 1), (9, 0, 0), (12, 3, 4), (400, 1, 1)):
            want = R.select(q, pool, table, lengths, starts, count, first, last)
            got = select_kv_pages(q.to(DEV), _pages(pool), table.to(DEV), _i32(lengths).to(DEV), count, first=first,
                                  last=last, starts=st).cpu()
            assert torch.equal(got, want), (H, ps, count)


def test_selection_of_equal_pages():
    """All pages alike: the lowest entries, whatever the number of pages."""
    from proteus_attention import KVPages, select_kv_pages

    for P in (1, 63, 511, 512, 513, 1021, 1022, 4094, 5000, 8190, 16381, 16382, 40000):
        z = torch.zeros(1, 1, 16, 16, device=DEV)
        pages = KVPages(k=z, v=z.clone(), k_bounds=torch.ones(1, 1, 2, 16, device=DEV))
        q = torch.randn(1, 2, 16, device=DEV)
        table = torch.zeros(1, P, dtype=torch.int32, device=DEV)
        got = select_kv_pages(q, pages, table, _i32([16 * P]).to(DEV), 700, first=0, last=1).cpu()[0, 0]
        n = min(P, 700)
        want = list(range(n - 1)) + [P - 1]
        assert got.tolist() == want + [-1] * (700 - n)


@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_sparse_attention(pair, D):
    """Rows that select and attend in one launch, in several, with more heads than
    a tile has rows, with more pages asked for than there are, and windows."""
    from proteus_attention import paged_sparse_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(14)
    for H, G, ps, lengths, starts, count, first, last in (
            (2, 1, 16, [700, 0, 1, 16, 33], None, 6, 1, 1), (1, 16, 32, [1000, 40], [100, 39], 9, 2, 3),
            (2, 17, 16, [300, 90], None, 4, 0, 1), (3, 2, 64, [64, 3], [0, 7], 50, 1, 1),
            (1, 2, 16, [9000, 100], [33, 0], 70, 0, 0), (1, 1, 256, [700], None, 2, 1, 1)):
        B = len(lengths)
        N = sum(-(-n // ps) for n in lengths) + 1
        pool = R.make_pool(N, H, ps, D, cell, g, bounds=True)
        table = R.make_table(lengths, ps, N, g)
        if H == 2:
            table[0, 3] = -1
        q = torch.randn(B, H * G, D, generator=g).to(dt)
        st = None if starts is None else _i32(starts).to(DEV)
        out, chosen = paged_sparse_attention(q.to(DEV), _pages(pool), table.to(DEV), _i32(lengths).to(DEV), count,
                                             first=first, last=last, starts=st, scale=0.15)
        want = R.select(q, pool, table, lengths, starts, count, first, last)
        assert torch.equal(chosen.cpu(), want), (H, G, ps)
        ref = R.attend(q, pool, table, lengths, starts, want, scale=0.15)
        assert R.attend_error(out.cpu(), ref, dt, count * ps) <= 1, (H, G, ps)


# ---------------------------------------------------------------------------
# as they are used together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
def test_prompt_then_tokens(pair):
    """Prompts of two lengths, then tokens one at a time: written, attended to
    over the whole cache and over selected pages."""
    from proteus_attention import new_kv_pages, paged_attention, paged_sparse_attention, write_kv_pages

    dt, cell = pair
    g = torch.Generator().manual_seed(7)
    B, H, G, D, ps, n = 2, 2, 2, 64, 16, 150
    pages = new_kv_pages(30, H, ps, D, dtype=cell, bounds=True, device=DEV)
    pool = {m: t.cpu().clone() for m, t in pages._asdict().items() if t is not None}
    table = R.make_table([240, 200], ps, 30, g)
    lengths, counts = [0, 0], [150, 77]
    for step in range(4):
        k, v = (torch.randn(B, n, H, D, generator=g).to(dt) for _ in range(2))
        write_kv_pages(pages, k.to(DEV), v.to(DEV), table.to(DEV), _i32(lengths).to(DEV), counts=_i32(counts).to(DEV))
        pool = R.write(pool, k, v, table, lengths, counts)
        lengths = [a + c for a, c in zip(lengths, counts)]
        q = torch.randn(B, H * G, D, generator=g).to(dt)
        args = (q.to(DEV), pages, table.to(DEV), _i32(lengths).to(DEV))
        assert R.attend_error(paged_attention(*args).cpu(), R.attend(q, pool, table, lengths), dt, 200) <= 1
        got, chosen = paged_sparse_attention(*args, 4)
        want = R.select(q, pool, table, lengths, None, 4, 1, 1)
        assert torch.equal(chosen.cpu(), want)
        assert R.attend_error(got.cpu(), R.attend(q, pool, table, lengths, None, want), dt, 64) <= 1
        n, counts = 1, [1, 1]


def test_captured_step():
    """One token's step in a graph, replayed over growing lengths between eager
    calls of the same step, against the eager results."""
    from proteus_attention import new_kv_pages, paged_attention, paged_sparse_attention, write_kv_pages

    g = torch.Generator().manual_seed(8)
    B, H, D, ps, P = 3, 2, 64, 16, 700
    pages = [new_kv_pages(B * P, H, ps, D, bounds=True, device=DEV) for _ in range(2)]
    table = torch.randperm(B * P, generator=g).view(B, P).to(torch.int32).to(DEV)
    prompt = torch.randn(2, B, 9000, H, D, generator=g).bfloat16().to(DEV)
    at = _i32([0, 0, 0]).to(DEV)
    for p in pages:
        write_kv_pages(p, prompt[0], prompt[1], table, at, counts=_i32([9000, 31, 500]).to(DEV))
    lengths = [_i32([9000, 31, 500]).to(DEV) for _ in range(2)]
    new = [torch.zeros(3, B, 1, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]

    def step(i):
        write_kv_pages(pages[i], new[i][0], new[i][1], table, lengths[i])
        lengths[i] += 1
        q = new[i][2, :, 0]
        return paged_attention(q, pages[i], table, lengths[i]), *paged_sparse_attention(q, pages[i], table, lengths[i], 6)

    tokens = torch.randn(5, 3, B, 1, H, D, generator=g).bfloat16().to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            new[i].copy_(tokens[0])
            step(i)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(0)
    for t in range(1, 5):
        for i in range(2):
            new[i].copy_(tokens[t])
        want = step(1)
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(held, want):
            assert torch.equal(a, b), t
        for a, b in zip(pages[0], pages[1]):
            assert a is None or torch.equal(a, b)


def test_two_streams_at_once():
    from proteus_attention import paged_attention

    g = torch.Generator().manual_seed(9)
    lengths, H, ps, D = [20000, 7], 2, 64, 64
    N = sum(-(-n // ps) for n in lengths)
    pool, table = R.make_pool(N, H, ps, D, torch.bfloat16, g), R.make_table(lengths, ps, N, g).to(DEV)
    pages, n = _pages(pool), _i32(lengths).to(DEV)
    qs = [torch.randn(2, 2 * H, D, generator=g).bfloat16().to(DEV) for _ in range(2)]
    want = [paged_attention(q, pages, table, n) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(qs[i], pages, table, n))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 cells: rows of its last pages."""
    from proteus_attention import KVPages, paged_sparse_attention, read_kv_pages, write_kv_pages

    H, ps, D = 8, 256, 128
    N = (1 << 32) // (H * ps * D) + 40
    k, v = (torch.empty(N, H, ps, D, dtype=torch.int8, device=DEV) for _ in range(2))
    scales = [torch.empty(N, H, ps, device=DEV) for _ in range(2)]
    pages = KVPages(k, v, *scales, torch.empty(N, H, 2, D, device=DEV))
    g = torch.Generator().manual_seed(10)
    table = _i32([[N - 1, 3], [N - 20, N - 2]])
    kn, vn = (torch.randn(2, 300, H, D, generator=g) for _ in range(2))
    zero = _i32([0, 0]).to(DEV)
    write_kv_pages(pages, kn.to(DEV), vn.to(DEV), table.to(DEV), zero)
    rk, rv = (R.values(*R.quantise(x, torch.int8)) for x in (kn, vn))
    kd, vd = read_kv_pages(pages, table.to(DEV), zero, None, 300)
    assert torch.equal(kd.cpu(), rk) and torch.equal(vd.cpu(), rv)
    q = torch.randn(2, H, D, generator=g)
    out, chosen = paged_sparse_attention(q.to(DEV), pages, table.to(DEV), _i32([300, 300]).to(DEV), 2)
    assert chosen.cpu().tolist() == [[[0, 1]] * H] * 2
    s = torch.einsum("bhd,bthd->bht", q.double(), rk.double()) / math.sqrt(D)
    want = torch.einsum("bht,bthd->bhd", torch.softmax(s, -1), rv.double())
    # attend_error's bound with sum p |v| <= 5 and sum |q k| scale <= 60
    assert float((out.cpu().double() - want).norm(dim=-1).max()) <= 4 * 2.0 ** -24 * ((math.sqrt(D) + 3) * 60 + 22) * 5 * math.sqrt(D)


def test_layouts_and_empty_calls():
    """Tables and lengths that are slices, keys and queries that are expanded or
    transposed; calls with nothing to do."""
    from proteus_attention import (new_kv_pages, paged_attention, paged_sparse_attention, read_kv_pages,
                                   select_kv_pages, write_kv_pages)

    g = torch.Generator().manual_seed(12)
    B, H, D, ps = 3, 2, 32, 16
    pages = new_kv_pages(12, H, ps, D, dtype=torch.float32, bounds=True, device=DEV)
    pool = {m: t.cpu().clone() for m, t in pages._asdict().items() if t is not None}
    table = torch.randperm(12, generator=g).view(B, 4).to(torch.int32)
    lengths = [50, 17, 1]
    one = torch.randn(1, 50, 1, D, generator=g)
    k = one.expand(B, 50, H, D)  # every sequence and head the same
    v = torch.randn(B, H, D, 50, generator=g)
    want = R.write(pool, k, v.permute(0, 3, 1, 2), table, [0] * B, lengths)
    wide = torch.zeros(B, 3, dtype=torch.int32)
    wide[:, 1] = _i32(lengths)
    n = wide.to(DEV)[:, 1]
    columns = table.t().contiguous().to(DEV).t()
    write_kv_pages(pages, one.to(DEV).expand(B, 50, H, D), v.to(DEV).permute(0, 3, 1, 2), columns,
                   torch.zeros_like(n), counts=n)
    for m in want:
        assert _same(getattr(pages, m), want[m]), m
    q = torch.randn(1, D, generator=g).expand(B, 2 * H, D)
    qd = q[:1, :1].to(DEV).expand(B, 2 * H, D)
    ref = R.attend(q, want, table, lengths)
    assert R.attend_error(paged_attention(qd, pages, columns, n).cpu(), ref, torch.float32, 50) <= 1
    got, chosen = paged_sparse_attention(qd.transpose(1, 2).contiguous().transpose(1, 2), pages, columns, n, 3)
    sel = R.select(q, want, table, lengths, None, 3, 1, 1)
    assert torch.equal(chosen.cpu(), sel)
    assert R.attend_error(got.cpu(), R.attend(q, want, table, lengths, None, sel), torch.float32, 48) <= 1

    # no sequences, no tokens, no table
    none, t0, l0 = qd[:0], columns[:0], n[:0]
    assert paged_attention(none, pages, t0, l0).shape == (0, 2 * H, D)
    assert select_kv_pages(none, pages, t0, l0, 2).shape == (0, H, 2)
    assert read_kv_pages(pages, t0, l0, None, 5)[0].shape == (0, 5, H, D)
    assert read_kv_pages(pages, columns, n, None, 0)[0].shape == (B, 0, H, D)
    kd = one.to(DEV).expand(B, 50, H, D)
    write_kv_pages(pages, kd[:0], kd[:0], t0, l0)
    write_kv_pages(pages, kd[:, :0], kd[:, :0], columns, n)
    write_kv_pages(pages, kd, kd, columns[:, :0], n)
    for m in want:
        assert _same(getattr(pages, m), want[m]), m
    p0 = columns[:, :0]
    assert not paged_attention(qd, pages, p0, n).any()
    out, chosen = paged_sparse_attention(qd, pages, p0, n, 2)
    assert not out.any() and bool((chosen == -1).all())
    assert not any(x.any() for x in read_kv_pages(pages, p0, n, None, 7))


@pytest.mark.parametrize("ps", [16, 256])
def test_wide_tables(ps):
    """Tables far wider than the sequences: more pages than a run of tiles looks
    up at once, most of them gone."""
    from proteus_attention import paged_attention, paged_sparse_attention

    g = torch.Generator().manual_seed(13)
    H, G, D, P = 2, 2, 64, 1500
    lengths = [P * ps, (P - 3) * ps + 5]
    pool = R.make_pool(9, H, ps, D, torch.bfloat16, g, bounds=True)
    table = torch.full((2, P), -1, dtype=torch.int32)
    for b in range(2):
        at = torch.randperm(P, generator=g)[:9]
        table[b, at] = torch.randperm(9, generator=g).to(torch.int32)
        table[b, P - 1 - 3 * b] = b
    q = torch.randn(2, H * G, D, generator=g).bfloat16()
    args = (q.to(DEV), _pages(pool), table.to(DEV), _i32(lengths).to(DEV))
    ref = R.attend(q, pool, table, lengths)
    assert R.attend_error(paged_attention(*args).cpu(), ref, torch.bfloat16, 10 * ps) <= 1
    out, chosen = paged_sparse_attention(*args, 12, first=0, last=1)
    want = R.select(q, pool, table, lengths, None, 12, 0, 1)
    assert torch.equal(chosen.cpu(), want)
    assert R.attend_error(out.cpu(), ref, torch.bfloat16, 10 * ps) <= 1
