"""Weights that attention gives to keys, and eviction by them, on the GPU against plain
torch on the CPU: choices, moved cells, scales, bounds and weights bit for bit."""
from __future__ import annotations

import math

import pytest
import torch

import four_bits_reference as F
import paged_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
PAIRS = R.PAIRS + [(t, F.FP4) for t in TYPES]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _pool(cell, *args, **kw):
    if cell == F.FP4:
        return F.make_pool(*args, **kw)
    N, H, ps, D, g = args
    return R.make_pool(N, H, ps, D, cell, g, **kw)


def _pages(cell, pool):
    from proteus_attention import KVPages

    return F.pages(pool, DEV) if cell == F.FP4 else KVPages(**{m: t.to(DEV) for m, t in pool.items()})


def _plain(cell, pool):
    return F.as_values(pool) if cell == F.FP4 else pool


def weights(q, pool, table, lengths, starts=None, scale=None):
    """(B, H, P * ps) in 64 bits: the softmax weights of every position, summed over the
    query heads of its head; zero where none sees it.  With it, for each head, the largest
    score's magnitude sum_d |q_d k_d| * scale."""
    N, H, ps, D = pool["k"].shape
    B, G, P = q.shape[0], q.shape[1] // H, table.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    k = pool["k"].double()
    if "k_scale" in pool:
        k = k * pool["k_scale"].double()[..., None]
    out, most = torch.zeros(B, H, P * ps, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        length = min(max(int(lengths[b]), 0), P * ps)
        start = max(int(starts[b]), 0) if starts is not None else 0
        pos = torch.tensor([p for p in range(start, length) if R.page_of(table, b, p // ps, N) >= 0], dtype=torch.long)
        if not len(pos):
            continue
        ids = table[b].long()[pos // ps]
        for h in range(H):
            x, rows = q[b, h * G:h * G + G].double(), k[ids, h, pos % ps]
            out[b, h, pos] = torch.softmax(x @ rows.T * scale, -1).sum(0)
            most[b, h] = (x.abs() @ rows.abs().T * scale).max()
    return out, most


def holds(got, before, ref, G, D, n):
    """Bound of a position's sum: each weight is off by the roundings of its score,
    (sqrt(D) + 3) * 2^-24 of sum |q k| scale, four times over for the largest of many, of
    the exponential, the sum over n keys (a random walk) and the quotient, relatively; G of
    them are added in f32 to what was there."""
    want, most = ref
    step = 2.0 ** -24
    rel = 4 * step * ((math.sqrt(D) + 3) * most[..., None] + math.sqrt(max(n, 1)) + 4)
    T = want.shape[2]
    total = want + before[..., :T].double()
    bound = rel * want + (G + 1) * step * (want + before[..., :T].double().abs())
    off = (got[..., :T].double() - total).abs()
    seen = want > 0
    return bool((off <= bound)[seen].all()) and torch.equal(got[..., :T][~seen], before[..., :T][~seen]) and \
        torch.equal(got[..., T:], before[..., T:])


ATTENDS = [
    # H, G, ps, lengths
    (1, 1, 16, [1]),
    (2, 1, 16, [0, 1, 15, 16, 17, 33]),
    (3, 4, 64, [64, 65, 63, 300]),
    (1, 5, 32, [31, 1000]),
    (2, 16, 128, [129, 700]),
    (1, 20, 256, [513, 5]),  # more heads than a tile has rows, one workgroup a pair
    (1, 33, 16, [4000, 70]),  # the same, shared out
    (2, 8, 16, [9001, 0, 2500]),
]


@pytest.mark.parametrize("pair", PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_weights(pair, D):
    from proteus_attention import paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(D)
    for H, G, ps, lengths in ATTENDS:
        B = len(lengths)
        N = sum(-(-n // ps) for n in lengths) + 1
        pool, table = _pool(cell, N, H, ps, D, g), R.make_table(lengths, ps, N, g)
        plain = _plain(cell, pool)
        q = torch.randn(B, H * G, D, generator=g).to(dt)
        before = torch.rand(B, H, table.shape[1] * ps + 5, generator=g)
        w = before.to(DEV)
        args = (q.to(DEV), _pages(cell, pool), table.to(DEV), _i32(lengths).to(DEV))
        got = paged_attention(*args, key_weights=w)
        assert torch.equal(got, paged_attention(*args)), (H, G, ps)  # the output's bits are those without
        assert holds(w.cpu(), before, weights(q, plain, table, lengths), G, D, max(lengths)), (H, G, ps)
        again = before.to(DEV)
        paged_attention(*args, key_weights=again)
        assert torch.equal(again, w)


@pytest.mark.parametrize("pair", PAIRS, ids=R.pair_id)
def test_windows_and_pages_that_are_gone(pair):
    """Weights in rows of their own layout; what is not seen keeps its bits, NaN too, and
    what stands in the pool there has no effect."""
    from proteus_attention import paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(3)
    for D, ps, H, G in ((64, 32, 2, 3), (128, 16, 1, 1), (16, 128, 2, 2), (32, 16, 2, 17)):
        lengths = [5 * ps + 7, 3 * ps, 1, 0, 4 * ps + 1, 2 * ps, 10 ** 6]
        starts = [ps + 3, 0, 0, 0, 4 * ps + 1, -5, 2 * ps + 9]
        N = 30
        table = R.make_table([min(n, 5 * ps) for n in lengths], ps, N, g)
        table[0, 3], table[1, 0], table[5, 1] = -1, N, -2 ** 31
        pool = _pool(cell, N, H, ps, D, g)
        plain = _plain(cell, pool)
        q = torch.randn(len(lengths), H * G, D, generator=g).to(dt)
        ref = weights(q, plain, table, lengths, starts, scale=0.2)
        T = table.shape[1] * ps
        before = torch.rand(len(lengths), H, T, generator=g)
        before = before.masked_fill((ref[0] == 0) & (torch.rand(before.shape, generator=g) < 0.3), math.nan)
        args = (q.to(DEV), _pages(cell, pool), table.to(DEV), _i32(lengths).to(DEV))
        kw = dict(starts=_i32(starts).to(DEV), scale=0.2)
        rows = before.to(DEV)
        odd = torch.zeros(len(lengths), H, T + 1, device=DEV)[..., 1:].copy_(before)
        heads = torch.zeros(H, len(lengths), T + 4, device=DEV).transpose(0, 1)[..., :T].copy_(before)
        for w in (rows, odd, heads):
            paged_attention(*args, key_weights=w, **kw)
            seen = ref[0] > 0
            got = w.cpu()
            assert holds(got.nan_to_num(7.0), before.nan_to_num(7.0), ref, G, D, max(min(n, T) for n in lengths)), (D, ps)
            assert torch.equal(got, rows.cpu()) or torch.equal(got.nan_to_num(7.0), rows.cpu().nan_to_num(7.0))
            assert bool(seen.any())


@pytest.mark.parametrize("pair", [PAIRS[0], PAIRS[1], PAIRS[4], PAIRS[-1]], ids=R.pair_id)
def test_windows_of_rows_that_are_shared_out(pair):
    """Rows cut over many workgroups beside rows that see nothing: windows that start at,
    behind and next to their ends, a row of one key, sequences without tokens."""
    from proteus_attention import paged_attention

    dt, cell = pair
    g = torch.Generator().manual_seed(21)
    for D, ps, H, G in ((64, 16, 1, 4), (128, 64, 2, 1), (32, 16, 1, 18)):
        lengths = [9001, 4097, 9, 0, 4098, 5, 2050, 3]
        starts = [103, 4097, 10, 3, 4097, 7, 2047, -9]
        N = sum(-(-n // ps) for n in lengths) + 1
        table = R.make_table(lengths, ps, N, g)
        table[0, 7] = -1
        pool = _pool(cell, N, H, ps, D, g)
        q = torch.randn(len(lengths), H * G, D, generator=g).to(dt)
        ref = weights(q, _plain(cell, pool), table, lengths, starts)
        before = torch.rand(len(lengths), H, table.shape[1] * ps, generator=g)
        w = before.to(DEV)
        args = (q.to(DEV), _pages(cell, pool), table.to(DEV), _i32(lengths).to(DEV))
        out = paged_attention(*args, starts=_i32(starts).to(DEV), key_weights=w)
        assert torch.equal(out, paged_attention(*args, starts=_i32(starts).to(DEV)))
        assert holds(w.cpu(), before, ref, G, D, 9001), (D, ps)
        assert not out[[1, 2, 3, 5]].any()


def test_rows_without_a_weight_and_rows_that_are_not_numbers():
    """Scores of -inf alone leave nothing; a NaN among a row's scores makes its weights NaN,
    in its own head alone."""
    from proteus_attention import KVPages, paged_attention

    k = torch.zeros(2, 2, 16, 32)
    k[0, 0] = -math.inf
    k[1, 1, 3, 0] = math.nan
    pages = KVPages(k.to(DEV), torch.ones(2, 2, 16, 32, device=DEV))
    q = torch.ones(2, 2, 32)
    w = torch.zeros(2, 2, 16, device=DEV)
    out = paged_attention(q.to(DEV), pages, _i32([[0], [1]]).to(DEV), _i32([16, 16]).to(DEV), key_weights=w).cpu()
    w = w.cpu()
    assert not out[0, 0].any() and not w[0, 0].any()
    assert torch.equal(w[0, 1], torch.full((16,), 1 / 16)) and torch.equal(w[1, 0], torch.full((16,), 1 / 16))
    assert torch.isnan(out[1, 1]).all() and torch.isnan(w[1, 1]).all()


def test_no_sequences_no_table():
    from proteus_attention import evict_kv_tokens, new_kv_pages, paged_attention, select_kv_tokens

    pages = new_kv_pages(4, 2, 16, 32, bounds=True, device=DEV)
    before = [t.clone() for t in pages if t is not None]
    q, none = torch.randn(2, 4, 32, device=DEV).bfloat16(), torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    n, w = _i32([5, 0]).to(DEV), torch.ones(2, 2, 32, device=DEV)
    assert not paged_attention(q, pages, none, n, key_weights=w).any() and bool((w == 1).all())
    assert paged_attention(q[:0], pages, none[:0], n[:0], key_weights=w[:0]).shape == (0, 4, 32)
    into = _i32([[0], [1]]).to(DEV)
    kept, fresh = evict_kv_tokens(pages, w, none, n, 9, into)
    assert bool((kept == -1).all()) and not fresh.any() and kept.shape == (2, 2, 9)
    kept, fresh = evict_kv_tokens(pages, w[..., :0], into, n, 9, torch.flip(into, [0]))
    assert bool((kept == -1).all()) and fresh.shape == (2, 2, 0)
    assert evict_kv_tokens(pages, w[:0], none[:0], n[:0], 9, into[:0])[0].shape == (0, 2, 9)
    assert select_kv_tokens(w[:0], n[:0], 3).shape == (0, 2, 3)
    assert bool((select_kv_tokens(w[..., :0], n, 3) == -1).all())
    assert all(torch.equal(a, b) for a, b in zip(before, [t for t in pages if t is not None]))


# ---------------------------------------------------------------------------
# choice and move
# ---------------------------------------------------------------------------

def choose(w, lengths, count, first, last, have=None):
    """(B, H, count); have (B, T): positions that have a page."""
    B, H, T = w.shape
    kept = torch.full((B, H, count), -1, dtype=torch.int32)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), T)
        for h in range(H):
            ok = [True] * n if have is None else have[b, :n].tolist()
            rank = sorted((not (i < first or i >= n - last), x != x, 0.0 if x != x else -x, i)
                          for i, x in enumerate(w[b, h, :n].tolist()) if ok[i])
            take = sorted(i for *_, i in rank[:count])
            kept[b, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
    return kept


@pytest.mark.parametrize("T", [1, 7, 64, 1023, 1024, 1025, 4096, 5000, 16384, 16385, 40003, 65536, 65537, 140001])
def test_select_tokens(T):
    from proteus_attention import select_kv_tokens

    g = torch.Generator().manual_seed(T)
    w = torch.exp(3 * torch.randn(3, 2, T, generator=g))
    w[1] = torch.randint(0, 4, (2, T), generator=g).float()  # many ties
    w[1, 1, ::3] = -0.0
    if T > 20:
        w[0, 0, 5], w[0, 0, 9], w[0, 1, 11], w[0, 1, 12] = math.nan, math.inf, -math.inf, -3.0
        w[2, 0, ::2] = math.nan
    lengths = [T, T - T // 5, T // 3]
    wide = torch.zeros(2, 3, T + 1, device=DEV).transpose(0, 1)[..., 1:].copy_(w)
    for count, first, last in ((1, 0, 1), (1, 0, 0), (T // 2 + 2, 1, 1), (max(T // 7, 8), 3, 4), (T + 3, 1, 1)):
        want = choose(w, lengths, count, first, last)
        got = select_kv_tokens(w.to(DEV), _i32(lengths).to(DEV), count, first=first, last=last)
        assert torch.equal(got.cpu(), want), (count, first, last)
        assert torch.equal(select_kv_tokens(wide, _i32(lengths).to(DEV), count, first=first, last=last), got)
    odd = w.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)  # positions apart
    assert torch.equal(select_kv_tokens(odd, _i32([-5, 10 ** 9, 0]).to(DEV), 5).cpu(), choose(w, [0, T, 0], 5, 1, 1))


def choose_long(w, lengths, count, first, last):
    """choose() of whole rows, by a stable sort of their bits' order."""
    B, H, T = w.shape
    u = (w + 0.0).view(torch.int32).long()
    key = torch.where(w != w, -2 ** 40, torch.where(u < 0, -1 - (u & 0x7fffffff), u))
    kept = torch.full((B, H, count), -1, dtype=torch.int32)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), T)
        row = key[b, :, :n].clone()
        row[:, :first] = row[:, max(n - last, 0):] = 2 ** 40
        take = row.sort(dim=1, descending=True, stable=True).indices[:, :count].sort(1).values
        kept[b, :, :take.shape[1]] = take.int()
    return kept


@pytest.mark.parametrize("shape", [(1, 1, 1 << 20), (2, 3, 300007), (2, 130, 70001), (1, 40, 262144)], ids=str)
def test_select_tokens_of_long_rows(shape):
    """Rows of one to 32 slices: all distinct, few distinct, one value, numbers of either
    sign and none, the key to cut at in the first, a middle and the last bits."""
    from proteus_attention import select_kv_tokens

    B, H, T = shape
    g = torch.Generator().manual_seed(T)
    lengths = [T, 65000][:B]
    for kind in range(5):
        w = torch.rand(shape, generator=g)
        if kind == 1:
            w = torch.randint(0, 5, shape, generator=g).float()
        elif kind == 2:
            w.fill_(0.25)
        elif kind == 3:
            w = torch.exp(20 * torch.randn(shape, generator=g)) * torch.randn(shape, generator=g).sign()
            w[..., ::7] = math.nan
            w[..., 1::11], w[..., 2::5] = -0.0, 0.0
        elif kind == 4:  # neighbours in the last bits
            w = (torch.randint(0, 3000, shape, generator=g, dtype=torch.int32) + 0x3f000000).view(torch.float32)
            w[..., 5] = 1e30
        for count, first, last in ((1, 0, 0), (4096, 4, 64), (T // 3, 1, 1), (T + 9, 0, 1)):
            got = select_kv_tokens(w.to(DEV), _i32(lengths).to(DEV), count, first=first, last=last).cpu()
            assert torch.equal(got, choose_long(w, lengths, count, first, last)), (kind, count)


def test_evict_from_long_rows():
    from proteus_attention import evict_kv_tokens

    g = torch.Generator().manual_seed(5)
    cell, D, H, ps = torch.bfloat16, 16, 2, 256
    for lengths, count, bounds in (([70000, 300], 66000, True), ([140000], 257, False)):
        B, N = len(lengths), sum(-(-n // ps) for n in lengths) + len(lengths) * (-(-count // ps)) + 1
        pool = _pool(cell, N, H, ps, D, g, bounds=bounds)
        both = R.make_table(lengths + [count] * B, ps, N, g)
        table, into = both[:B].clone(), both[B:].contiguous()
        table[0, 7] = -1
        w = torch.rand(B, H, table.shape[1] * ps, generator=g)
        have = (torch.arange(w.shape[2]) // ps != 7).expand(B, -1).clone()
        have[1:] = True
        kept = choose(w, lengths, count, 2, 5, have)
        raw = _bytes(cell, pool)
        want, weights_after = moved(raw, kept, w, table, into, _values(cell))
        pages = _pages(cell, pool)
        got, after = evict_kv_tokens(pages, w.to(DEV), table.to(DEV), _i32(lengths).to(DEV), count, into.to(DEV), first=2,
                                     last=5)
        assert torch.equal(got.cpu(), kept) and torch.equal(after.cpu(), weights_after)
        for m in want:
            assert torch.equal(getattr(pages, m).cpu(), want[m]), m


def moved(raw, kept, w, table, into, cells_of):
    """Pool and weights after the move; cells_of(pool, page, head, slots): key values."""
    raw = {m: t.clone() for m, t in raw.items()}
    N, H, ps = raw["k"].shape[:3]
    fresh = torch.zeros_like(w)
    old = {m: t.clone() for m, t in raw.items()}
    for b in range(kept.shape[0]):
        for h in range(H):
            take = [p for p in kept[b, h].tolist() if p >= 0]
            fresh[b, h, :len(take)] = w[b, h, take]
            for i0 in range(0, len(take), ps):
                page = R.page_of(into, b, i0 // ps, N)
                if page < 0:
                    continue
                some = take[i0:i0 + ps]
                for s, p in enumerate(some):
                    src = R.page_of(table, b, p // ps, N)
                    for m in ("k", "v", "k_scale", "v_scale"):
                        if m in raw:
                            raw[m][page, h, s] = old[m][src, h, p % ps]
                if "k_bounds" in raw:
                    x = cells_of(raw, page, h, len(some)).to(raw["k_bounds"].dtype)
                    raw["k_bounds"][page, h, 0], raw["k_bounds"][page, h, 1] = x.amin(0), x.amax(0)
    return raw, fresh


def _bytes(cell, pool):
    return {m: t.view(torch.uint8) if m in "kv" and cell in R.TOP else t for m, t in pool.items()}


def _values(cell):
    def of(raw, page, h, n):
        k, s = raw["k"][page, h, :n], raw["k_scale"][page, h, :n] if "k_scale" in raw else None
        if cell == F.FP4:
            return F.values(k, s)
        return R.values(k.view(cell) if cell in R.TOP else k, s)
    return of


CELLS = [torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn, F.FP4]


@pytest.mark.parametrize("cell", CELLS, ids=str)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_evict(cell, D):
    from proteus_attention import evict_kv_tokens

    g = torch.Generator().manual_seed(D)
    for H, ps, lengths, count, first, last, bounds in (
            (1, 16, [1], 1, 0, 1, True), (2, 16, [0, 40, 16, 17], 17, 1, 3, True), (3, 64, [300, 64, 129], 70, 4, 16, False),
            (1, 128, [1000, 40], 256, 0, 0, True), (2, 256, [700], 300, 1, 200, True), (2, 32, [2100, 5], 1500, 1, 1, False)):
        B = len(lengths)
        held, fresh = sum(-(-n // ps) for n in lengths), B * (-(-count // ps))
        N = held + fresh + 2
        pool = _pool(cell, N, H, ps, D, g, bounds=bounds)
        both = R.make_table([n for n in lengths] + [count] * B, ps, N, g)
        table, into = both[:B], both[B:]
        if count > 200:
            into = into[:, :-(-count // ps) - 1].contiguous()  # what is behind its last page is left out
        if B == 3:
            table[0, 2] = -1  # tokens that are gone
            into[1, 1] = N + 3  # and a page that takes none
        w = torch.rand(B, H, table.shape[1] * ps, generator=g)
        w[0, 0, ::5] = w[0, 0, 0]
        have = torch.tensor([[R.page_of(table, b, p // ps, N) >= 0 for p in range(w.shape[2])] for b in range(B)])
        raw = _bytes(cell, pool)
        kept = choose(w, lengths, count, first, last, have)
        want, weights_after = moved(raw, kept, w, table, into, _values(cell))
        pages = _pages(cell, pool)
        before = w.to(DEV)
        got, after = evict_kv_tokens(pages, before, table.to(DEV), _i32(lengths).to(DEV), count, into.to(DEV), first=first,
                                     last=last)
        assert torch.equal(got.cpu(), kept), (H, ps)
        assert torch.equal(after.cpu(), weights_after) and torch.equal(before.cpu(), w), (H, ps)
        for m in want:
            x = getattr(pages, m)
            x = x.view(torch.uint8).cpu() if want[m].dtype == torch.uint8 else x.cpu()
            assert torch.equal(x, want[m]), (m, H, ps)  # every other page included


@pytest.mark.parametrize("cell", [torch.bfloat16, torch.int8, F.FP4], ids=str)
def test_evicted_sequences_go_on(cell):
    """Attention that weighs its keys, eviction into fresh pages, more tokens, attention
    again over the pages that were freed and taken anew: against the same in plain torch."""
    from proteus_attention import (apply_rotary, evict_kv_tokens, new_kv_pages, new_rotary_positions, paged_attention,
                                   paged_sparse_attention, read_kv_pages, write_kv_pages)

    g = torch.Generator().manual_seed(11)
    dt, B, H, G, D, ps, keep = torch.bfloat16, 2, 2, 3, 64, 16, 48
    rotary = new_rotary_positions(D, device=DEV)
    pages = new_kv_pages(40, H, ps, D, dtype=cell, bounds=True, device=DEV)
    tables = [torch.randperm(40, generator=g)[:2 * B * 6].to(torch.int32).view(2, B, 6)[i].to(DEV) for i in range(2)]
    tables[1] = _i32([[p for p in range(40) if p not in tables[0].cpu().view(-1).tolist()][b * 6:b * 6 + 6] for b in range(B)]).to(DEV)
    lengths, position = _i32([90, 55]).to(DEV), _i32([0, 0]).to(DEV)
    w = torch.zeros(B, H, 6 * ps, device=DEV)
    n, first = 90, True
    for turn in range(3):
        for step in range(1 if first else 20):
            q, k, v = (torch.randn(B, n, h, D, generator=g).to(dt).to(DEV) for h in (H * G, H, H))
            q, k = apply_rotary(q, k, position, rotary)
            at = torch.zeros_like(lengths) if first else lengths
            write_kv_pages(pages, k, v, tables[0], at, counts=lengths if first else None)
            if not first:
                lengths = lengths + 1
            position = position + (lengths if first else 1)
            first, n = False, 1
            before = w.cpu()
            one = q[:, -1].contiguous()
            out = paged_attention(one, pages, tables[0], lengths, key_weights=w)
            kd, vd = (x.cpu() for x in read_kv_pages(pages, tables[0], torch.zeros_like(lengths), lengths, 6 * ps,
                                                     dtype=torch.float32))
            pool = {m: x.view(B * 6, ps, H, D).transpose(1, 2).contiguous() for m, x in (("k", kd), ("v", vd))}
            line = torch.arange(B * 6, dtype=torch.int32).view(B, 6)
            many = lengths.cpu().tolist()
            assert R.attend_error(out.cpu(), R.attend(one.cpu(), pool, line, many), dt, 96) <= 1
            assert holds(w.cpu(), before, weights(one.cpu(), pool, line, many), G, D, 96)
        into = tables[1]
        kept, fresh = evict_kv_tokens(pages, w, tables[0], lengths, keep, into, first=2, last=8)
        assert torch.equal(kept.cpu(), choose(w.cpu(), many, keep, 2, 8))
        after = [x.cpu() for x in read_kv_pages(pages, into, torch.zeros_like(lengths), None, keep, dtype=torch.float32)]
        for b in range(B):
            for h in range(H):
                take = kept[b, h].cpu().long()
                take = take[take >= 0]
                assert torch.equal(after[0][b, :len(take), h], kd[b, take, h])
                assert torch.equal(after[1][b, :len(take), h], vd[b, take, h])
        tables, w, lengths = [into, tables[0]], fresh, lengths.clamp(max=keep)
        paged_sparse_attention(one, pages, tables[0], lengths, 2)


def test_captured_step():
    """Attention with weights and an eviction in a graph, replayed between eager calls of
    the same over other queries and lengths."""
    from proteus_attention import evict_kv_tokens, paged_attention

    g = torch.Generator().manual_seed(8)
    B, H, G, D, ps, P, keep = 3, 2, 4, 64, 16, 700, 500
    pool = R.make_pool(B * (P + 32), H, ps, D, torch.bfloat16, g, bounds=True)
    table = torch.randperm(B * (P + 32), generator=g).view(B, P + 32).to(torch.int32)
    table, into = table[:, :P].contiguous().to(DEV), table[:, P:].contiguous().to(DEV)
    pages = [_pages(torch.bfloat16, pool) for _ in range(2)]
    q = [torch.zeros(B, H * G, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    lengths = [_i32([9000, 31, 500]).to(DEV) for _ in range(2)]
    w = [torch.zeros(B, H, P * ps, device=DEV) for _ in range(2)]

    def step(i):
        out = paged_attention(q[i], pages[i], table, lengths[i], key_weights=w[i])
        return out, *evict_kv_tokens(pages[i], w[i], table, lengths[i], keep, into, last=7)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
            w[i].zero_()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(0)
    for t in range(4):
        x = torch.randn(B, H * G, D, generator=g).bfloat16().to(DEV)
        for i in range(2):
            q[i].copy_(x)
            lengths[i] += 13
        want = step(1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)) and torch.equal(w[0], w[1]), t
        assert all(a is None or torch.equal(a, b) for a, b in zip(*pages)), t


def test_two_streams_at_once():
    from proteus_attention import evict_kv_tokens, paged_attention

    g = torch.Generator().manual_seed(9)
    lengths, H, G, ps, D = [20000, 7], 2, 2, 64, 64
    N = sum(-(-n // ps) for n in lengths) + 40
    pool = R.make_pool(N, H, ps, D, torch.bfloat16, g)
    both = R.make_table(lengths + [1200, 1200], ps, N, g).to(DEV)
    table, into, n = both[:2].contiguous(), both[2:].contiguous(), _i32(lengths).to(DEV)
    q = torch.randn(2, G * H, D, generator=g).bfloat16().to(DEV)

    def step(pages):
        w = torch.zeros(2, H, table.shape[1] * ps, device=DEV)
        return paged_attention(q, pages, table, n, key_weights=w), w, *evict_kv_tokens(pages, w, table, n, 1200, into)

    own = [_pages(torch.bfloat16, pool) for _ in range(2)]
    want = step(own[0])
    torch.cuda.synchronize()
    got = []
    for s, pages in zip([torch.cuda.Stream() for _ in range(2)], own):
        with torch.cuda.stream(s):
            for _ in range(4):
                got.append(step(pages))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x in got for a, b in zip(x, want))
    assert all(a is None or torch.equal(a, b) for a, b in zip(*own))


def test_captured_choice_of_long_rows():
    from proteus_attention import select_kv_tokens

    g = torch.Generator().manual_seed(10)
    w, lengths = torch.zeros(2, 2, 70003, device=DEV), _i32([70003, 69000]).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        select_kv_tokens(w, lengths, 5000)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    held = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(select_kv_tokens(w, lengths, 5000))
    for t in range(4):
        w.copy_(torch.rand(w.shape, generator=g) ** (t + 1))
        want = select_kv_tokens(w, lengths, 5000)
        torch.cuda.synchronize()
        graphs[t % 2].replay()
        graphs[1 - t % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want) and torch.equal(held[1], want), t
        lengths -= 17


def test_eviction_of_pages_beyond_32_bits():
    """A pool of more than 2^32 cells, from its last pages to its first and back."""
    from proteus_attention import KVPages, evict_kv_tokens

    H, ps, D = 2, 256, 128
    N = (1 << 32) // (H * ps * D) + 30
    k, v = (torch.empty(N, H, ps, D, dtype=torch.int8, device=DEV) for _ in range(2))
    scales = [torch.empty(N, H, ps, device=DEV) for _ in range(2)]
    pages = KVPages(k, v, *scales, torch.empty(N, H, 2, D, device=DEV))
    g = torch.Generator().manual_seed(11)
    some = [N - 1, 2, N - 9, 5, N - 3, 1]
    small = _pool(torch.int8, len(some), H, ps, D, g, bounds=True)
    for i, page in enumerate(some):
        for m, t in small.items():
            getattr(pages, m)[page] = t[i].to(DEV)
    table, into, lengths, count = _i32([[0, 1], [2, 3]]), _i32([[5], [4]]), [500, 300], 200
    w = torch.rand(2, H, 2 * ps, generator=g)
    kept = choose(w, lengths, count, 1, 3)
    want, fresh = moved(small, kept, w, table, into, _values(torch.int8))
    names = _i32(some)
    got, after = evict_kv_tokens(pages, w.to(DEV), names[table.long()].to(DEV), _i32(lengths).to(DEV), count,
                                 names[into.long()].to(DEV), last=3)
    assert torch.equal(got.cpu(), kept) and torch.equal(after.cpu(), fresh)
    for i, page in enumerate(some):
        for m in want:
            assert torch.equal(getattr(pages, m)[page].cpu(), want[m][i]), (m, page)


@pytest.mark.parametrize("G", [16, 32])
def test_scores_beyond_32_bits(G):
    """A workspace of more than 2^32 bytes: the weights of its last sequence's keys."""
    from proteus_attention import paged_attention

    g = torch.Generator().manual_seed(12)
    B, D, ps, N = 80, 32, 256, 50
    T = 1 << 20
    pool = _pool(torch.bfloat16, N, 1, ps, D, g)
    table = torch.randint(0, N, (B, T // ps), generator=g, dtype=torch.int32)
    lengths = [1] * (B - 1) + [T - 5]
    q = torch.randn(B, G, D, generator=g).bfloat16()
    before = torch.zeros(B, 1, T, device=DEV)
    paged_attention(q.to(DEV), _pages(torch.bfloat16, pool), table.to(DEV), _i32(lengths).to(DEV), key_weights=before)
    assert bool((before[:-1, 0, 0] == G).all()) and not before[:-1, :, 1:].any() and not before[-1, :, T - 5:].any()
    ref = weights(q[-1:], pool, table[-1:], lengths[-1:])
    assert holds(before[-1:].cpu(), torch.zeros(1, 1, T), ref, G, D, T)
