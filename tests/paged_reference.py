"""Paged key-value cache in plain torch on the CPU, 64 bits where a value is
computed: what the tests hold the kernels against."""
from __future__ import annotations

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
PAIRS = [(t, t) for t in (torch.float32, torch.bfloat16, torch.float16)] + \
    [(t, c) for c in TOP for t in (torch.float32, torch.bfloat16, torch.float16)]


def pair_id(p):
    return "-".join(str(t).replace("torch.", "") for t in p)


def quantise(x: torch.Tensor, cell: torch.dtype):
    """Cells and scales of rows x (..., D)."""
    x = x.float()
    most = x.abs().amax(-1)
    scale = torch.clamp(most / torch.tensor(TOP[cell]), min=1e-6)
    ok = torch.isfinite(most)
    q = torch.where(ok[..., None], x / scale[..., None], torch.zeros(()))
    cells = (q.round() if cell == torch.int8 else q).to(cell)
    return cells, torch.where(ok, scale, torch.full((), math.nan))


def values(cells: torch.Tensor, scale) -> torch.Tensor:
    """What cells stand for, f32."""
    return cells.float() if scale is None else cells.float() * scale[..., None]


def make_pool(N, H, ps, D, cell, g, bounds=False, garbage=False):
    """A pool (k, v, k_scale, v_scale, k_bounds) on the CPU with rows of N(0, 1)
    values; `garbage`: NaN, infinities and the like in all of it instead."""
    pool = {}
    for m in "kv":
        x = torch.randn(N, H, ps, D, generator=g)
        if m == "k":
            x += torch.randn(H, 1, D, generator=g)
        if garbage:
            x = torch.full_like(x, math.nan)
            x[..., ::3] = math.inf
            x[..., 1::3] = -math.inf
        if cell in TOP:
            if garbage:
                pool[m] = torch.full((N, H, ps, D), 0x7f, dtype=torch.uint8).view(cell)
                pool[m + "_scale"] = torch.full((N, H, ps), math.nan)
            else:
                pool[m], pool[m + "_scale"] = quantise(x, cell)
        else:
            pool[m] = x.to(cell)
    if bounds:
        bt = torch.float32 if cell in TOP else cell
        if garbage:
            pool["k_bounds"] = torch.full((N, H, 2, D), math.nan).to(bt)
        else:
            x = values(pool["k"], pool.get("k_scale"))
            pool["k_bounds"] = torch.stack([x.amin(2), x.amax(2)], 2).to(bt)
    return pool


def make_table(lengths, ps, N, g, extra=1):
    """Pages of a pool of N in random order, -1 behind the last."""
    held = [-(-max(n, 0) // ps) for n in lengths]
    assert sum(held) <= N
    order = torch.randperm(N, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(held) + extra), -1, dtype=torch.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    return table


def page_of(table, b, p, N):
    if not 0 <= p < table.shape[1]:
        return -1
    i = int(table[b, p])
    return i if 0 <= i < N else -1


def write(pool, k, v, table, starts, counts):
    """The pool after the new rows, and the positions (page, slot) written."""
    pool = {m: t.clone() for m, t in pool.items()}
    N, H, ps, D = pool["k"].shape
    cell = pool["k"].dtype
    raw8 = {m: pool[m].view(torch.uint8) for m in "kv"} if cell in TOP else None
    for b in range(k.shape[0]):
        pages = {}
        for i in range(min(int(counts[b]), k.shape[1])):
            pos = int(starts[b]) + i
            if pos < 0:
                continue
            page = page_of(table, b, pos // ps, N)
            if page >= 0:
                pages.setdefault(page, []).append((pos % ps, i))
        for page, rows in pages.items():
            slots, at = (torch.tensor(x) for x in zip(*rows))
            for m, new in (("k", k), ("v", v)):
                x = new[b, at].transpose(0, 1)  # (H, rows, D)
                if cell in TOP:
                    c, s = quantise(x, cell)
                    raw8[m][page, :, slots] = c.view(torch.uint8)
                    pool[m + "_scale"][page, :, slots] = s
                    x = values(c, s)
                else:
                    pool[m][page, :, slots] = x
                if m == "k" and "k_bounds" in pool:
                    b2 = pool["k_bounds"]
                    x = x.to(b2.dtype)
                    lo, hi = x.amin(1), x.amax(1)
                    if int(slots[0]) > 0:
                        lo, hi = torch.minimum(lo, b2[page, :, 0]), torch.maximum(hi, b2[page, :, 1])
                    b2[page, :, 0], b2[page, :, 1] = lo, hi
    return pool


def read(pool, table, starts, counts, n, dtype):
    N, H, ps, D = pool["k"].shape
    out = {m: torch.zeros(table.shape[0], n, H, D, dtype=dtype) for m in "kv"}
    for m in "kv":
        x = values(pool[m], pool.get(m + "_scale")).to(dtype)
        for b in range(table.shape[0]):
            for i in range(min(int(counts[b]), n)):
                pos = int(starts[b]) + i
                page = page_of(table, b, pos // ps, N) if pos >= 0 else -1
                if page >= 0:
                    out[m][b, i] = x[page, :, pos % ps]
    return out["k"], out["v"]


def select(q, pool, table, lengths, starts, count, first, last):
    N, H, ps, D = pool["k"].shape
    B, G = q.shape[0], q.shape[1] // H
    chosen = torch.full((B, H, count), -1, dtype=torch.int32)
    bounds = pool["k_bounds"].double()
    for b in range(B):
        length = min(max(int(lengths[b]), 0), table.shape[1] * ps)
        start = max(int(starts[b]), 0) if starts is not None else 0
        if start >= length:
            continue
        p0, pe = start // ps, -(-length // ps)
        for h in range(H):
            found = []
            for p in range(p0, pe):
                page = page_of(table, b, p, N)
                if page < 0:
                    continue
                x = q[b, h * G:h * G + G].double()
                s = (x * torch.where(x > 0, bounds[page, h, 1], bounds[page, h, 0])).sum(-1).float()
                nan = bool(torch.isnan(s).any())
                s = -math.inf if nan else float(s.max())
                forced = p < p0 + first or p >= pe - last
                found.append((not forced, nan, -s, p))
            take = sorted(p for *_, p in sorted(found)[:count])
            chosen[b, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
    return chosen


def attend(q, pool, table, lengths, starts=None, selected=None, scale=None):
    """(B, heads, D) in 64 bits; with it, for each row, the sum of p |v| and
    the largest score's magnitude sum_d |q_d k_d| * scale: what an f32
    computation's error is measured by."""
    N, H, ps, D = pool["k"].shape
    B, G = q.shape[0], q.shape[1] // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    most = torch.zeros(q.shape[:2], dtype=torch.float64)
    cells = {}
    for m in "kv":
        cells[m] = pool[m].double()
        if m + "_scale" in pool:
            cells[m] = cells[m] * pool[m + "_scale"].double()[..., None]
    for b in range(B):
        length = min(max(int(lengths[b]), 0), table.shape[1] * ps)
        start = max(int(starts[b]), 0) if starts is not None else 0
        for h in range(H):
            entries = range(-(-length // ps)) if selected is None else selected[b, h].tolist()
            ks, vs = [], []
            for e in entries:
                page = page_of(table, b, e, N)
                if page < 0:
                    continue
                a, z = max(start - e * ps, 0), min(length - e * ps, ps)
                if a < z:
                    ks.append(cells["k"][page, h, a:z])
                    vs.append(cells["v"][page, h, a:z])
            if not ks:
                continue
            k, v = torch.cat(ks), torch.cat(vs)
            x = q[b, h * G:h * G + G].double()
            p = torch.softmax(x @ k.T * scale, -1)
            out[b, h * G:h * G + G] = p @ v
            size[b, h * G:h * G + G] = p @ v.abs()
            most[b, h * G:h * G + G] = (x.abs() @ k.abs().T * scale).amax(-1)
    return out, size, most


def attend_error(got, ref, dtype, n):
    """The largest row error over its bound (<= 1 passes).  Bound of a row, in
    its 2-norm: half a step of the result's type on every value, plus, on the
    sum of p |v|, the f32 rounding of a score, sqrt(D) + 3 roundings (sums as a
    random walk; scale, maximum and exponential) of up to sum |q k| scale each,
    four times over for the largest of many; sqrt(n) roundings of the sums over
    n keys, four times over; and, for 16-bit results, p held in two parts of
    eight bits or more: 2^-16."""
    out, size, most = ref
    D = out.shape[-1]
    step = 2.0 ** -24
    f32 = 4 * step * ((math.sqrt(D) + 3) * most + math.sqrt(max(n, 1)) + 4)
    if dtype != torch.float32:
        f32 = f32 + 2.0 ** -16
    bound = HALF[dtype] * out.norm(dim=-1) + f32 * size.norm(dim=-1)
    err = (got.double() - out).norm(dim=-1)
    if not bool(torch.isfinite(got.double()).all()):
        return math.inf
    zero = bound == 0
    if bool((err[zero] != 0).any()):
        return math.inf
    return float((err / bound.clamp(min=1e-300)).masked_fill(zero, 0.0).max())
