"""Pages of 4 bits in plain torch on the CPU: what the tests hold the kernels
against, on top of paged_reference, which takes pools of values."""
from __future__ import annotations

import math

import torch

import paged_reference as R

FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def group(D):
    return min(D, 32)


def quantise(x):
    """Codes (..., D) and scale bytes (..., groups) of rows x (..., D) by the
    definition: the scale tried one power after the other, the nearest of eight."""
    g = x.double().unflatten(-1, (-1, group(x.shape[-1])))
    most = g.abs().amax(-1)
    ok = torch.isfinite(most)
    power = torch.full(most.shape, -20)
    for e in range(-20, 125):
        power = torch.where(most > 7.0 * 2.0 ** e, e + 1, power)
    a = torch.where(ok[..., None], g.abs() / torch.exp2(power.double())[..., None], torch.zeros((), dtype=torch.float64))
    code = torch.zeros(a.shape, dtype=torch.uint8)
    for c in range(1, 8):
        middle = (GRID[c - 1] + GRID[c]) / 2
        code = torch.where(a >= middle if c % 2 == 0 else a > middle, c, code).to(torch.uint8)
    sign = torch.signbit(g) & ok[..., None]
    byte = torch.where(ok, power + 127, 255).to(torch.uint8)
    return (code | sign.to(torch.uint8) << 3).flatten(-2), byte


def pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def values(cells, scales):
    """What bytes of cells (..., D / 2) with scale bytes stand for, f32."""
    codes = torch.stack([cells & 15, cells >> 4], -1).flatten(-2)
    x = torch.where(codes > 7, -1.0, 1.0).double() * GRID[(codes & 7).long()]
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127))
    return (x.unflatten(-1, (scales.shape[-1], -1)) * s[..., None]).flatten(-2).float()


def make_pool(N, H, ps, D, g, bounds=False, garbage=False):
    """(k, v, k_scale, v_scale, k_bounds) as bytes, bounds bf16."""
    pool = {}
    for m in "kv":
        x = torch.randn(N, H, ps, D, generator=g)
        if m == "k":
            x += torch.randn(H, 1, D, generator=g)
        codes, pool[m + "_scale"] = quantise(x)
        pool[m] = pack(codes)
        if garbage:
            pool[m + "_scale"] = torch.full_like(pool[m + "_scale"], 255)
    if bounds:
        x = values(pool["k"], pool["k_scale"])
        pool["k_bounds"] = torch.stack([x.amin(2), x.amax(2)], 2).bfloat16()
    return pool


def as_values(pool):
    """A pool of paged_reference."""
    out = {m: values(pool[m], pool[m + "_scale"]) for m in "kv"}
    return dict(out, **{m: t for m, t in pool.items() if m == "k_bounds"})


def pages(pool, dev):
    from proteus_attention import KVPages

    d = {m: t.to(dev) for m, t in pool.items()}
    return KVPages(d["k"].view(FP4), d["v"].view(FP4), d["k_scale"].view(E8M0), d["v_scale"].view(E8M0), d.get("k_bounds"))


def raw(pages_):
    """Bytes of a KVPages on the CPU."""
    out = {m: getattr(pages_, m).view(torch.uint8).cpu() for m in ("k", "v", "k_scale", "v_scale")}
    return out if pages_.k_bounds is None else dict(out, k_bounds=pages_.k_bounds.cpu())


def write(pool, k, v, table, starts, counts):
    """The pool after the new rows."""
    pool = {m: t.clone() for m, t in pool.items()}
    N, ps = pool["k"].shape[0], pool["k"].shape[2]
    for b in range(k.shape[0]):
        found = {}
        for i in range(min(int(counts[b]), k.shape[1])):
            pos = int(starts[b]) + i
            page = R.page_of(table, b, pos // ps, N) if pos >= 0 else -1
            if page >= 0:
                found.setdefault(page, []).append((pos % ps, i))
        for page, rows in found.items():
            slots, at = (torch.tensor(x) for x in zip(*rows))
            for m, new in (("k", k), ("v", v)):
                codes, s = quantise(new[b, at].transpose(0, 1))
                c = pack(codes)
                pool[m][page, :, slots], pool[m + "_scale"][page, :, slots] = c, s
                if m == "k" and "k_bounds" in pool:
                    x = values(c, s).bfloat16()
                    lo, hi, b2 = x.amin(1), x.amax(1), pool["k_bounds"]
                    if int(slots[0]) > 0:
                        lo, hi = torch.minimum(lo, b2[page, :, 0]), torch.maximum(hi, b2[page, :, 1])
                    b2[page, :, 0], b2[page, :, 1] = lo, hi
    return pool
