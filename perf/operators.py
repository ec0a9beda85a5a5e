"""Performance cases of the paged key-value cache and the attention that reads
it: the calls that a program makes once a prompt is in and tokens come one by
one.

Four kinds of call (``op``):

* ``write``  -- ``write_kv_pages``: new tokens' keys and values into the pages of
  their sequences, in the cache's type (8-bit caches with one scale per token
  and head), and the pages' key bounds with them;
* ``read``   -- ``read_kv_pages``: a range of every sequence back out of its pages;
* ``attend`` -- ``paged_attention``: one new token of each sequence over all of its
  cache, or over a window of it;
* ``sparse`` -- ``paged_sparse_attention``: the same over the pages that the bounds
  of their keys select for each sequence and key-value head.

A pool holds the pages of all sequences in a random order, as it does after
some hours of sequences that come and go.  Keys are N(0, 1) around an offset of
their own for each head and channel, queries and values N(0, 1).  Lengths are
spread over a case's range evenly in their logarithm.  Everything is made from
the seed on the GPU.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "proteus-flux-attention_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "int8": torch.int8,
          "e4m3": torch.float8_e4m3fn}
ESIZE = {"bf16": 2, "f16": 2, "f32": 4, "int8": 1, "e4m3": 1}
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest value that an 8-bit cell holds
LEAST_SCALE = 1e-6
DEVICE = "cuda"


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _case(op, name=None, **kw):
    # H query heads of D share Hkv key-value heads; `lo`..`hi` tokens are in the
    # cache; `n`: tokens to write or read; `window`: the last keys that attend
    # sees (0: all); `keep`: pages that sparse attends to; `strided`: new tokens
    # are slices of one projection's output
    case = dict(op=op, dtype="bf16", cache="bf16", B=1, H=8, Hkv=8, D=64, page=64, lo=1, hi=64, n=0, window=0, keep=0,
                bounds=False, strided=False)
    case.update(kw)
    return dict(case, name=name) if name else case


def listed():
    return [
        # One interactive sequence with a short prompt behind it: latency alone.
        _case("attend", "attend_one_short_bf16", page=16, lo=173, hi=173),
        # A serving batch of grouped-query heads, lengths from a first token to 8K.
        _case("attend", "attend_batch_ragged_bf16", B=64, H=32, D=128, lo=1, hi=8192),
        # One book-length context of about a million tokens in an 8-bit cache: few
        # rows, a long axis.
        _case("attend", "attend_one_million_int8", cache="int8", H=32, Hkv=4, D=128, page=128, lo=1000003, hi=1000003),
        # Full-precision heads of the layer's own width with a sliding window.
        _case("attend", "attend_window_f32", dtype="f32", cache="f32", B=24, page=32, lo=700, hi=20000, window=6000),
        # The token that a batch of sequences has just computed, with its page's bounds.
        _case("write", "write_token_bf16", B=128, D=128, lo=1, hi=2000, n=1, bounds=True, strided=True),
        # Prompts of a batch quantised as they are written, and read back for checking.
        _case("write", "write_prompts_int8", cache="int8", B=8, D=128, lo=0, hi=0, n=4099, bounds=True),
        # One 64K prompt of the layer's shape, written from the projection's output.
        _case("write", "write_prompt_64k_f16", dtype="f16", cache="f16", lo=0, hi=0, n=65536, page=128, strided=True),
        # A chunk of a running prompt read back to be attended to by a dense kernel.
        _case("read", "read_chunk_bf16", B=3, page=16, D=32, lo=1500, hi=4000, n=1000),
        # Two long contexts dequantised, as before moving them elsewhere.
        _case("read", "read_long_e4m3", cache="e4m3", B=2, Hkv=8, D=128, page=256, lo=100000, hi=131072, n=131072),
        # A single sequence of the layer's heads with selected pages.
        _case("sparse", "sparse_one_4k_bf16", page=16, lo=4001, hi=4001, keep=32, bounds=True),
        # Four contexts of up to half a million tokens, grouped-query heads, 64 pages each.
        _case("sparse", "sparse_long_bf16", B=4, H=32, D=128, lo=260000, hi=524288, keep=64, bounds=True),
        # A ragged batch on an 8-bit cache, few key-value heads.
        _case("sparse", "sparse_batch_e4m3", dtype="f16", cache="e4m3", B=48, H=16, Hkv=2, D=128, page=32, lo=90,
              hi=65536, keep=48, bounds=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "sparse"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    cache = rng.choice([dtype, dtype, "int8", "e4m3"])
    D = rng.choice([16, 32, 64, 64, 128, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    page = rng.choice([16, 32, 64, 128, 256])
    B = _log(rng, 1, 96)
    case = _case(op, dtype=dtype, cache=cache, B=B, Hkv=Hkv, H=Hkv * rng.choice([1, 1, 2, 4, 5, 8, 16]), D=D, page=page,
                 bounds=op == "sparse" or (op == "write" and rng.random() < 0.5), strided=rng.random() < 0.5)
    # at most 400 MB of cache in the pool, 100 MB where it is written
    most = max(64, min(1 << 20, int((1e8 if op == "write" else 4e8) / (B * Hkv * D * 2 * ESIZE[cache]))))
    hi = _log(rng, 40, most)
    lo = _log(rng, 1, hi)
    if op == "write":
        n = 1 if rng.random() < 0.3 else _log(rng, 2, most)
        lo, hi = (0, 0) if rng.random() < 0.4 else (lo, max(lo, min(hi, most - n)))
        case.update(n=n)
    elif op == "read":
        case.update(n=_log(rng, 1, hi))
    elif op == "attend":
        case.update(window=_log(rng, 1, hi) if rng.random() < 0.25 else 0)
    else:
        case.update(keep=_log(rng, 2, 96))
    case.update(lo=lo, hi=hi)
    return case


def _lengths(case):
    """Tokens in the cache of each sequence, from the case alone."""
    lo, hi = case["lo"], case["hi"]
    if hi <= 0:
        return [0] * case["B"]
    lo = max(lo, 1)
    if case["B"] == 1:
        return [hi]
    return [int(round(lo * (hi / lo) ** ((0.618034 * (b + 1)) % 1.0))) for b in range(case["B"])]


def _counts(case):
    """Tokens of each sequence that a call writes or reads: all `n` of the
    first one, fewer of the others (down to half), no more than a read has."""
    n = case["n"]
    got = [max(1, n - (b * n) // (2 * case["B"])) for b in range(case["B"])]
    if case["op"] == "read":
        got = [min(c, m) for c, m in zip(got, _lengths(case))]
    return got


def _tokens(case):
    """Positions that a sequence has pages for."""
    more = _counts(case) if case["op"] == "write" else [0] * case["B"]
    return [m + c for m, c in zip(_lengths(case), more)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _cells(x, cache):
    """x (..., D) f32 in the cache's type, with its scales (..., ) or None."""
    if cache not in TOP:
        return x.to(DTYPES[cache]), None
    top = torch.full((), TOP[cache], device=x.device)
    scale = torch.clamp(x.abs().amax(-1) / top, min=LEAST_SCALE)
    cells = x / scale[..., None]
    return (cells.round() if cache == "int8" else cells).to(DTYPES[cache]), scale


def _values(cells, scale):
    return cells.float() if scale is None else cells.float() * scale[..., None]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, ct = DTYPES[case["dtype"]], DTYPES[case["cache"]]
    B, H, Hkv, D, ps = (case[k] for k in ("B", "H", "Hkv", "D", "page"))
    held = [-(-t // ps) for t in _tokens(case)]
    N = sum(held) + 3
    order = torch.randperm(N, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((B, max(held) + 1), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
    offset = torch.randn(Hkv, 1, D, generator=g, device=DEVICE)

    pages = {}
    for which in "kv":
        raw = torch.randn(N, Hkv, ps, D, generator=g, device=DEVICE, dtype=dt)
        if which == "k":
            raw += offset.to(dt)
        pages[which], scale = (raw, None) if ct == dt else _cells(raw.float(), case["cache"])
        del raw
        if scale is not None:
            pages[which + "_scale"] = scale
    if case["bounds"]:
        keys = pages["k"] if ct == dt else _values(pages["k"], pages["k_scale"])
        pages["k_bounds"] = torch.stack([keys.amin(2), keys.amax(2)], 2)
    state = dict(case=case, pages=pages, table=table, lengths=lengths)
    if case["op"] in ("write", "read"):
        state["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEVICE)
    if case["op"] == "write":
        if case["strided"]:  # slices of a fused q, k, v projection's output
            qkv = torch.randn(B, case["n"], 3, Hkv, D, generator=g, device=DEVICE, dtype=dt)
            qkv[:, :, 1] += offset[:, 0].to(dt)
            state["k"], state["v"] = qkv[:, :, 1], qkv[:, :, 2]
        else:
            state["k"] = torch.randn(B, case["n"], Hkv, D, generator=g, device=DEVICE, dtype=dt) + offset[:, 0].to(dt)
            state["v"] = torch.randn(B, case["n"], Hkv, D, generator=g, device=DEVICE, dtype=dt)
    elif case["op"] == "read":  # the last tokens of each sequence
        state["starts"] = lengths - state["counts"]
    else:
        state["q"] = torch.randn(B, H, D, generator=g, device=DEVICE, dtype=dt)
        if case["window"]:
            state["starts"] = torch.clamp(lengths - case["window"], min=0)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from proteus_attention.kernels.paged_attn import (KVPages, paged_attention, paged_sparse_attention, read_kv_pages,
                                                      write_kv_pages)

    case, table, lengths = state["case"], state["table"], state["lengths"]
    pages = KVPages(**state["pages"])
    if case["op"] == "write":
        write_kv_pages(pages, state["k"], state["v"], table, lengths, counts=state["counts"])
        if pages.k_scale is None:
            return state["pages"]
        k, v = read_kv_pages(pages, table, lengths, state["counts"], case["n"])
        return dict(k=k, v=v, **{m: t for m, t in state["pages"].items() if m == "k_bounds"})
    if case["op"] == "read":
        k, v = read_kv_pages(pages, table, state["starts"], state["counts"], case["n"],
                             dtype=DTYPES[case["dtype"]])
        return dict(k=k, v=v)
    if case["op"] == "attend":
        return paged_attention(state["q"], pages, table, lengths, starts=state.get("starts"))
    out, chosen = paged_sparse_attention(state["q"], pages, table, lengths, case["keep"])
    return dict(out=out, pages=chosen)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "write":
        return _plain_write(state)
    if case["op"] == "read":
        k, v = _plain_read(state, state["starts"], DTYPES[case["dtype"]])
        return dict(k=k, v=v)
    if case["op"] == "attend":
        return _plain_attend(state)
    return _plain_sparse(state)


def _where(state, starts):
    """Page and slot (B, n) of the positions starts[b] + i, and whether the call has them."""
    case, table = state["case"], state["table"]
    i = torch.arange(case["n"], device=DEVICE)
    pos = starts[:, None].long() + i
    page = torch.gather(table.long(), 1, (pos // case["page"]).clamp(max=table.shape[1] - 1))
    return page, pos % case["page"], (i < state["counts"][:, None]) & (page >= 0)


def _plain_write(state):
    case, pages, starts = state["case"], state["pages"], state["lengths"]
    ps, n = case["page"], case["n"]
    page, slot, have = _where(state, starts)
    fresh = None
    for which in "kv":
        cells, scale = _cells(state[which].float(), case["cache"])
        pages[which][page[have], :, slot[have]] = cells[have]
        if scale is not None:
            pages[which + "_scale"][page[have], :, slot[have]] = scale[have]
        if which == "k" and case["bounds"]:
            fresh = _values(cells, scale)
    if fresh is not None:
        # the written keys by the page that they lie in: (B, touched, ps, Hkv, D)
        touched = (n + ps - 2) // ps + 1
        first = starts.long() // ps
        pos = (first[:, None] + torch.arange(touched, device=DEVICE))[:, :, None] * ps + torch.arange(ps, device=DEVICE)
        i = pos - starts[:, None, None]
        inside = (i >= 0) & (i < state["counts"][:, None, None])
        rows = fresh[torch.arange(case["B"], device=DEVICE)[:, None, None], i.clamp(0, n - 1)]
        gone = ~inside[..., None, None]
        low = rows.masked_fill(gone, math.inf).amin(2)
        high = rows.masked_fill(gone, -math.inf).amax(2)
        cover = (first[:, None] + torch.arange(touched, device=DEVICE))
        ids = torch.gather(state["table"].long(), 1, cover.clamp(max=state["table"].shape[1] - 1))
        hit = inside.any(2) & (ids >= 0)
        bounds = pages["k_bounds"]
        old = bounds[ids.clamp(min=0)].float()
        joins = (cover * ps < starts[:, None])[..., None, None]
        low = torch.where(joins, torch.minimum(low, old[:, :, :, 0]), low)
        high = torch.where(joins, torch.maximum(high, old[:, :, :, 1]), high)
        bounds[ids[hit]] = torch.stack([low, high], 3)[hit].to(bounds.dtype)
    if case["cache"] not in TOP:
        return pages
    k, v = _plain_read(state, starts, torch.float32)
    return dict(k=k, v=v, **{m: t for m, t in pages.items() if m == "k_bounds"})


def _plain_read(state, starts, dtype):
    pages = state["pages"]
    page, slot, have = _where(state, starts)
    page = page.clamp(min=0)
    got = []
    for which in "kv":
        scale = pages.get(which + "_scale")
        rows = _values(pages[which][page, :, slot], scale[page, :, slot] if scale is not None else None)
        got.append(rows.masked_fill(~have[..., None, None], 0.0).to(dtype))
    return got


def _weights(scores, seen):
    """Softmax over the keys that are seen; zeros where a row sees none."""
    scores = scores.masked_fill(~seen, -math.inf)
    most = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(most), torch.zeros_like(most), most)).masked_fill(~seen, 0.0)
    return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _gathered(pages, which, ids):
    """Pages ids (B, P) or (B, Hkv, P) as (B, Hkv, P * page, D) f32."""
    scale = pages.get(which + "_scale")
    if ids.dim() == 2:
        x = _values(pages[which][ids], scale[ids] if scale is not None else None).transpose(1, 2)
    else:
        h = torch.arange(ids.shape[1], device=DEVICE)[:, None]
        x = _values(pages[which][ids, h], scale[ids, h] if scale is not None else None)
    return x.flatten(2, 3)


def _plain_attention(state, ids, seen):
    case = state["case"]
    q = state["q"].float().view(case["B"], case["Hkv"], -1, case["D"])
    scores = torch.matmul(q, _gathered(state["pages"], "k", ids).transpose(2, 3).contiguous()) / math.sqrt(case["D"])
    out = torch.matmul(_weights(scores, seen), _gathered(state["pages"], "v", ids))
    return out.reshape(state["q"].shape).to(state["q"].dtype)


def _plain_attend(state):
    case, table = state["case"], state["table"]
    pos = torch.arange(table.shape[1] * case["page"], device=DEVICE)
    seen = pos < state["lengths"][:, None]
    if "starts" in state:
        seen &= pos >= state["starts"][:, None]
    return _plain_attention(state, table.long().clamp(min=0), seen[:, None, None, :])


def _plain_sparse(state):
    """A page's score for a key-value head: the largest of its query heads'
    sums over the channels of q * (max if q > 0 else min), in 64 bits, held in
    32.  The first and the last page of a sequence always count."""
    case, pages, table = state["case"], state["pages"], state["table"]
    B, Hkv, D, ps, keep = (case[k] for k in ("B", "Hkv", "D", "page", "keep"))
    P = table.shape[1]
    q = state["q"].double().view(B, Hkv, -1, D)
    bounds = pages["k_bounds"][table.long().clamp(min=0)].double()  # (B, P, Hkv, 2, D)
    low = bounds[:, :, :, 0].permute(0, 2, 3, 1).contiguous()
    high = bounds[:, :, :, 1].permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(q.clamp(min=0), high) + torch.matmul(q.clamp(max=0), low)
    score = score.amax(2).float()
    held = (state["lengths"].long() + ps - 1) // ps
    page = torch.arange(P, device=DEVICE)
    score = score.masked_fill(((page == 0) | (page == held[:, None] - 1))[:, None], math.inf)
    score = score.masked_fill((page >= held[:, None])[:, None], -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    if P < keep:
        order = torch.nn.functional.pad(order, (0, keep - P), value=P)
    none = torch.full_like(order, P)
    chosen = torch.where(torch.arange(keep, device=DEVICE) < held[:, None, None], order, none).sort(-1).values
    chosen = chosen.masked_fill(chosen == P, -1)
    ids = torch.gather(table.long()[:, None].expand(B, Hkv, P), 2, chosen.clamp(min=0)).clamp(min=0)
    pos = chosen[..., None] * ps + torch.arange(ps, device=DEVICE)
    seen = (chosen[..., None] >= 0) & (pos < state["lengths"][:, None, None, None])
    out = _plain_attention(state, ids, seen.flatten(2)[:, :, None])
    return dict(out=out, pages=chosen.to(torch.int32))


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _quantised64(x, cache):
    """Cells and scales of x (..., D) by the definition, which holds a scale and
    the quotient by it in 32 bits: computed in 64 and rounded there."""
    x = x.double()
    scale = (x.abs().amax(-1) / TOP[cache]).float().double()
    scale = torch.where(scale < LEAST_SCALE, torch.full_like(scale, LEAST_SCALE).float().double(), scale)
    quotient = (x / scale[..., None]).float()
    if cache == "int8":
        return torch.round(quotient.double()), scale
    a = quotient.double().abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))).clamp(min=-6.0) - 3.0)
    return torch.sign(quotient.double()) * torch.round(a / step) * step, scale


def _held64(case, state, b, which):
    """All cached rows of sequence b: (tokens, Hkv, D) in 64 bits."""
    pages, ps = state["pages"], case["page"]
    ids = state["table"][b][:-(-_lengths(case)[b] // ps)].long()
    x = pages[which][ids].double()
    if which + "_scale" in pages:
        x = x * pages[which + "_scale"][ids].double()[..., None]
    return x.permute(0, 2, 1, 3).reshape(-1, case["Hkv"], case["D"])[:_lengths(case)[b]]


def exact(case, seed):
    state = prepare(case, seed)
    return dict(write=_exact_write, read=_exact_read, attend=_exact_attend, sparse=_exact_sparse)[case["op"]](case, state)


def _exact_write(case, state):
    pages, ps, cache = state["pages"], case["page"], case["cache"]
    table = state["table"].tolist()
    new = {m: pages[m].double() for m in pages if cache not in TOP or m == "k_bounds"}
    back = {w: torch.zeros(case["B"], case["n"], case["Hkv"], case["D"], dtype=torch.float64, device=DEVICE) for w in "kv"}
    for b, (start, count) in enumerate(zip(_lengths(case), _counts(case))):
        for which in "kv":
            rows = state[which][b, :count].double()
            if cache in TOP:
                cells, scale = _quantised64(rows, cache)
                rows = cells * scale[..., None]
                back[which][b, :count] = rows
            at = 0
            while at < count:
                p, s = divmod(start + at, ps)
                m = min(ps - s, count - at)
                some = rows[at:at + m].transpose(0, 1)
                if cache not in TOP:
                    new[which][table[b][p], :, s:s + m] = some
                if which == "k" and case["bounds"]:
                    low, high = some.amin(1), some.amax(1)
                    here = new["k_bounds"][table[b][p]]
                    if s > 0:
                        low, high = torch.minimum(low, here[:, 0]), torch.maximum(high, here[:, 1])
                    here[:, 0], here[:, 1] = low, high
                at += m
    return new if cache not in TOP else dict(back, **new)


def _exact_read(case, state):
    got = {w: torch.zeros(case["B"], case["n"], case["Hkv"], case["D"], dtype=torch.float64, device=DEVICE) for w in "kv"}
    for b, (length, count) in enumerate(zip(_lengths(case), _counts(case))):
        for which in "kv":
            got[which][b, :count] = _held64(case, state, b, which)[length - count:]
    return got


def _softmax64(q, k, v):
    """q (G, D), k and v (n, D)."""
    s = (k * q[:, None]).sum(-1) / math.sqrt(q.shape[-1]) if k.shape[0] * q.numel() < 1 << 26 else q @ k.T / math.sqrt(q.shape[-1])
    return torch.softmax(s, -1) @ v


def _exact_attend(case, state):
    out = torch.zeros(case["B"], case["H"], case["D"], dtype=torch.float64, device=DEVICE)
    G = case["H"] // case["Hkv"]
    for b, length in enumerate(_lengths(case)):
        first = max(0, length - case["window"]) if case["window"] else 0
        k, v = (_held64(case, state, b, w)[first:] for w in "kv")
        for h in range(case["Hkv"]):
            out[b, h * G:h * G + G] = _softmax64(state["q"][b, h * G:h * G + G].double(), k[:, h], v[:, h])
    return out


def _exact_sparse(case, state):
    B, H, Hkv, D, ps, keep = (case[k] for k in ("B", "H", "Hkv", "D", "page", "keep"))
    G = H // Hkv
    out = torch.zeros(B, H, D, dtype=torch.float64, device=DEVICE)
    chosen = torch.full((B, Hkv, keep), -1, dtype=torch.int32, device=DEVICE)
    for b, length in enumerate(_lengths(case)):
        held = -(-length // ps)
        ids = state["table"][b, :held].long()
        bounds = state["pages"]["k_bounds"][ids].double()
        for h in range(Hkv):
            q = state["q"][b, h * G:h * G + G].double()
            score = torch.full((held,), -math.inf, device=DEVICE)
            for row in q:
                side = torch.where(row > 0, bounds[:, h, 1], bounds[:, h, 0])
                score = torch.maximum(score, (side * row).sum(-1).float())
            score[0] = score[held - 1] = math.inf
            take = torch.sort(score, descending=True, stable=True).indices[:keep].sort().values
            chosen[b, h, :take.numel()] = take.int()
            rows = {}
            for w in "kv":
                x = state["pages"][w][ids[take], h].double()
                if w + "_scale" in state["pages"]:
                    x = x * state["pages"][w + "_scale"][ids[take], h].double()[..., None]
                pos = take[:, None] * ps + torch.arange(ps, device=DEVICE)
                rows[w] = x[pos < length]
            out[b, h * G:h * G + G] = _softmax64(q, rows["k"], rows["v"])
    return dict(out=out, pages=chosen)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    H, Hkv, D, ps = (case[k] for k in ("H", "Hkv", "D", "page"))
    E, C = ESIZE[case["dtype"]], ESIZE[case["cache"]]
    row = 2 * Hkv * (D * C + (4 if case["cache"] in TOP else 0))  # one token in the cache
    token = 2 * Hkv * D * E  # one token outside of it
    page_bounds = Hkv * 2 * D * (4 if case["cache"] in TOP else C)
    lens = _lengths(case)
    if case["op"] == "write":
        tokens = sum(_counts(case))
        nbytes = tokens * (token + row)
        if case["bounds"]:
            nbytes += sum((m + c - 1) // ps - m // ps + 1 for m, c in zip(lens, _counts(case))) * page_bounds
        if case["cache"] in TOP:  # read back as f32
            nbytes += tokens * row + case["B"] * case["n"] * 2 * Hkv * D * 4
        return dict(bytes=nbytes, flops=0)
    if case["op"] == "read":
        return dict(bytes=sum(_counts(case)) * row + case["B"] * case["n"] * token, flops=0)
    ends = 2 * case["B"] * H * D * E
    if case["op"] == "attend":
        keys = sum(min(m, case["window"] or m) for m in lens)
        return dict(bytes=keys * row + ends, flops=4 * keys * H * D)
    held = [-(-m // ps) for m in lens]
    keys = sum(min(m, case["keep"] * ps) for m in lens)
    return dict(bytes=sum(held) * page_bounds + keys * row + ends, flops=4 * keys * H * D + 2 * sum(held) * H * D)
