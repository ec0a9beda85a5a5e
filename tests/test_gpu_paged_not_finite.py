"""One-token attention where what is seen is not finite: values, keys and queries,
whichever wave or workgroup of a row sees them and however little they weigh."""
from __future__ import annotations

import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"

# sequences, tokens, tokens of low score: one wave's tile beside others of the
# workgroup; a row in a few workgroups; in more than 16
FORMS = [(1, 100, 64), (16, 1500, 512), (1, 40001, 4096)]


def _case(pair, B, n, low, D, g):
    """Rows whose first `low` keys weigh 2^-300 and less of the others."""
    dt, cell = pair
    H, G, ps = 2, 2, 16
    P = -(-n // ps)
    pool = R.make_pool(B * P, H, ps, D, cell, g)
    table = torch.randperm(B * P, generator=g).view(B, P).to(torch.int32)
    k = torch.full((B, P * ps, 1, 1), 4.0)
    k[:, :low] = -4.0
    rows = (k * torch.ones(H, D)).view(B, P, ps, H, D).transpose(2, 3).flatten(0, 1)
    at = table.flatten().long()
    if cell in R.TOP:
        cells, scale = R.quantise(rows, cell)
        pool["k"].view(torch.uint8)[at] = cells.view(torch.uint8)
        pool["k_scale"][at] = scale
    else:
        pool["k"][at] = rows.to(cell)
    q = (4.0 + 0.1 * torch.rand(B, H * G, D, generator=g)).to(dt)
    return pool, table, q, torch.full((B,), n, dtype=torch.int32)


def _run(q, pool, table, lengths, **kw):
    from proteus_attention import KVPages, paged_attention

    pages = KVPages(**{m: t.to(DEV) for m, t in pool.items()})
    return paged_attention(q.to(DEV), pages, table.to(DEV), lengths.to(DEV), **kw).cpu()


@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_a_value_that_weighs_nothing(pair, form):
    """0 * inf is NaN: the channel is not finite, the others and the other heads are
    what they are without it."""
    dt, cell = pair
    B, n, low = FORMS[form]
    for D in (16, 64):
        g = torch.Generator().manual_seed(form)
        pool, table, q, lengths = _case(pair, B, n, low, D, g)
        want = R.attend(q, pool, table, lengths, scale=1.0)
        for bad in (math.inf, -math.inf, math.nan):
            b, t = B - 1, 17
            page, slot = int(table[b, t // 16]), t % 16
            channels = [5]
            if cell in R.TOP:
                channels = list(range(D))
                keep = pool["v_scale"][page, 0, slot].clone()
                pool["v_scale"][page, 0, slot] = bad
            else:
                keep = pool["v"][page, 0, slot, 5].clone()
                pool["v"][page, 0, slot, 5] = bad
            got = _run(q, pool, table, lengths, scale=1.0)
            if cell in R.TOP:
                pool["v_scale"][page, 0, slot] = keep
            else:
                pool["v"][page, 0, slot, 5] = keep
            assert not torch.isfinite(got[b, :2, channels]).any(), (D, bad)
            got[b, :2, channels] = want[0][b, :2, channels].to(dt)
            assert R.attend_error(got, want, dt, n) <= 1, (D, bad)


@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_a_key_that_is_not_finite(pair, form):
    """A score that is NaN or +inf leaves its rows NaN, wherever it lies."""
    dt, cell = pair
    B, n, low = FORMS[form]
    D = 64
    g = torch.Generator().manual_seed(form + 10)
    pool, table, q, lengths = _case(pair, B, n, low, D, g)
    want = R.attend(q, pool, table, lengths, scale=1.0)
    page = int(table[0, 1])
    for bad in (math.nan,) if cell in R.TOP else (math.nan, math.inf):
        if cell in R.TOP:
            pool["k_scale"][page, 1, 3] = bad
        else:
            pool["k"][page, 1, 3, 7] = bad
        got = _run(q, pool, table, lengths, scale=1.0)
        assert torch.isnan(got[0, 2:]).all(), bad
        got[0, 2:] = want[0][0, 2:].to(dt)
        assert R.attend_error(got, want, dt, n) <= 1, bad


@pytest.mark.parametrize("pair", R.PAIRS, ids=R.pair_id)
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_scores_of_minus_infinity(pair, form):
    """Rows with no score above -inf are zero, whatever their values are; next to
    other scores a score of -inf weighs nothing.  Queries of -inf on keys above
    zero, and, in float cells, keys of -inf."""
    dt, cell = pair
    B, n, low = FORMS[form]
    D = 32
    g = torch.Generator().manual_seed(form + 20)
    pool, table, q, lengths = _case(pair, B, n, 0, D, g)  # every key 4
    want = R.attend(q, pool, table, lengths, scale=1.0)
    minus = q.clone()
    minus[0, 1, 3] = -math.inf
    page = int(table[0, 0])
    if cell in R.TOP:
        pool["v_scale"][page, 0, 2] = math.nan
    else:
        pool["v"][page, 0, 2] = math.nan
    got = _run(minus, pool, table, lengths, scale=1.0)
    assert not got[0, 1].any()
    assert not torch.isfinite(got[0, 0]).any()
    got[0, :2] = want[0][0, :2].to(dt)
    assert R.attend_error(got, want, dt, n) <= 1
    if cell in R.TOP:
        return
    pool["v"][page, 0, 2] = 1.0
    at = table.long()
    P = at.shape[1]
    half = max(P // 2, 1)
    pool["k"][at[:, :half], 1, :, 9] = -math.inf  # the first half of each sequence, head 1
    pool["k"][at[0], 0, :, 9] = -math.inf  # all of the first one's, head 0
    got = _run(q, pool, table, lengths, scale=1.0)
    assert not got[0, :2].any()
    ref = R.attend(q[:, 2:], {m: t[:, 1:] for m, t in pool.items()}, table, lengths, starts=[half * 16] * B, scale=1.0)
    assert R.attend_error(got[:, 2:], ref, dt, n) <= 1
