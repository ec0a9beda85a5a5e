"""Rotary positions on the CPU: frequencies against their formulas, refusals in Python
and at the C entry; no kernel runs."""
from __future__ import annotations

import ctypes
import math
import struct

import pytest
import torch

from proteus_attention import RotaryPositions, _hip, apply_rotary, new_rotary_positions, rotary_frequencies


def test_plain_linear_and_ntk():
    for width in (2, 4, 16, 64, 128, 256):
        plain, m = rotary_frequencies(width, base=5000.0)
        assert m == 1.0 and len(plain) == width // 2 and plain[0] == 1.0
        assert all(math.isclose(f, 5000.0 ** (-2 * j / width), rel_tol=1e-14) for j, f in enumerate(plain))
        linear, m = rotary_frequencies(width, base=5000.0, scaling="linear", factor=8.0)
        assert m == 1.0 and linear == [f / 8.0 for f in plain]
        if width >= 4:
            ntk, m = rotary_frequencies(width, base=5000.0, scaling="ntk", factor=8.0)
            assert m == 1.0 and ntk[0] == plain[0] and math.isclose(ntk[-1], plain[-1] / 8.0, rel_tol=1e-12)


def test_yarn_between_its_bounds():
    """64 channels, base 10000, 4096 positions: pair j turns 4096 * 10000^(-j / 32) / 2 pi
    times.  32 times at j = 10.47, once at j = 22.51: 10 and 23."""
    plain, _ = rotary_frequencies(64)
    yarn, m = rotary_frequencies(64, scaling="yarn", factor=4.0, trained=4096)
    assert math.isclose(m, 0.1 * math.log(4.0) + 1.0)
    for j, (a, b) in enumerate(zip(plain, yarn)):
        part = min(max((j - 10) / 13, 0.0), 1.0)
        assert math.isclose(b, a * (1 - part) + a / 4.0 * part, rel_tol=1e-14)
    assert yarn[:11] == plain[:11] and yarn[23:] == [f / 4.0 for f in plain[23:]]
    same, m = rotary_frequencies(64, scaling="yarn", factor=1.0, trained=4096)
    assert m == 1.0 and all(math.isclose(a, b, rel_tol=1e-15) for a, b in zip(plain, same))


def test_turns_hold_the_frequencies():
    """64 bits after the point: a frequency of up to a turn a position is off by 2^-53 of
    itself, a 64-bit float's rounding in the division by 2 pi, and 2^-65 of a turn."""
    own = [1.0, 0.3, 1e-9, 5.0, -0.25, 2 * math.pi * 3.5, 0.0, 123.456]
    rotary = new_rotary_positions(16, frequencies=own, magnitude=1.5, interleaved=True, device="cpu")
    assert rotary.magnitude == 1.5 and rotary.interleaved and rotary.turns.dtype == torch.int64
    for f, t in zip(own, rotary.turns.tolist()):
        got = (t % (1 << 64)) / 2.0 ** 64
        off = (got - f / (2 * math.pi)) % 1.0
        assert min(off, 1.0 - off) <= abs(f) * 2.0 ** -52 + 2.0 ** -60
    same = new_rotary_positions(64, device="cpu")
    given = new_rotary_positions(64, frequencies=torch.tensor(rotary_frequencies(64)[0], dtype=torch.float64), device="cpu")
    assert torch.equal(same.turns, given.turns) and same[1:] == given[1:] == (1.0, False)


@pytest.mark.parametrize("kw", [
    dict(width=0), dict(width=7), dict(width=258), dict(width=64, base=1.0), dict(width=64, base=math.inf),
    dict(width=64, factor=2.0), dict(width=64, scaling="linear", factor=0.5), dict(width=64, scaling="dynamic", factor=2.0),
    dict(width=64, scaling="yarn", factor=2.0), dict(width=64, scaling="yarn", factor=2.0, trained=0),
    dict(width=2, scaling="ntk", factor=2.0), dict(width=64, scaling="linear", factor=math.nan),
    dict(width=64, magnitude=0.0), dict(width=64, magnitude=math.inf), dict(width=4, frequencies=[1.0]),
    dict(width=4, frequencies=[1.0, math.nan]), dict(width=4, frequencies=[1.0, 0.5], scaling="linear", factor=2.0),
    dict(width=3, frequencies=[1.0]),
], ids=str)
def test_positions_that_are_not_made(kw):
    with pytest.raises(ValueError):
        new_rotary_positions(device="cpu", **kw)


ROT = new_rotary_positions(32, device="cpu")
Q, K = torch.zeros(2, 3, 4, 32), torch.zeros(2, 3, 2, 32)
POS = torch.zeros(2, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    lambda: apply_rotary(Q[0, 0], None, POS, ROT),
    lambda: apply_rotary(Q, K[:, 0], POS, ROT),
    lambda: apply_rotary(Q, K[:, :2], POS, ROT),
    lambda: apply_rotary(Q, K[:1], POS, ROT),
    lambda: apply_rotary(Q, K[..., :16], POS, ROT),
    lambda: apply_rotary(Q, K[:, :, :0], POS, ROT),
    lambda: apply_rotary(Q[:, :, :0], K, POS, ROT),
    lambda: apply_rotary(Q, K.half(), POS, ROT),
    lambda: apply_rotary(Q.double(), K.double(), POS, ROT),
    lambda: apply_rotary(Q[..., :30], None, POS, ROT),
    lambda: apply_rotary(torch.zeros(2, 3, 1, 300), None, POS, ROT),
    lambda: apply_rotary(Q, K, POS.long(), ROT),
    lambda: apply_rotary(Q, K, POS[:1], ROT),
    lambda: apply_rotary(Q, K, torch.zeros(2, 4, dtype=torch.int32), ROT),
    lambda: apply_rotary(Q, K, POS, ROT._replace(turns=ROT.turns.int())),
    lambda: apply_rotary(Q, K, POS, ROT._replace(turns=ROT.turns[:0])),
    lambda: apply_rotary(Q, K, POS, ROT._replace(turns=ROT.turns[::2])),
    lambda: apply_rotary(Q, Q, POS, ROT, inplace=True),
    lambda: apply_rotary(Q, Q[:, :, :2], POS, ROT, inplace=True),
    lambda: apply_rotary(Q[:, :, :1].expand(2, 3, 4, 32), None, POS, ROT, inplace=True),
])
def test_arguments_that_do_not_fit(call):
    with pytest.raises(ValueError):
        call()


def test_no_backward_and_no_cpu_path():
    for q, k in ((Q.clone().requires_grad_(), K), (Q, K.clone().requires_grad_())):
        with pytest.raises(NotImplementedError):
            apply_rotary(q, k, POS, ROT)
        with torch.no_grad(), pytest.raises(_hip.HipLibraryError):
            apply_rotary(q, k, POS, ROT)


def test_c_entry_refuses_before_any_launch():
    def call(H=2, Hk=1, D=64, width=64, B=1, n=3, dtype=0, magnitude=1.0, q=256, k=256, out=256, turns=256, pos=256):
        t4 = [64 * H, 64, 64]
        return _hip.lib().pfa_rotary(struct.pack("PqqqPqqqPqqqPqqqPPqqqiiiiiiiif4x", q, *t4, k, *t4, out, *t4, out, *t4,
                                                 turns, pos, 1, 0, n, 0, B, H, Hk, D, width, 0, dtype, magnitude), None)

    bad = [call(H=0), call(H=70000), call(Hk=-1), call(D=0), call(D=300, width=64), call(width=0), call(width=63),
           call(width=128), call(B=-1), call(B=70000), call(n=-1), call(n=1 << 31), call(dtype=3), call(dtype=9),
           call(magnitude=0.0), call(magnitude=math.nan), call(magnitude=math.inf), call(q=0), call(k=0), call(out=0),
           call(turns=0), call(pos=0), _hip.lib().pfa_rotary(ctypes.c_void_p(0), None)]
    assert bad == [-1] * len(bad)
    assert call(B=0) == 0 and call(n=0) == 0
