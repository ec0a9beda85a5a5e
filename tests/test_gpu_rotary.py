"""Rotary positions on the GPU against 64 bits on the CPU.

Bound of a value y = m (a cos - b sin): half a step of the result's type, and in
f32 the angle's rounding (pi / 4 at most, 2^-24 of it), three roundings of 2^-24 or
less in the sine's and cosine's polynomials, the magnitude's, and those of the
products and their sum: 6 * 2^-24 m (|a| + |b|) hold them all.  The angle itself is
exact, which its reference is in whole numbers."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def turned(x, positions, rotary):
    """x (B, n, H, D) at positions (B, n), in 64 bits, and the bound of its error."""
    turns = [t % (1 << 64) for t in rotary.turns.tolist()]
    width, m = 2 * len(turns), torch.tensor(rotary.magnitude, dtype=torch.float32).item()
    part = torch.tensor([[[(p * t) % (1 << 64) / 2.0 ** 64 for t in turns] for p in row] for row in positions.tolist()],
                        dtype=torch.float64).view(*positions.shape, width // 2)
    angle = (2 * math.pi * part)[:, :, None]
    c, s = angle.cos() * m, angle.sin() * m
    at = (slice(0, width, 2), slice(1, width, 2)) if rotary.interleaved else (slice(0, width // 2), slice(width // 2, width))
    y, x = x.double().clone(), x.double()
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    size = torch.zeros_like(x)
    size[..., at[0]] = size[..., at[1]] = m * (a.abs() + b.abs())
    return y, size


def holds(got, x, positions, rotary):
    y, size = turned(x, positions, rotary)
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * y.abs() + 6 * 2.0 ** -24 * size + info.tiny * info.eps / 2
    return got.shape == x.shape and got.dtype == x.dtype and bool(((got.cpu().double() - y).abs() <= bound).all())


SHAPES = [
    # B, n, H, Hk, D, width
    (1, 1, 1, 1, 64, 64),
    (1, 1, 8, 8, 64, 64),
    (3, 1, 32, 8, 128, 128),
    (2, 37, 4, 1, 128, 64),
    (1, 300, 3, 2, 16, 16),
    (2, 17, 5, 5, 32, 16),
    (2, 9, 2, 1, 80, 80),
    (1, 5, 7, 1, 96, 32),
    (2, 3, 3, 1, 50, 50),
    (1, 4, 2, 2, 33, 30),
    (2, 6, 1, 1, 2, 2),
    (1, 3, 40, 1, 256, 256),
    (1, 2, 3, 200, 255, 6),
    (1, 700, 1, 1, 24, 8),
]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(dt, interleaved):
    from proteus_attention import apply_rotary, new_rotary_positions

    g = torch.Generator().manual_seed(0)
    for B, n, H, Hk, D, width in SHAPES:
        rotary = new_rotary_positions(width, interleaved=interleaved, magnitude=1.25, device=DEV)
        q, k = torch.randn(B, n, H, D, generator=g).to(dt), torch.randn(B, n, Hk, D, generator=g).to(dt)
        first = torch.randint(0, 5000, (B,), generator=g, dtype=torch.int32)
        every = first[:, None] + torch.arange(n, dtype=torch.int32)
        q1, k1 = apply_rotary(q.to(DEV), k.to(DEV), first.to(DEV), rotary)
        assert holds(q1, q, every, rotary) and holds(k1, k, every, rotary), (B, n, H, Hk, D, width)
        # every token's position given; queries alone; in place
        q2, none = apply_rotary(q.to(DEV), None, every.to(DEV), rotary)
        assert none is None and torch.equal(q1, q2), (B, n, H, D, width)
        q3, k3 = q.to(DEV), k.to(DEV)
        q4, k4 = apply_rotary(q3, k3, first.to(DEV), rotary, inplace=True)
        assert q4 is q3 and k4 is k3 and torch.equal(q3, q1) and torch.equal(k3, k1), (B, n, H, D, width)
        if n == 1:
            q5, k5 = apply_rotary(q[:, 0].to(DEV), k[:, 0].to(DEV), first.to(DEV), rotary)
            assert torch.equal(q5, q1[:, 0]) and torch.equal(k5, k1[:, 0])


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_far_positions(dt):
    """Angles of millions of turns, the ends of 32 bits and positions below zero."""
    from proteus_attention import apply_rotary, new_rotary_positions

    g = torch.Generator().manual_seed(1)
    pos = torch.tensor([[0, 1, 2 ** 20 + 1, 2 ** 31 - 1], [-1, -2 ** 31, 123456789, -777777]], dtype=torch.int32)
    for kw in (dict(), dict(interleaved=True, scaling="yarn", factor=40.0, trained=4096), dict(scaling="linear", factor=3.0),
               dict(scaling="ntk", factor=16.0), dict(base=500000.0)):
        rotary = new_rotary_positions(128, device=DEV, **kw)
        q = torch.randn(2, 4, 2, 128, generator=g).to(dt)
        assert holds(apply_rotary(q.to(DEV), None, pos.to(DEV), rotary)[0], q, pos, rotary), kw
    # a first position from which the tokens leave 32 bits
    rotary, q = new_rotary_positions(64, device=DEV), torch.randn(1, 3, 1, 64, generator=g).to(dt)
    got = apply_rotary(q.to(DEV), None, pos[0, 3:].to(DEV), rotary)[0]
    assert holds(got, q, pos[:1, 3:].long() + torch.arange(3), rotary)


def test_sines_of_an_octant_and_its_borders():
    """One pair, a turn in 2^20 steps: every octant and its ends."""
    from proteus_attention import RotaryPositions, apply_rotary

    n = 1 << 20
    rotary = RotaryPositions(torch.tensor([1 << 44], dtype=torch.int64, device=DEV))
    x = torch.tensor([1.0, 0.0]).expand(1, n, 1, 2)
    got = apply_rotary(x.to(DEV), None, torch.zeros(1, dtype=torch.int32, device=DEV), rotary)[0].cpu().double()[0, :, 0]
    angle = 2 * math.pi * torch.arange(n, dtype=torch.float64) / n
    want = torch.stack([angle.cos(), angle.sin()], -1)
    # the rounding of the angle and three of the polynomial, relative to the value near
    # the axes, where the reference's own angle is off by 2^-52 at most
    assert float((got - want).abs().max()) <= 4 * 2.0 ** -24
    small = want.abs() < 0.5
    assert float(((got - want).abs()[small] / (want.abs()[small] + 2.0 ** -26)).max()) <= 4 * 2.0 ** -24
    assert got[0].tolist() == [1, 0] and got[n // 4].tolist() == [0, 1] and got[n // 2].tolist() == [-1, 0]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(dt, interleaved):
    """Slices of a projection's output (in place too, its values left alone), rows off a
    16-byte line, heads first, expanded and transposed inputs, strided positions."""
    from proteus_attention import apply_rotary, new_rotary_positions

    g = torch.Generator().manual_seed(2)
    B, n, H, Hk, D = 2, 21, 6, 2, 64
    rotary = new_rotary_positions(32, interleaved=interleaved, device=DEV)
    qkv = torch.randn(B, n, H + 2 * Hk, D, generator=g).to(dt)
    wide = torch.zeros(B, 3, dtype=torch.int32)
    wide[:, 1] = torch.tensor([5, 70])
    pos = wide[:, 1, None] + torch.arange(n, dtype=torch.int32)
    first = wide.to(DEV)[:, 1]
    columns = pos.t().contiguous().to(DEV).t()
    d = qkv.to(DEV)
    q, k = apply_rotary(d[:, :, :H], d[:, :, H:H + Hk], first, rotary)
    assert q.is_contiguous() and holds(q, qkv[:, :, :H], pos, rotary) and holds(k, qkv[:, :, H:H + Hk], pos, rotary)
    assert torch.equal(d.cpu(), qkv)
    apply_rotary(d[:, :, :H], d[:, :, H:H + Hk], columns, rotary, inplace=True)
    assert torch.equal(d[:, :, :H], q) and torch.equal(d[:, :, H:H + Hk], k)
    assert torch.equal(d[:, :, H + Hk:].cpu(), qkv[:, :, H + Hk:])
    odd = torch.empty(B, n, H, D + 1, dtype=dt, device=DEV)[..., 1:].copy_(qkv[:, :, :H])
    assert torch.equal(apply_rotary(odd, None, first, rotary)[0], q)
    apply_rotary(odd, None, first, rotary, inplace=True)
    assert torch.equal(odd, q)
    heads = qkv[:, :, :H].transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    assert torch.equal(apply_rotary(heads, None, first, rotary)[0], q)
    dims = qkv[:, :, :H].transpose(2, 3).contiguous().to(DEV).transpose(2, 3)
    assert torch.equal(apply_rotary(dims, None, first, rotary)[0], q)
    same = qkv[:, :, :1].to(DEV).expand(B, n, H, D)
    assert torch.equal(apply_rotary(same, None, first, rotary)[0], q[:, :, :1].expand(B, n, H, D))
    for x in (dims, same):
        with pytest.raises(ValueError):
            apply_rotary(x, None, first, rotary, inplace=True)
    # nothing to do
    assert apply_rotary(d[:0], None, first[:0], rotary)[0].shape == (0, n, H + 2 * Hk, D)
    assert apply_rotary(d[:, :0], None, first, rotary)[0].shape == (B, 0, H + 2 * Hk, D)


def test_values_that_are_not_finite_stay_in_their_pair():
    from proteus_attention import apply_rotary, new_rotary_positions

    rotary = new_rotary_positions(32, device=DEV)
    x = torch.ones(1, 2, 1, 64, device=DEV)
    x[0, 0, 0, 3], x[0, 1, 0, 40] = math.nan, math.inf
    y = apply_rotary(x, None, torch.zeros(1, dtype=torch.int32, device=DEV), rotary)[0].cpu()
    bad = ~torch.isfinite(y)
    assert bad.nonzero().tolist() == [[0, 0, 0, 3], [0, 0, 0, 19], [0, 1, 0, 40]] and y[0, 1, 0, 40] == math.inf


def test_captured_and_on_two_streams():
    from proteus_attention import apply_rotary, new_rotary_positions

    g = torch.Generator().manual_seed(3)
    rotary = new_rotary_positions(64, device=DEV)
    q, k = (torch.randn(4, 1, h, 64, generator=g).bfloat16().to(DEV) for h in (8, 2))
    pos = torch.tensor([3, 900, 0, 77], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apply_rotary(q, k, pos, rotary)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = apply_rotary(q, k, pos, rotary)
    for _ in range(4):
        pos += 1
        q.neg_()
        want = apply_rotary(q, k, pos, rotary)
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    want = apply_rotary(q, k, pos, rotary)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(apply_rotary(q, k, pos, rotary))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x in got for a, b in zip(x, want))


def test_offsets_beyond_32_bits():
    """Rows of a tensor of more than 2^32 elements, in place: the others stay as they are."""
    from proteus_attention import apply_rotary, new_rotary_positions

    g = torch.Generator().manual_seed(12)
    B, n, H, D, apart = 3, 5, 2, 64, (1 << 31) + 4096
    rotary = new_rotary_positions(D, device=DEV)
    far = torch.empty((B - 1) * apart + 4 * n * H * D, dtype=torch.float16, device=DEV)
    x = torch.randn(B, n, H, D, generator=g).half()
    rows = far.as_strided((B, n, H, D), (apart, 2 * H * D, D, 1))
    between = far.as_strided((B, n, H, D), (apart, 2 * H * D, D, 1), H * D)
    rows.copy_(x)
    between.fill_(7.0)
    positions = torch.tensor([5, 2 ** 31 - 9, -4], dtype=torch.int32)
    every = positions.long()[:, None] + torch.arange(n)
    out, _ = apply_rotary(rows, None, positions.to(DEV), rotary)
    assert holds(out, x, every, rotary)
    apply_rotary(rows, None, positions.to(DEV), rotary, inplace=True)
    assert torch.equal(rows, out) and bool((between == 7.0).all())
