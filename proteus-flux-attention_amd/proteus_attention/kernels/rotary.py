"""Rotary positions of new tokens' queries and keys.

The layer turns the heads of whole sequences itself.  A program that generates
turns the queries and keys of the tokens that it has just computed, by their
positions, before the keys go into their pages:

* :func:`new_rotary_positions` -- frequencies of the pairs of channels, plain or
  stretched for contexts that are longer than the trained ones;
* :func:`apply_rotary` -- queries and keys turned, prompts and single tokens.

Like the rest of the package this is the inference path: tensors that require a
gradient raise ``NotImplementedError``.  The reference turns whole heads of whole
sequences alone (models/aspa.py:590-618).
"""
from __future__ import annotations

import math
import struct
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from .. import _hip
from .paged_attn import _call, _device, _VALUE_TAG

WIDEST_HEAD = 256


class RotaryPositions(NamedTuple):
    """``turns``: ``(width / 2,)`` int64 on the device, what each pair of channels
    turns by from one position to the next, in 2^-64 of a turn (modulo 2^64);
    ``magnitude``: what turned channels are multiplied by; ``interleaved``: pairs
    are channels (2j, 2j + 1), else (j, j + width / 2)."""

    turns: torch.Tensor
    magnitude: float = 1.0
    interleaved: bool = False


def rotary_frequencies(width: int, *, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       trained: Optional[int] = None, slow: float = 1.0, fast: float = 32.0) -> Tuple[list, float]:
    """Radians a position of each of ``width / 2`` pairs, and the magnitude.

    Plain: ``base ** (-2j / width)``, 1.  ``scaling`` for contexts ``factor``
    times as long as the ``trained`` positions:

    * ``"linear"``: all frequencies divided by ``factor``;
    * ``"ntk"``: ``base`` times ``factor ** (width / (width - 2))``, which leaves
      the fastest pair and divides the slowest by ``factor``;
    * ``"yarn"``: pairs that turn more than ``fast`` times over the trained
      positions stay, those that turn less than ``slow`` times are divided by
      ``factor``, and those between go over linearly in j (its bounds rounded
      outwards); the magnitude is ``0.1 ln(factor) + 1``.
    """

    width = int(width)
    if width < 2 or width % 2 or width > WIDEST_HEAD:
        raise ValueError(f"width must be even, 2 to {WIDEST_HEAD} (got {width})")
    base, factor = float(base), float(factor)
    if not 1.0 < base < math.inf:
        raise ValueError("base must be above 1 and finite")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}: None, 'linear', 'ntk' or 'yarn'")
    if scaling is None and factor != 1.0:
        raise ValueError("factor needs a scaling")
    if not 1.0 <= factor < math.inf:
        raise ValueError("factor must be at least 1 and finite")
    pairs = width // 2
    if scaling == "ntk":
        if width < 4:
            raise ValueError("'ntk' needs a width of at least 4")
        base *= factor ** (width / (width - 2))
    plain = [base ** (-2 * j / width) for j in range(pairs)]
    if scaling == "linear":
        return [f / factor for f in plain], 1.0
    if scaling != "yarn":
        return plain, 1.0
    if trained is None or not 1 <= int(trained):
        raise ValueError("'yarn' needs the number of trained positions")
    if not 0.0 < slow < fast:
        raise ValueError("'yarn' needs 0 < slow < fast")

    def at(turns: float) -> float:  # the pair, as a real number, that turns so often over the trained positions
        return width * math.log(int(trained) / (2 * math.pi * turns)) / (2 * math.log(base))

    low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), width - 1)
    ramp = [min(max((j - low) / max(high - low, 0.001), 0.0), 1.0) for j in range(pairs)]
    return [f * (1 - r) + f / factor * r for f, r in zip(plain, ramp)], 0.1 * math.log(factor) + 1.0


def new_rotary_positions(width: int, *, base: float = 10000.0, interleaved: bool = False, scaling: Optional[str] = None,
                         factor: float = 1.0, trained: Optional[int] = None,
                         frequencies: Union[None, Sequence[float], torch.Tensor] = None,
                         magnitude: Optional[float] = None, device="cuda") -> RotaryPositions:
    """Positions for the first ``width`` channels of a head, by
    :func:`rotary_frequencies`, or with ``frequencies`` of the caller's own
    (radians a position, ``width / 2`` of them); ``magnitude`` overrides theirs."""

    if frequencies is None:
        radians, length = rotary_frequencies(width, base=base, scaling=scaling, factor=factor, trained=trained)
    else:
        if scaling is not None or factor != 1.0:
            raise ValueError("frequencies of the caller's own are scaled by the caller")
        radians = frequencies.double().cpu().tolist() if isinstance(frequencies, torch.Tensor) else [float(f) for f in frequencies]
        length = 1.0
        if int(width) % 2 or not 2 <= int(width) <= WIDEST_HEAD or len(radians) != int(width) // 2:
            raise ValueError(f"a width of 2 to {WIDEST_HEAD} needs width / 2 frequencies (got {width}, {len(radians)})")
        if not all(math.isfinite(f) for f in radians):
            raise ValueError("frequencies must be finite")
    length = length if magnitude is None else float(magnitude)
    if not 0.0 < length < math.inf:
        raise ValueError("magnitude must be positive and finite")
    # a frequency is a whole number of 2^-64 turns: what a double's radians leave, off by 2^-53 of it and half a unit
    turns = [round(math.fmod(f / (2 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64) for f in radians]
    turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64, device=device)
    return RotaryPositions(turns, length, bool(interleaved))


_CALL = struct.Struct("PqqqPqqqPqqqPqqqPPqqqiiiiiiiif4x")  # pfa_rotary_call of include/pfa_hip.h
_NONE = (0, 0, 0, 0)


def _sides(x: torch.Tensor, inplace: bool) -> Tuple[torch.Tensor, torch.Tensor, tuple, tuple]:
    """x with a dense last dimension, the result, and the library's descriptions of both."""

    shape, s = x.shape, x.stride()
    if s[-1] != 1 and shape[-1] > 1:
        x = x.contiguous()
        s = x.stride()
    many = len(shape) == 4
    source = (x.data_ptr(), s[0], s[2], s[1]) if many else (x.data_ptr(), s[0], s[1], 0)
    if inplace:
        return x, x, source, source
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    s = y.stride()
    return x, y, source, (y.data_ptr(), s[0], s[2], s[1]) if many else (y.data_ptr(), s[0], s[1], 0)


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: RotaryPositions, *,
                 inplace: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Queries ``q`` ``(B, n, heads, head_dim)`` and keys ``k`` ``(B, n, kv_heads,
    head_dim)`` (or None) of n new tokens a sequence, turned by their positions;
    without the n, of one.  f32, bf16 or f16, any strides with a dense last
    dimension.  ``positions`` int32 on the device: ``(B,)``, each sequence's
    first, or ``(B, n)``, every token's; any values of 32 bits.

    The first ``width`` channels of a head turn, the others stay.  Angles are
    exact at any position, products f32, rounded once at the end.  Returns
    contiguous tensors in the inputs' type, or with ``inplace`` the inputs,
    written over: their rows must not overlap, and q and k not be the same.
    """

    turns, magnitude, interleaved = rotary
    shape, dtype = q.shape, q.dtype
    if len(shape) == 4:
        B, n, H, D = shape
    elif len(shape) == 3:
        (B, H, D), n = shape, 1
    else:
        raise ValueError("q must be (B, n, heads, head_dim), or (B, heads, head_dim): one new token a sequence")
    tag = _VALUE_TAG.get(dtype)
    if tag is None:
        raise ValueError(f"unsupported value dtype {dtype}")
    width = 2 * turns.numel()
    if turns.dtype != torch.int64 or turns.dim() != 1 or width == 0 or not turns.is_contiguous():
        raise ValueError("turns must be a contiguous (width / 2,) int64 tensor")
    if not 0 < D <= WIDEST_HEAD or width > D or H == 0:
        raise ValueError(f"q has {H} heads of {D} channels for {width} that turn: up to {WIDEST_HEAD}, and a head at least")
    Hk = 0
    if k is not None:
        other = k.shape
        Hk = other[-2] if len(other) == len(shape) else 0
        if k.dtype != dtype or Hk == 0 or other[:-2] != shape[:-2] or other[-1] != D:
            raise ValueError(f"k must be {tuple(shape[:-2])} x kv_heads x {D} of {dtype} (got {tuple(other)}, {k.dtype})")
    at = positions.shape
    if positions.dtype != torch.int32 or (at != (B,) and at != (B, n)):
        raise ValueError(f"positions must be a ({B},) or ({B}, {n}) int32 tensor")
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
        raise NotImplementedError("apply_rotary has no backward pass: call it under torch.no_grad()")
    if inplace:
        for x in (q, k) if Hk else (q,):
            if x.stride(-1) != 1 and D > 1:
                raise ValueError("inplace needs a dense last dimension")
            if any(stride == 0 and size > 1 for stride, size in zip(x.stride(), x.shape)):
                raise ValueError("inplace needs rows of their own: an expanded tensor has none")
        if Hk and q.data_ptr() == k.data_ptr() and q.numel():
            raise ValueError("inplace needs q and k apart: one tensor would be turned twice")
    index = _device("apply_rotary", q, k, positions, turns)
    pos = positions.stride()
    q, q_out, q_from, q_to = _sides(q, inplace)
    k_out, k_from, k_to = None, _NONE, _NONE
    if Hk:
        k, k_out, k_from, k_to = _sides(k, inplace)
    per_token = len(pos) == 2
    packed = _CALL.pack(*q_from, *k_from, *q_to, *k_to, turns.data_ptr(), positions.data_ptr(), pos[0],
                        pos[1] if per_token else 0, n, per_token, B, H, Hk, D, width, interleaved, tag, magnitude)
    _call(index, "rotary", _hip.lib().pfa_rotary, packed)
    return q_out, k_out


__all__ = ["RotaryPositions", "new_rotary_positions", "rotary_frequencies", "apply_rotary"]
