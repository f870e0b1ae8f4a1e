"""Rotary positions with one or several axes (time, height, width), for queries and keys before any of the attention operators.

Of every head the first ``rotary_dim`` values are pairs (x1, x2), each of which belongs to one axis and has a frequency; a pair is
turned by w = frequency * position on its axis:

    y1 = x1 cos(w) - x2 sin(w),        y2 = x2 cos(w) + x1 sin(w)

The reference has no counterpart (its cells know positions by ``alibi`` only).
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib, _traced

__all__ = ["Rotary"]

MAX_HEAD_DIM = 256


@functools.lru_cache(maxsize=8)
def _two_pi(bits):
    """2 pi times 2^bits, off by less than one (Machin: pi / 4 = 4 atan(1/5) - atan(1/239))."""
    guard = 32

    def atan_inverse(n):      # atan(1 / n), its series, truncated term by term
        power = (1 << (bits + guard)) // n
        total, k = power, 1
        while power:
            power //= n * n
            total += (-power if k % 2 else power) // (2 * k + 1)
            k += 1
        return total
    return (8 * (4 * atan_inverse(5) - atan_inverse(239))) >> guard


def turns_of(frequency):
    """Turns per position modulo one, in units of 2^-64, nearest to frequency / 2 pi as it is, as a signed 64-bit number."""
    numerator, denominator = float(frequency).as_integer_ratio()
    bits = 96 + max(0, numerator.bit_length() - denominator.bit_length())      # (what a large frequency multiplies)
    period = denominator * _two_pi(bits)
    turns = ((numerator << (64 + bits)) + period // 2) // period % 2 ** 64
    return turns - 2 ** 64 if turns >= 2 ** 63 else turns


class Rotary:
    """The plan of a model's rotary positions.

    ``sections``: how many pairs belong to each axis, the first pairs to the first axis and so on (default: all to one axis); their
    sum is half of ``rotary_dim``, the values behind which are left as they are.  Frequencies are ``base ** (-i / pairs)``: i counts
    through all axes' pairs, or with ``per_axis`` anew for every axis among the pairs of that axis.  ``frequencies`` (radians per
    position, one for each pair) takes their place.  A pair is values i and i + rotary_dim / 2, with ``adjacent`` 2 i and 2 i + 1.

        rotary = Rotary(128, (16, 24, 24))
        q, k = rotary(q, k, positions)          # [T, heads, D] with positions [3, T], or [B, heads, S, D] with [3, B, S] or [3, S]
        rotary.apply_(q, k, positions)          # in place, for serving
    """

    def __init__(self, head_dim, sections=None, *, base=10000.0, per_axis=False, adjacent=False, frequencies=None, device="cuda"):
        if head_dim < 8 or head_dim > MAX_HEAD_DIM or head_dim % 8:
            raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}, got {head_dim}")
        sections = (head_dim // 2,) if sections is None else tuple(int(n) for n in sections)
        pairs = sum(sections)
        if not sections or min(sections) < 0 or pairs < 1 or 2 * pairs > head_dim:
            raise ValueError(f"sections must be numbers of pairs, 1 to {head_dim // 2} in all, got {sections}")
        if frequencies is None:
            if not (base > 0 and math.isfinite(base)):
                raise ValueError(f"base must be a positive number, got {base}")
            if per_axis:
                frequencies = [float(base) ** (-i / n) for n in sections for i in range(n)]
            else:
                frequencies = [float(base) ** (-i / pairs) for i in range(pairs)]
        else:
            frequencies = [float(f) for f in frequencies]
            if len(frequencies) != pairs or not all(math.isfinite(f) for f in frequencies):
                raise ValueError(f"frequencies must be {pairs} finite numbers, one for each pair")
        self.head_dim, self.rotary_dim, self.sections, self.adjacent = head_dim, 2 * pairs, sections, bool(adjacent)
        turns = [turns_of(f) for f in frequencies]
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
        self.turns = torch.tensor(turns, dtype=torch.int64, device=device)
        self.axis = torch.tensor(axis, dtype=torch.int32, device=device)
        if not self.turns.is_cuda:
            raise ValueError("the plan must be on a CUDA device (this library has no CPU path)")
        self._plan = (head_dim, 2 * pairs, len(sections), int(self.adjacent))

    def __call__(self, q, k, positions):
        """(q, k) turned, as new tensors; differentiable in both, either may be None.  ``positions``: integers of up to 64 bits, [axes, T] for rows
        [T, heads, D], [axes, B, S] or [axes, S] for [B, heads, S, D]; with one axis that dimension may be missing."""
        out = _lib.host().rotary(q, k, positions, self.turns, self.axis, self._plan, False)
        return self._recorded(q, k, positions) if out is None else out

    def apply_(self, q, k, positions):
        """The same in place, without a gradient; rows must be contiguous, and addresses and strides whole 16 bytes."""
        return _lib.host().rotary(q, k, positions, self.turns, self.axis, self._plan, True)

    def _recorded(self, q, k, positions):
        out = list(_traced.call(self._defined, q, k, positions))
        return tuple(None if x is None else out.pop(0) for x in (q, k))

    def _defined(self, q, k, positions):
        return tuple(x for x in _lib.host().rotary(q, k, positions, self.turns, self.axis, self._plan, False) if x is not None)
