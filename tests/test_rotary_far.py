"""Rotary positions far out: the angle is that of the frequency as it was given, whatever the position.

The reference takes position * frequency / 2 pi modulo one in whole numbers, with 64 bits more than the plan's table.  Tolerance as in
test_rotary.py: sine and cosine off by 2^-22, three operations in fp32, one rounding: u |y| + 2^-21 (|x1| + |x2|); the table adds position * 2^-65
turns, 2 pi 2^-65 |position| (|x1| + |x2|)."""
import math

import pytest
import torch

from tests.test_rotary_turns_cpu import PI

pytestmark = pytest.mark.gpu


def _angles(positions, f):
    """[rows] in float64, in [0, 2 pi)"""
    num, den = f.as_integer_ratio()
    turn = num * PI.denominator * 2 ** 128 // (den * 2 * PI.numerator)
    return torch.tensor([(p * turn % 2 ** 128) / 2 ** 128 for p in positions.tolist()], dtype=torch.float64, device="cuda") * (2 * math.pi)


def _check(positions, frequencies, dtype=torch.float16):
    from acctransformer_b200 import Rotary
    D, T = 8 * ((2 * len(frequencies) + 7) // 8), positions.numel()
    x = torch.randn(T, 1, D, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dtype)
    y = Rotary(D, (len(frequencies),), frequencies=frequencies)(x, None, positions)[0].double()
    pairs, far, x = len(frequencies), positions.abs().max().item(), x.double()
    for i, f in enumerate(frequencies):
        w = _angles(positions, f)[:, None]
        a, b = x[..., i], x[..., i + pairs]
        most = (a.abs() + b.abs()) * (2.0 ** -21 + 2 * math.pi * far * 2.0 ** -65)
        for got, want in ((y[..., i], a * w.cos() - b * w.sin()), (y[..., i + pairs], b * w.cos() + a * w.sin())):
            bound = torch.finfo(dtype).eps / 2 * want.abs() + most + torch.finfo(dtype).tiny
            worst = ((got - want).abs() / bound).max().item()
            assert worst <= 1, f"frequency {f}: off by {worst:.1f} of the bound"


@pytest.mark.parametrize("around", [0, 1 << 20, 2 ** 31 - 30001, -2 ** 31])
def test_positions_of_32_bits(around):
    _check(torch.arange(30000, device="cuda", dtype=torch.int32) + around, [1.0, 100.0, 12345.678, 10000.0 ** (-5 / 64)])
