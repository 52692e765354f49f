"""Angles of far positions against frequencies and pi that are computed here, in decimal numbers and fractions.

A frequency is base ** (-2i / rotary_dim) held in 64 bits, its turns a position the quotient by 2 pi, rounded to 64 bits
again and then to the nearest 2^-64. The quotient is off by 2^-53 for its own rounding and 2^-54.5 for that of pi, so by 1.4
* 2^-53 of itself; the frequency f by the rounding of its exponent, which counts -ln(f) times, and by the power's, less than a
whole step: 2^-53 * (-ln(f) + 2) of itself. An angle is off by the position times that: for f of a radian a position or less,
f * (3.4 - ln(f)) is at most 3.4, so by less than 4e-16 radians a position.
"""

import math
from decimal import Decimal, localcontext
from fractions import Fraction

import pytest
import torch

from adaptive_sparse.append import append_rotary, make_rotary

FAR = 2 ** 30

def inverse_tangent(n, digits=60):
    """atan(1 / n) by its series."""
    total, power, k = Fraction(0), Fraction(1, n), 0
    while power > Fraction(1, 10 ** digits):
        total += power / (2 * k + 1) * (-1) ** k
        power, k = power / (n * n), k + 1
    return total


PI = 16 * inverse_tangent(5) - 4 * inverse_tangent(239)        # Machin's formula


def frequency(base, i, size):
    """base ** (-2i / size) in 50 digits."""
    with localcontext() as context:
        context.prec = 50
        return Fraction(Decimal(base) ** (Decimal(-2 * i) / Decimal(size)))


def off_by(f):
    """How far the turns of a pair of f radians a position may be off, of themselves, but for their last bit."""
    return Fraction(3.4 - math.log(f)) / 2 ** 53


def test_pi():
    assert abs(PI - Fraction("3.14159265358979323846264338327950288419716939937510")) < Fraction(1, 10 ** 49)


@pytest.mark.parametrize("size,base", [(2, 10000), (64, 10000), (128, 10000), (128, 500000), (256, 1000000)])
def test_turns_are_those_of_the_frequencies(size, base):
    rotary = make_rotary(size, device="cpu", base=float(base))
    for i, turn in enumerate(rotary.turns.tolist()):
        radians = frequency(base, i, size)
        want = radians / (2 * PI) * 2 ** 64
        off = (turn - want) % 2 ** 64
        off = min(off, 2 ** 64 - off)
        assert off <= want * off_by(radians) + Fraction(1, 2)
        assert off / 2 ** 64 * 2 * PI < Fraction(4, 10 ** 16)


@pytest.mark.parametrize("given", [
    dict(scaling="ramp", original=math.inf), dict(scaling="ramp", original=4096, fast=math.inf),
    dict(scaling="ramp", original=math.nan), dict(scaling="base", factor=1e308, base=1e300),
    dict(rotary_dim=4, scaling="base", factor=1e200), dict(rotary_dim=4, scaling="base", factor=1e-200),
    dict(rotary_dim=256, base=5e-324),
    dict(scaling="linear", factor=5e-324, base=0.5),
])
def test_frequencies_past_the_numbers_are_refused(given):
    with pytest.raises(ValueError):
        make_rotary(**{"rotary_dim": 64, "device": "cpu", **given})


@pytest.mark.gpu
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("base", [10000, 500000])
def test_far_positions_turn_by_their_frequencies(gpu, base, neighbours):
    size = 128
    rotary = make_rotary(size, device=gpu, base=float(base), interleaved=neighbours)
    positions = [0, 1, 1000003, FAR, FAR + 12345, 2 ** 31 - 2]
    query = torch.randn((len(positions), 3, size), generator=torch.Generator(device=gpu).manual_seed(base),
                        device=gpu).to(torch.float16)
    out = torch.empty_like(query)
    append_rotary(query, None, None, None, None, torch.tensor(positions, device=gpu), rotary, out)
    i = torch.arange(size // 2, device=gpu)
    a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + size // 2)
    m, n = query[..., a].double(), query[..., b].double()
    radians = [frequency(base, k, size) for k in range(size // 2)]
    angle = torch.tensor([[float(f * p % (2 * PI)) for f in radians] for p in positions], dtype=torch.float64, device=gpu)
    slack = torch.tensor([[float(p * (f * off_by(f) + PI / 2 ** 64)) for f in radians] for p in positions],
                         dtype=torch.float64, device=gpu)
    cos, sin, slack = (x.unsqueeze(1) for x in (angle.cos(), angle.sin(), slack))
    # The kernel's sine and cosine, of an angle of at most pi / 4 in 32 bits, are 2^-22 off, and products and sum in 32 bits
    # add less than 2^-22 of both elements.
    for got, want in ((out[..., a], m * cos - n * sin), (out[..., b], n * cos + m * sin)):
        bound = want.abs() * 2.0 ** -11 + (m.abs() + n.abs()) * (2.0 ** -21 + slack) + 2.0 ** -25
        assert bool(((got.double() - want).abs() <= bound).all())
