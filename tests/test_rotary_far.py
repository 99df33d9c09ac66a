"""Rotary angles at far positions: the table of frequencies to its last bit, and the rotation by positions that a
double angle does not resolve, against integers and rational arithmetic."""
from fractions import Fraction

import pytest
import torch

DIGITS = 60


def _root(base: Fraction, n: int) -> int:
    """floor(base^(-1/n) * 10^DIGITS), by bisection over integers."""
    scale = 10 ** DIGITS
    lo, hi = 0, scale
    while hi - lo > 1:  # x^n * base < 1
        mid = (lo + hi) // 2
        if mid ** n * base.numerator < scale ** n * base.denominator:
            lo = mid
        else:
            hi = mid
    return lo


def _two_pi() -> Fraction:
    """2 pi = 32 atan(1/5) - 8 atan(1/239), the series to 10^-70."""
    def atan(n):
        total, k = Fraction(0), 0
        while n ** (2 * k + 1) < 10 ** 70:
            total += Fraction((-1) ** k, (2 * k + 1) * n ** (2 * k + 1))
            k += 1
        return total
    return 32 * atan(5) - 8 * atan(239)


def _fractions_of_a_turn(half, base):
    """base^(-i / half) / 2 pi, rational, to 10^-50 or better."""
    step, two_pi = Fraction(_root(Fraction(base), half), 10 ** DIGITS), _two_pi()
    out, f = [], Fraction(1)
    for _ in range(half):
        out.append(f / two_pi)
        f = Fraction(int(f * step * 10 ** 58), 10 ** 58)
    return out


@pytest.mark.parametrize("half,base", [(16, 10000.0), (32, 500000.0), (64, 1e6), (128, 10000.0), (32, 1.5)])
def test_table_is_the_rounded_frequency(half, base):
    from embodied_efficiency_b200.prompt import _turn_fractions
    for have, want in zip(_turn_fractions(half, base), _fractions_of_a_turn(half, base)):
        assert 0 < have < 2 ** 63 and abs(have - want * 2 ** 64) <= Fraction(1, 2) + Fraction(1, 10 ** 20)


def test_table_in_another_decimal_context():
    import decimal
    from embodied_efficiency_b200.prompt import _turn_fractions
    want = _turn_fractions(16, 10000.0)
    with decimal.localcontext(decimal.Context(prec=5, rounding=decimal.ROUND_UP, traps=[decimal.Inexact])):
        assert _turn_fractions(16, 10000.0) == want


@pytest.mark.gpu
@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(cuda, base, interleaved):
    """Half a step of the result, and an angle that is off by 2^-25 turns (the table's 2^40 * 2^-65) and the fp32
    value of a half turn (2^-25 half turns), 2^-25 * 3 pi < 2^-21, with the sine's two ulps (2^-22) below 2^-20 of
    |a| + |b|. Elements where the sum nearly cancels show the angle alone."""
    from embodied_efficiency_b200 import rotary_embed
    hd, half = 64, 32
    places = [1 << 31, (1 << 31) - 1, -(1 << 31), 1 << 36, (1 << 40) - 12345, 1 << 40, -(1 << 40), 987654321012]
    turns = _fractions_of_a_turn(half, base)
    angle = torch.tensor([[float((p * f) % 1) for f in turns] for p in places], device=cuda,
                         dtype=torch.float64)[:, None] * (2 * torch.pi)
    q = torch.randn(len(places), 200, hd, generator=torch.Generator(device=cuda).manual_seed(3), device=cuda).half()
    out, _ = rotary_embed(q, None, torch.tensor(places, device=cuda), (half,), base=base, interleaved=interleaved)

    def pairs(x):
        return (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])

    a, b = pairs(q.double())
    mag = a.abs() + b.abs()
    for have, ref in zip(pairs(out.double()), (a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos())):
        tol = 2 ** -11 * ref.abs() * (1 + 2 ** -10) + mag * 2 ** -20 + 2 ** -25
        assert bool(((have - ref).abs() <= tol).all()), float(((have - ref).abs() / tol).max())
