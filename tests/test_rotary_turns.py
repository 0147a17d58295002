"""The turns that `rotary` makes of frequencies, and angles at far coordinates, against the frequencies themselves with pi to 60 digits."""
import math
import random
from decimal import Decimal, localcontext
from fractions import Fraction

import pytest
import torch

TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494")


def off_by(turns, exact):
    """Distance of int64 `turns` from `exact` times 2^64, modulo whole turns, in units of 2^-64 of a turn."""
    d = (turns - exact * 2**64) % 2**64
    return min(d, 2**64 - d)


def spectra():
    r = random.Random(5)
    yield [10000.0 ** (-j / 64) for j in range(64)]
    yield [500000.0 ** (-j / 64) for j in range(64)]
    yield [r.uniform(-1, 1) * 10.0 ** r.uniform(-12, 6) for _ in range(64)]
    yield [2 * math.pi * r.randint(-40, 40) / 8 for _ in range(64)]  # whole eighths, of that pi


@pytest.mark.parametrize("frequencies", list(spectra()))
def test_turns_are_those_of_the_frequencies(frequencies):
    """A quotient of doubles is off by 2^-53 of itself, and for pi rounded by 2^-54.5: less than 2^-52 with both.  What is cut off is less than 2^-64 of a turn."""
    import flex_block_attn_amd as fba

    for x, f in zip(fba.rotary(frequencies=frequencies, device="cpu").turns.tolist(), frequencies):
        exact = Fraction(f) / TWO_PI
        assert off_by(x, exact) <= abs(exact) * 2**64 / 2**52 + 1


@pytest.mark.parametrize("theta,dims", [(10000.0, (128,)), (256.0, (16, 56, 56)), (500000.0, (128,)), (3.7, (44, 42, 42))])
def test_turns_are_those_of_theta(theta, dims):
    """The frequency's own rounding comes on top: 2^-53 of the exponent, and 2^-52 for the power."""
    import flex_block_attn_amd as fba

    with localcontext() as context:
        context.prec = 60
        powers = [(Decimal(theta).ln() * (-2 * j) / d, j, d) for d in dims for j in range(d // 2)]
        exact = [Fraction(x.exp()) / TWO_PI for x, _, _ in powers]
    for x, e, (log, _, _) in zip(fba.rotary(dims, theta=theta, device="cpu").turns.tolist(), exact, powers):
        assert off_by(x, e) <= e * 2**64 * (Fraction(2) / 2**52 + Fraction(abs(log)) / 2**53) * (1 + Fraction(1, 2**40)) + 1


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_angles_are_those_of_the_frequencies(gpu, interleaved):
    """(1, 0) turned is (cos, sin).  Angles may be off by 2^-52 |c| frequency and what cutting off makes, 2 pi 2^-64 |c|; the kernel's sines by 2^-21; fp16 rounds by 2^-11 of the value, or by
    2^-25 where it is small."""
    import flex_block_attn_amd as fba

    where = [0, 1, -1, 115199, -2**20, 10**9, 2**31 - 1, -2**31, 1234567890]
    at = torch.tensor(where, dtype=torch.int32, device=gpu)[:, None]
    for frequencies in spectra():
        turn = fba.rotary(frequencies=frequencies, interleaved=interleaved, device=gpu)
        x = torch.zeros((1, 1, len(where), 128), dtype=torch.float16, device=gpu)
        first = slice(0, 128, 2) if interleaved else slice(0, 64)
        second = slice(1, 128, 2) if interleaved else slice(64, 128)
        x[..., first] = 1.0
        got = fba.rotary_func(x, None, turn, coordinates=at)[0][0, 0].double().cpu()
        for i, c in enumerate(where):
            for j, f in enumerate(frequencies):
                part = Fraction(f) * c / TWO_PI
                angle = float((part - math.floor(part + Fraction(1, 2))) * TWO_PI)  # half a turn at most, and off by 2^-53 of itself
                off = 2.0**-52 * abs(c * f) + 2.0**-61 * abs(c) + 2.0**-21 + 2.0**-51
                for value, want in ((got[i, first][j], math.cos(angle)), (got[i, second][j], math.sin(angle))):
                    assert abs(float(value) - want) <= off + 2.0**-11 * (abs(want) + off) + 2.0**-25, (c, f)
