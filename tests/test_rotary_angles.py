"""Rotary angles against the formulas themselves: the frequencies of every
scaling, the fractions of a turn made of them, and what ``Rotary`` gives for its
arguments. (``rotary_oracle`` takes its angles from the table under test.)"""
import math
from fractions import Fraction

import pytest
import torch

from kotflash_amd.rotary import Rotary, rotary_frequencies
from tests.rotary_definition import PI, assert_definition, frequencies

SCALINGS = [dict(), dict(base=500000.0), dict(base=1.5), dict(scaling="linear", factor=4.0),
            dict(scaling="base", factor=8.0, base=1000.0), dict(scaling="linear", factor=1.0),
            dict(scaling="ramp", factor=4.0, original_length=4096),
            dict(scaling="ramp", factor=32.0, original_length=8192, slow_turns=0.0, fast_turns=32.0, base=500000.0)]


def test_pi():
    assert abs(float(PI) - math.pi) == 0 and abs(PI - Fraction(math.pi)) < Fraction(1, 2 ** 52)


@pytest.mark.parametrize("kw", SCALINGS)
@pytest.mark.parametrize("r", [4, 64, 72, 128])
def test_frequencies(kw, r):
    got, want = rotary_frequencies(r, **kw), frequencies(r, **kw)
    assert len(got) == r // 2
    assert all(abs(Fraction(g) / Fraction(w) - 1) <= Fraction(1, 2 ** 44) for g, w in zip(got, want))


@pytest.mark.parametrize("kw", SCALINGS + [dict(frequencies=[1.0, -0.3, 3.1415926535897927, 1e-9, 2.0 ** -60, 0.0])])
def test_turns_are_rounded_once(kw):
    """The table is f / 2 pi in units of 2^-64, to half a unit."""
    r = 12 if "frequencies" in kw else 128
    rot = Rotary(128, rotary_dim=r, device="cpu", **kw)
    for f, t in zip(rot.frequencies, rot.turns.tolist()):
        exact = Fraction(f) * 2 ** 64 / (2 * PI)
        assert abs(exact - t) <= Fraction(1, 2), (f, float(exact - t))


def test_far_positions():
    """At position n an angle is off by at most n / 2^65 of a turn: at 2^40 by
    6e-8, of which the doubles' own products would keep nothing below 1e-4."""
    rot = Rotary(64, device="cpu")
    n = 2 ** 40 + 12345
    x = torch.zeros(1, 1, 1, 64, dtype=torch.float64)
    x[..., :32] = 1
    y = rot(x, positions=n)[0, 0, 0]
    for i, f in enumerate(rot.frequencies):
        turn = Fraction(f) * n / (2 * PI)
        a = 2 * math.pi * float(turn - math.floor(turn))
        tol = n * 2.0 ** -65 * 2 * math.pi + 2.0 ** -48
        assert abs(float(y[i]) - math.cos(a)) <= tol and abs(float(y[i + 32]) - math.sin(a)) <= tol, i


@pytest.mark.parametrize("kw", SCALINGS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_outputs(kw, interleaved):
    rot = Rotary(72, rotary_dim=40, interleaved=interleaved, amplitude=1.25, device="cpu", **kw)
    f = frequencies(40, **kw)
    q = torch.randn(2, 3, 5, 72, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    t = torch.arange(5)
    for positions, where in ((7, (7 + t).expand(2, 5)), (torch.tensor([3, 100000]), torch.tensor([3, 100000])[:, None] + t),
                             (torch.tensor([[5, 0, 9, 131072, 1]]), torch.tensor([[5, 0, 9, 131072, 1]]).expand(2, 5))):
        assert_definition(rot(q, positions=positions), q, f, where, interleaved=interleaved, amplitude=1.25)


def test_given_frequencies():
    given = [1.0, -0.3, 0.01, 3.0]
    rot = Rotary(8, frequencies=given, device="cpu")
    q = torch.randn(1, 2, 4, 8, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    assert_definition(rot(q, positions=1000), q, given, (1000 + torch.arange(4))[None])
