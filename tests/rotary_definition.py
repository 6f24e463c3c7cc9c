"""Rotary positions from the formulas alone, without the table of turns that the
code under test makes: frequencies in decimal arithmetic of 50 digits, pi by
Machin's formula, pairs as complex numbers."""
from decimal import Decimal, getcontext
from fractions import Fraction

import torch

getcontext().prec = 50


def _arctan_inverse(n, digits=60):
    """arctan(1 / n) in whole units of 10^-digits."""
    power = 10 ** digits // n
    total, k, sign = power, 1, 1
    while power:
        power //= n * n
        k, sign = k + 2, -sign
        total += sign * (power // k)
    return total


# pi / 4 = 4 arctan(1/5) - arctan(1/239); off by the truncations of the last
# digits, below 10^-57.
PI = Fraction(4 * (4 * _arctan_inverse(5) - _arctan_inverse(239)), 10 ** 60)


def frequencies(r, *, base=10000.0, scaling="none", factor=1.0, original_length=None, slow_turns=1.0, fast_turns=4.0):
    """f_i as decimals."""
    base, factor = Decimal(base), Decimal(factor)
    if scaling == "base":
        base *= factor ** (Decimal(r) / (r - 2))
    f = [base ** (Decimal(-2 * i) / r) for i in range(r // 2)]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "ramp":
        two_pi = 2 * Decimal(PI.numerator) / Decimal(PI.denominator)
        out = []
        for x in f:
            w = (original_length * x / two_pi - Decimal(slow_turns)) / (Decimal(fast_turns) - Decimal(slow_turns))
            w = min(max(w, Decimal(0)), Decimal(1))
            out.append(w * x + (1 - w) * x / factor)
        return out
    return f


def turned(x, f, positions, *, interleaved=False, amplitude=1.0):
    """x [B, H, S, D] with its pairs turned by positions [B, S] times f, in 64
    bits on the CPU."""
    x, half = x.detach().cpu().double(), len(f)
    angle = positions.cpu().double()[:, None, :, None] * torch.tensor([float(v) for v in f], dtype=torch.float64)
    out = x.clone()
    i = torch.arange(half)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    z = torch.complex(x[..., one], x[..., two]) * torch.polar(torch.full_like(angle, amplitude), angle)
    out[..., one], out[..., two] = z.real, z.imag
    return out


def assert_definition(got, x, f, positions, *, interleaved=False, amplitude=1.0):
    """The code's frequencies are doubles: a power whose exponent and result are
    rounded, 2^-53 each, the exponent's times ln base (below 16), a few products
    and a weight: below 2^-44 of each f. So an angle n f is off by n f 2^-44, and
    by 2^-52 n f for this product; the table's half unit of 2^-64 turns is off by
    2 pi n 2^-65, which is more for the slowest pairs; sines, cosines and the
    rotation by 2^-48 in 64 bits, 2^-20 in the kernel's 32 (as ``rotary_oracle``
    adds them up), all times |x| + |y|; then the type's half step."""
    want = turned(x, f, positions, interleaved=interleaved, amplitude=amplitude)
    x, half = x.detach().cpu().double().abs(), len(f)
    i = torch.arange(half)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    both = (x[..., one] + x[..., two]) * abs(amplitude)
    angle = positions.cpu().double()[:, None, :, None].abs() * torch.tensor([abs(float(v)) for v in f], dtype=torch.float64)
    table = positions.cpu().double()[:, None, :, None].abs() * (2.0 ** -64 * float(PI))
    inner = both * (angle * 2.0 ** -43 + table + (2.0 ** -48 if got.dtype == torch.float64 else 2.0 ** -20))
    tol = torch.zeros_like(want)
    tol[..., one] = tol[..., two] = inner
    info = torch.finfo(got.dtype)
    tol = tol + info.eps / 2 * (want.abs() + tol) + info.smallest_normal * info.eps / 2
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
