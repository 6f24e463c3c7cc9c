"""Rotary positions from their definition: the angle of every pair by exact
whole numbers, sines and cosines in 64 bits."""
import math

import torch


def turned64(x, rot, positions, inverse=False):
    """x turned, in 64 bits on the CPU."""
    x = x.detach().cpu().double()
    b, _, s, _ = x.shape
    if isinstance(positions, int):
        rows = [[positions + t for t in range(s)]] * b
    elif positions.ndim == 1:
        rows = [[n + t for t in range(s)] for n in positions.tolist()]
    else:
        rows = positions.expand(b, s).tolist()
    turns = rot.turns.tolist()
    # Python's whole numbers: the fraction of a turn, without rounding.
    angle = torch.tensor([[[(n * f) % 2 ** 64 / 2 ** 64 * 2 * math.pi for f in turns] for n in row] for row in rows],
                         dtype=torch.float64)[:, None]
    c, sn = angle.cos() * rot.amplitude, angle.sin() * rot.amplitude * (-1 if inverse else 1)
    out, half = x.clone(), len(turns)
    i = torch.arange(half)
    one, two = (2 * i, 2 * i + 1) if rot.interleaved else (i, i + half)
    out[..., one] = x[..., one] * c - x[..., two] * sn
    out[..., two] = x[..., one] * sn + x[..., two] * c
    return out


def assert_turned(got, x, rot, positions, inverse=False):
    """A turned element is a sum of two products: the sine and cosine are good
    to 2^-22 (their polynomials to 2^-25, the angle's fp32 rounding 2^-24 of at
    most pi / 4, its 32-bit fraction 2 pi 2^-33, and roundings of 2^-24 at each
    of the last steps), the amplitude's product, the two products and the sum
    round to 2^-24 each: in all below 2^-20 amplitude (|x| + |y|). Then one
    rounding to the type: eps / 2 of the value, at least half its smallest
    step. In fp64 (angles of 53 bits): 2^-48. Dims that pass are equal."""
    want = turned64(x, rot, positions, inverse)
    r = 2 * rot.turns.numel()
    big = x.detach().cpu().double().abs()
    half = r // 2
    i = torch.arange(half)
    one, two = (2 * i, 2 * i + 1) if rot.interleaved else (i, i + half)
    pair = torch.zeros_like(want)
    pair[..., one] = pair[..., two] = big[..., one] + big[..., two]
    inner = 2.0 ** -48 if got.dtype == torch.float64 else 2.0 ** -20
    info = torch.finfo(got.dtype)
    tol = inner * abs(rot.amplitude) * pair
    tol = tol + info.eps / 2 * (want.abs() + tol) + info.smallest_normal * info.eps / 2
    assert torch.equal(got.detach().cpu()[..., r:], x.detach().cpu()[..., r:])
    err = (got.detach().cpu().double() - want).abs()[..., :r]
    worst = int((err - tol[..., :r]).argmax())
    assert bool((err <= tol[..., :r]).all()), (
        f"{int((err > tol[..., :r]).sum())} of {err.numel()} outside; worst: {float(err.flatten()[worst])} > "
        f"{float(tol[..., :r].flatten()[worst])}")
