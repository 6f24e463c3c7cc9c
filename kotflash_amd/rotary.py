"""Rotary positions: queries and keys turned by the positions of their tokens.

``Rotary`` holds a model's frequencies and turns what its projections give,
before the attention and before keys go into a cache:

    rotary = Rotary(head_dim, base=10000.0, device="cuda")
    q, k = rotary(q, k)                                   # a sequence from position 0
    q, k = rotary(q, k, positions=table.lengths)          # decoding: each request's next tokens
    out = attention(q, k, v, causal=True)

Pair i of the first ``rotary_dim`` dims of a head, (x, y), becomes (x cos a -
y sin a, x sin a + y cos a) at a = position * f_i; the other dims pass as they
are. Differentiable in q and k. An extension of the reference, whose attention
takes what it is given (kotflash/attention.py:223-312).
"""
from __future__ import annotations

import math
from fractions import Fraction
from typing import Optional, Sequence, Union

import torch
from torch.autograd import forward_ad

from . import _hip
from .kernels import hip_rotary

ROTARY_BACKENDS = ("auto", "hip", "torch")
SCALINGS = ("none", "linear", "base", "ramp")

_HALF = (torch.float16, torch.bfloat16)

# To 50 digits: a double's 2 pi would leave 53 of the table's 64 bits.
_TWO_PI = 2 * Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str = "none",
                       factor: float = 1.0, original_length: Optional[int] = None,
                       slow_turns: float = 1.0, fast_turns: float = 4.0) -> list:
    """Radians per position of every pair: f_i = base^(-2 i / rotary_dim), for
    contexts ``factor`` times as long as trained for:

    - ``linear``: f_i / factor, as if positions were;
    - ``base``: base * factor^(r / (r - 2)), which divides the slowest by the
      factor and leaves the fastest;
    - ``ramp``: pairs that turn at least ``fast_turns`` times within
      ``original_length`` positions as they are, those that turn at most
      ``slow_turns`` times f_i / factor, and a line in the turns between."""
    if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, int) or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even integer")
    if scaling not in SCALINGS:
        raise ValueError("scaling must be one of: none, linear, base, ramp")
    if not (math.isfinite(base) and base > 1):
        raise ValueError("base must be a finite number above 1")
    if not (math.isfinite(factor) and factor >= 1) or scaling == "none" and factor != 1:
        raise ValueError("factor must be finite and at least 1, and 1 without scaling")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("scaling='base' needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "ramp":
        if isinstance(original_length, bool) or not isinstance(original_length, int) or original_length <= 0:
            raise ValueError("scaling='ramp' needs original_length, a positive integer")
        if not 0 <= slow_turns < fast_turns < math.inf:
            raise ValueError("slow_turns must be at least 0 and below fast_turns")
        kept = [(original_length * x / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns) for x in f]
        kept = [min(max(w, 0.0), 1.0) for w in kept]
        return [x * w + x / factor * (1 - w) for x, w in zip(f, kept)]
    return f


class _HipRotary(torch.autograd.Function):
    """Eager autograd over the kernel where the native path does not take the
    call. The gradient turns back, by the same function."""

    @staticmethod
    def forward(ctx, q, k, turns, positions, interleaved, inverse, amplitude):
        tensor = isinstance(positions, torch.Tensor)
        ctx.save_for_backward(turns, *((positions,) if tensor else ()))
        ctx.first = None if tensor else positions
        ctx.rest = interleaved, inverse, amplitude
        ctx.set_materialize_grads(False)
        out = hip_rotary.rotate(q, k, turns, positions, interleaved=interleaved, inverse=inverse,
                                amplitude=amplitude)
        return out if k is not None else out[0]

    @staticmethod
    def backward(ctx, dq, dk=None):
        turns, *positions = ctx.saved_tensors
        positions = positions[0] if positions else ctx.first
        interleaved, inverse, amplitude = ctx.rest
        grads = [g if need else None for g, need in zip((dq, dk), ctx.needs_input_grad)]
        there = [g for g in grads if g is not None]
        if there:
            out = _HipRotary.apply(there[0], there[1] if len(there) > 1 else None, turns, positions,
                                   interleaved, not inverse, amplitude)
            out = iter(out if len(there) > 1 else (out,))
            grads = [None if g is None else next(out) for g in grads]
        return (*grads, None, None, None, None, None)


def _transformed(*tensors) -> bool:
    """Whether a torch.func transform or a forward-mode gradient is under way:
    the kernel's autograd node has reverse mode alone."""
    return not torch.compiler.is_compiling() and (
        torch._C._are_functorch_transforms_active()
        or any(forward_ad.unpack_dual(t).tangent is not None for t in tensors if t is not None))


def _torch_rotate(x, turns, positions, interleaved: bool, amplitude: float):
    """The same in torch operations, in fp32 (fp64 for fp64)."""
    b, _, s, _ = x.shape
    if not isinstance(positions, torch.Tensor):
        positions = positions + torch.arange(s, device=x.device)[None]
    elif positions.ndim == 1:
        positions = positions.long()[:, None] + torch.arange(s, device=x.device)
    # The position times the 64-bit fraction of a turn, modulo whole turns.
    fraction = (positions.long()[:, None, :, None] * turns) >> 11
    angle = fraction.double() * (2 * math.pi / 2 ** 53)
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    c, sn = (amplitude * angle.cos()).to(wide), (amplitude * angle.sin()).to(wide)
    r = 2 * turns.numel()
    y = x[..., :r].to(wide)
    one, two = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :r // 2], y[..., r // 2:])
    one, two = one * c - two * sn, one * sn + two * c
    out = torch.stack((one, two), -1).flatten(-2) if interleaved else torch.cat((one, two), -1)
    return torch.cat((out.to(x.dtype), x[..., r:]), -1)


class Rotary:
    """The frequencies of a model's rotary positions.

    ``rotary_dim`` dims of each head turn (default: all), in pairs (i, i +
    rotary_dim / 2), or of neighbours (2 i, 2 i + 1) when ``interleaved``.
    ``base``, ``scaling`` and the arguments behind it are those of
    ``rotary_frequencies``; ``frequencies`` (radians per position of every pair,
    below half a turn) replaces them. Turned dims are multiplied by
    ``amplitude``.

    ``turns`` (int64 [rotary_dim / 2], on the device) holds f_i / 2 pi in units
    of 2^-64 turns, rounded once from the frequencies as doubles
    (``frequencies``): products with positions wrap at whole turns, and the angle
    at position n is off by at most n / 2^65 of a turn (2^-22 of a radian at 2^40).
    """

    def __init__(self, head_dim: int, *, rotary_dim: Optional[int] = None, base: float = 10000.0,
                 interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
                 original_length: Optional[int] = None, slow_turns: float = 1.0,
                 fast_turns: float = 4.0, amplitude: float = 1.0,
                 frequencies: Optional[Sequence[float]] = None,
                 device: Union[torch.device, str] = "cuda") -> None:
        if isinstance(head_dim, bool) or not isinstance(head_dim, int) or head_dim <= 0:
            raise ValueError("head_dim must be a positive integer")
        self.head_dim = head_dim
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        computed = rotary_frequencies(self.rotary_dim, base=base, scaling=scaling, factor=factor,
                                      original_length=original_length, slow_turns=slow_turns,
                                      fast_turns=fast_turns)
        if self.rotary_dim > head_dim:
            raise ValueError("rotary_dim must not exceed head_dim")
        if not isinstance(interleaved, bool):
            raise TypeError("interleaved must be a bool")
        if isinstance(amplitude, bool) or not isinstance(amplitude, (int, float)) or not math.isfinite(amplitude):
            raise ValueError("amplitude must be a finite number")
        if frequencies is not None:
            computed = [float(x) for x in frequencies]
            if len(computed) != self.rotary_dim // 2 or not all(abs(x) < math.pi for x in computed):
                raise ValueError("frequencies must be rotary_dim / 2 numbers of magnitude below pi")
        self.interleaved = interleaved
        self.amplitude = float(amplitude)
        self.frequencies = tuple(computed)
        # An inference tensor could not be saved for a backward pass later.
        with torch.inference_mode(False):
            self.turns = torch.tensor([round(Fraction(x) * 2 ** 64 / _TWO_PI) for x in computed],
                                      dtype=torch.int64, device=device)

    def __call__(self, q, k=None, *, positions: Union[int, torch.Tensor] = 0, backend: str = "auto"):
        """q [B, Hq, S, D] and k [B, Hk, S, D] turned, as new tensors; q alone
        without k. Token t of request b is at position ``positions + t`` (an
        int), ``positions[b] + t`` (int32 or int64 [B], on the device) or
        ``positions[b, t]`` ([B, S], or [1, S] for all).

        ``auto`` takes ``hip`` for fp16 and bf16 on gfx950, but not under
        torch.func's transforms and forward-mode gradients, which ``hip``
        refuses; ``torch`` takes any floating-point type, and computes in 32 bits
        (64 for fp64)."""
        if backend in ("auto", "hip") and not torch.compiler.is_compiling():
            out = _hip.native().rotary(q, k, self.turns, positions, self.head_dim, self.interleaved,
                                       self.amplitude)
            if out is not NotImplemented:
                return out
        if backend not in ROTARY_BACKENDS:
            raise ValueError("backend must be one of: auto, hip, torch")
        hip_rotary.check_rotary(q, k, self.head_dim, positions, self.turns.device)
        on_gfx950 = q.is_cuda and _hip.is_gfx950(q.device)
        if backend == "hip" and not on_gfx950:
            raise RuntimeError("HIP backend requires an AMD MI355X (gfx950) GPU")
        if backend == "hip" and q.dtype not in _HALF:
            raise TypeError(f"HIP rotary supports float16 and bfloat16, got {q.dtype}")
        on_hip = backend != "torch" and on_gfx950 and q.dtype in _HALF
        if on_hip and _transformed(q, k):
            if backend == "hip":
                raise RuntimeError("HIP rotary has no torch.func transforms and forward-mode gradients; "
                                   "backend='torch' has")
            on_hip = False
        if not on_hip:
            out = tuple(None if x is None else
                        _torch_rotate(x, self.turns, positions, self.interleaved, self.amplitude)
                        for x in (q, k))
            return out[0] if k is None else out
        if torch.compiler.is_compiling():
            from .ops import rotary

            tensor = isinstance(positions, torch.Tensor)
            out = rotary(q, q[:, :0] if k is None else k, self.turns, positions if tensor else None,
                         0 if tensor else positions, self.interleaved, False, self.amplitude)
            return out[0] if k is None else out
        return _HipRotary.apply(q, k, self.turns, positions, self.interleaved, False, self.amplitude)
