"""Launcher of the rotary kernel (gfx950). Arguments are checked before
anything is launched; there is no fallback here (``kotflash_amd.rotary``
chooses)."""
from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _hip


def check_rotary(q, k, head_dim: int, positions, device: torch.device) -> None:
    """The contract of ``Rotary``'s call, whatever runs it."""
    for name, t in (("q", q), ("k", k)):
        if t is None and name == "k":
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.ndim != 4:
            raise ValueError(f"{name} must use [B, heads, S, D] layout")
        if not t.is_floating_point():
            raise TypeError(f"{name} must be a floating-point tensor")
        if t.device != device:
            raise ValueError(f"{name} must be on the rotary frequencies' device")
    if min(q.shape) == 0:
        raise ValueError("q must be non-empty")
    if q.shape[3] != head_dim:
        raise ValueError(f"q must have head_dim {head_dim}")
    if k is not None and ((k.shape[0], k.shape[2], k.shape[3]) != (q.shape[0], q.shape[2], q.shape[3])
                          or k.shape[1] == 0):
        raise ValueError("k must have q's batch, sequence and head_dim")
    if k is not None and k.dtype != q.dtype:
        raise ValueError("q and k must have the same dtype")
    if isinstance(positions, torch.Tensor):
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be int32 or int64")
        b, s = q.shape[0], q.shape[2]
        if tuple(positions.shape) not in ((b,), (b, s), (1, s)):
            raise ValueError("positions must be an int or a tensor of shape [B], [B, S] or [1, S]")
        if positions.device != q.device:
            raise ValueError("positions must be on q's device")
    elif isinstance(positions, bool) or not isinstance(positions, int):
        raise TypeError("positions must be an int or a tensor of int32 or int64")
    elif not -2 ** 62 <= positions < 2 ** 62:
        raise ValueError("positions must be in [-2**62, 2**62)")


def rotate(q, k: Optional[torch.Tensor], turns, positions: Union[int, torch.Tensor], *,
           interleaved: bool, inverse: bool, amplitude: float):
    """q and k turned (``kf_rotary``), as fresh contiguous tensors; the
    arguments have passed ``check_rotary``."""
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"HIP rotary supports float16 and bfloat16, got {q.dtype}")
    if not _hip.is_gfx950(q.device):
        raise RuntimeError("HIP rotary requires an AMD gfx950 (MI355X) device")
    q_out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    k_out = None if k is None else torch.empty(k.shape, device=k.device, dtype=k.dtype)
    _hip.rotary(q, k, q_out, k_out, turns, positions, interleaved=interleaved, inverse=inverse,
                amplitude=amplitude)
    return q_out, k_out
