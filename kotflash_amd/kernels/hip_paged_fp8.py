"""Launchers of the 8-bit paged cache's kernels (gfx950): the quantising store,
the read back, and attention over the pages. Arguments are checked before
anything is launched; there is no fallback here (``kotflash_amd.paged_fp8``
chooses)."""
from __future__ import annotations

from typing import Union

import torch

from .. import _hip
from ._layout import require_hip_tensors
from .hip_paged import _check_int32, _written

FP8 = torch.float8_e4m3fn
BLOCK = 16  # positions that share a scale, per head


def check_pools(k_pages, v_pages, scales) -> None:
    for name, t in (("K/V pages", k_pages), ("K/V pages", v_pages), ("scales", scales)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be torch.Tensor instances")
    if k_pages.ndim != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("K/V pages must have matching [pages, Hkv, page_size, D] shapes")
    if min(k_pages.shape) == 0:
        raise ValueError("K/V pages must be non-empty")
    if k_pages.dtype != FP8 or v_pages.dtype != FP8:
        raise ValueError("8-bit K/V pages must be float8_e4m3fn")
    pages, hkv, page, _ = k_pages.shape
    if page % BLOCK:
        raise ValueError(f"8-bit K/V pages need a page_size that is a multiple of {BLOCK}")
    if scales.dtype != torch.float32 or tuple(scales.shape) != (pages, hkv, page // BLOCK, 2):
        raise ValueError(f"scales must be a float32 tensor of shape {[pages, hkv, page // BLOCK, 2]}")
    if v_pages.device != k_pages.device or scales.device != k_pages.device:
        raise ValueError("K/V pages and scales must be on the same device")


def check_append(k_pages, v_pages, scales, new_k, new_v, slots) -> None:
    """The contract of ``fp8_append``, whatever runs it."""
    check_pools(k_pages, v_pages, scales)
    if not isinstance(new_k, torch.Tensor) or not isinstance(new_v, torch.Tensor):
        raise TypeError("new_k and new_v must be torch.Tensor instances")
    if new_k.ndim != 4 or new_v.shape != new_k.shape:
        raise ValueError("new K/V must have matching [B, Hkv, S, D] shapes")
    if min(new_k.shape) == 0:
        raise ValueError("cannot append an empty K/V sequence")
    if new_k.shape[1] != k_pages.shape[1] or new_k.shape[3] != k_pages.shape[3]:
        raise ValueError("new K/V heads and head_dim must match the K/V pages")
    if new_k.device != k_pages.device or new_v.device != k_pages.device:
        raise ValueError("new K/V must be on the K/V pages' device")
    if new_v.dtype != new_k.dtype or new_k.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("new K/V must share one dtype, float16, bfloat16 or float32")
    if not isinstance(slots, torch.Tensor):
        raise TypeError("slots must be a torch.Tensor")
    if slots.dtype != torch.int64 or tuple(slots.shape) != (new_k.shape[0], new_k.shape[2]):
        raise ValueError("slots must be an int64 tensor of shape [B, S]")
    if slots.device != k_pages.device:
        raise ValueError("slots must be on the K/V pages' device")
    for pool in (k_pages, v_pages, scales):
        if any(s == 0 and n > 1 for s, n in zip(pool.stride(), pool.shape)):
            raise ValueError("K/V pages and scales must not be expanded views")


def check_tables(tables, lengths, device) -> None:
    if not isinstance(tables, torch.Tensor) or tables.ndim != 2 or min(tables.shape) == 0:
        raise ValueError("tables must be an int32 tensor of shape [B, columns]")
    _check_int32("tables", tables, tables.shape, device)
    _check_int32("lengths", lengths, (tables.shape[0],), device)


def check_read(k_pages, v_pages, scales, tables, lengths, width, start, dtype) -> None:
    """The contract of ``fp8_read``, whatever runs it."""
    check_pools(k_pages, v_pages, scales)
    check_tables(tables, lengths, k_pages.device)
    if isinstance(width, bool) or not isinstance(width, int):
        raise TypeError("width must be an int")
    if not 0 < width < 2 ** 30:
        raise ValueError("width must be in [1, 2**30)")
    if isinstance(start, torch.Tensor):
        _check_int32("start", start, (tables.shape[0],), tables.device)
    elif isinstance(start, bool) or not isinstance(start, int):
        raise TypeError("start must be an int or a device int32 tensor")
    elif not 0 <= start < 2 ** 30:
        raise ValueError("start must be in [0, 2**30)")
    if dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("dtype must be float16, bfloat16 or float32")


def check_attention(q, k_pages, v_pages, scales, tables, lengths) -> None:
    """The contract of ``fp8_attention``, whatever runs it."""
    check_pools(k_pages, v_pages, scales)
    if not isinstance(q, torch.Tensor) or q.ndim != 4:
        raise ValueError("q must use [B, Hq, Sq, D] layout")
    if min(q.shape) == 0:
        raise ValueError("q must be non-empty")
    if q.shape[3] != k_pages.shape[3]:
        raise ValueError("Query head dimension must match the K/V pages")
    if q.shape[1] % k_pages.shape[1]:
        raise ValueError("Query heads must be divisible by the K/V pages' head count")
    if q.device != k_pages.device:
        raise ValueError("Query device must match the K/V pages")
    if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("q must be float16, bfloat16 or float32")
    check_tables(tables, lengths, q.device)
    if tables.shape[0] != q.shape[0]:
        raise ValueError("tables must be an int32 tensor of shape [B, columns]")


def sizes_ok(q, k_pages, v_pages, scales, tables) -> bool:
    """Whether the decode kernel addresses these sizes (pools that pass
    ``pages_in_place``). Under torch.compile it is left to the call."""
    return (torch.compiler.is_compiling()
            or _hip.fp8_decode_check(q, k_pages, v_pages, scales, tables.shape[1]) == 0)


def require_readable(q, k_pages, v_pages, scales, tables) -> None:
    require_hip_tensors("8-bit attention", q)
    require_in_place("8-bit attention", k_pages, v_pages, scales)
    if not torch.compiler.is_compiling():
        _hip._check(_hip.fp8_decode_check(q, k_pages, v_pages, scales, tables.shape[1]), "kf_fp8_decode")


def attention_fp8(q, k_pages, v_pages, scales, tables, lengths, *, causal: bool, scale: float,
                  with_lse: bool = False):
    """O (and LSE) of q over the pages (``kf_fp8_decode``); the arguments have
    passed ``check_attention`` and ``require_readable``."""
    if not _hip.layout_ok(q):
        q = q.contiguous()
    tables, lengths = dense_tables(tables, lengths)
    b, hq, sq, d = q.shape
    out = torch.empty((b, hq, sq, d), device=q.device, dtype=q.dtype)
    lse = torch.empty((b, hq, sq), device=q.device, dtype=torch.float32) if with_lse else None
    ws = _hip.workspace(q.device, _hip.fp8_decode_workspace_bytes(b, hq, k_pages.shape[1], sq, d))
    _hip.fp8_decode(q, k_pages, v_pages, scales, out, lse, tables, lengths, scale=scale, causal=causal,
                    workspace=ws)
    return (out, lse) if with_lse else out


def pages_in_place(k_pages, v_pages, scales) -> bool:
    """Whether the kernels read and write these pools as they are."""
    if k_pages.shape[3] % 8 or k_pages.shape[3] > 128:
        return False
    for t, unit, granule in ((k_pages, 1, 16), (v_pages, 1, 16), (scales, 1, 2)):
        st = t.stride()
        if st[3] != unit or any(s % granule for s in st[:3]):
            return False
        # There is no address under torch.compile; the ops check it.
        if not torch.compiler.is_compiling() and t.data_ptr() % (16 if t is not scales else 8):
            return False
    if k_pages.shape[3] % 16 and not all(_row_padded(t) for t in (k_pages, v_pages)):
        return False
    return scales.stride(2) == 2


def _row_padded(t) -> bool:
    """Whether a row of 8 (2 n + 1) bytes has its last 8 bytes of padding in the
    tensor's own storage, behind the last row too."""
    if t.stride(2) < t.shape[3] + 8:
        return False
    if torch.compiler.is_compiling():
        return True
    end = t.storage_offset() + t.shape[3] + 8 + sum((n - 1) * s for n, s in zip(t.shape[:3], t.stride()))
    return end <= t.untyped_storage().nbytes()


def require_in_place(what: str, k_pages, v_pages, scales) -> None:
    if not _hip.is_gfx950(k_pages.device):
        raise RuntimeError(f"{what} requires an AMD gfx950 (MI355X) device")
    if not pages_in_place(k_pages, v_pages, scales):
        raise ValueError(f"{what} needs head_dim a multiple of 8 in [8, 128], inner-contiguous K/V pages, "
                         "rows and pages 16-byte aligned, and scales in pairs")


def append_fp8(k_pages, v_pages, scales, new_k, new_v, slots) -> None:
    """Quantises new_k/new_v into their slots (``kf_fp8_append``); the
    arguments have passed ``check_append``."""
    require_hip_tensors("8-bit append", new_k, new_v)
    require_in_place("8-bit append", k_pages, v_pages, scales)
    new_k, new_v = (t if _hip.layout_ok(t) else t.contiguous() for t in (new_k, new_v))
    if slots.stride(1) != 1:
        slots = slots.contiguous()
    _hip.fp8_append(k_pages, v_pages, scales, new_k, new_v, slots)
    _written(k_pages, v_pages, scales)


def dense_tables(tables, lengths):
    if tables.stride(1) != 1 or (tables.shape[0] > 1 and tables.stride(0) < 0):
        tables = tables.contiguous()
    return tables, lengths if lengths.is_contiguous() else lengths.contiguous()


def read_fp8(k_pages, v_pages, scales, tables, lengths, width: int,
             start: Union[int, torch.Tensor], dtype: torch.dtype):
    """K and V [B, Hkv, width, D] in ``dtype`` (``kf_fp8_read``); the arguments
    have passed ``check_read``."""
    require_in_place("8-bit read", k_pages, v_pages, scales)
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"8-bit read supports float16 and bfloat16, got {dtype}")
    tables, lengths = dense_tables(tables, lengths)
    if isinstance(start, torch.Tensor):
        start = start.contiguous()
    shape = (tables.shape[0], k_pages.shape[1], width, k_pages.shape[3])
    k, v = (torch.empty(shape, device=k_pages.device, dtype=dtype) for _ in range(2))
    _hip.fp8_read(k_pages, v_pages, scales, k, v, tables, lengths, start)
    return k, v
