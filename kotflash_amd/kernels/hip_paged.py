"""Launchers of the paged K/V cache's kernels (gfx950): page tables, stores by
slot, and attention over the pages. Arguments are checked before anything is
launched; there is no fallback here (``kotflash_amd.paged`` chooses)."""
from __future__ import annotations

from typing import Union

import torch

from .. import _hip
from .._planning import gfx950_head_dim_ok
from ._layout import require_hip_tensors

PAGE_GRANULE = 16  # rows that the decode kernel loads from one page at a time

# Most new rows that ``append_backend="auto"`` has stored by the attention's
# launches: those save a launch and 1.6 us of GPU time for short requests and
# cost a large call 1 us of 57; beyond this many they cost more than they save
# (256 rows 70.5 us and 65.7, also 23.0 and 20.6).
FUSED_STEP_ROWS = 64


def check_pools(k_pages, v_pages) -> None:
    if not isinstance(k_pages, torch.Tensor) or not isinstance(v_pages, torch.Tensor):
        raise TypeError("K/V pages must be torch.Tensor instances")
    if k_pages.ndim != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("K/V pages must have matching [pages, Hkv, page_size, D] shapes")
    if min(k_pages.shape) == 0:
        raise ValueError("K/V pages must be non-empty")
    if v_pages.dtype != k_pages.dtype:
        raise ValueError("K/V pages must have the same dtype")
    if v_pages.device != k_pages.device:
        raise ValueError("K/V pages must be on the same device")


def _check_int32(name: str, t, shape, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be an int32 tensor of shape {list(shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on the same device")


def check_attention(q, k_pages, v_pages, tables, lengths) -> None:
    """The contract of ``paged_attention``, whatever runs it."""
    check_pools(k_pages, v_pages)
    if not isinstance(q, torch.Tensor) or q.ndim != 4:
        raise ValueError("q must use [B, Hq, Sq, D] layout")
    if min(q.shape) == 0:
        raise ValueError("q must be non-empty")
    if q.shape[3] != k_pages.shape[3]:
        raise ValueError("Query head dimension must match the K/V pages")
    if q.shape[1] % k_pages.shape[1]:
        raise ValueError("Query heads must be divisible by the K/V pages' head count")
    if q.device != k_pages.device or q.dtype != k_pages.dtype:
        raise ValueError("Query device and dtype must match the K/V pages")
    if not isinstance(tables, torch.Tensor) or tables.ndim != 2 or tables.shape[1] == 0:
        raise ValueError("tables must be an int32 tensor of shape [B, columns]")
    _check_int32("tables", tables, (q.shape[0], tables.shape[1]), q.device)
    _check_int32("lengths", lengths, (q.shape[0],), q.device)


def check_append(k_pages, v_pages, new_k, new_v, slots) -> None:
    """The contract of ``paged_append``, whatever runs it."""
    check_pools(k_pages, v_pages)
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
    if new_k.dtype != k_pages.dtype or new_v.dtype != k_pages.dtype:
        raise ValueError("new K/V dtype must match the K/V pages")
    if not isinstance(slots, torch.Tensor):
        raise TypeError("slots must be a torch.Tensor")
    if slots.dtype != torch.int64 or tuple(slots.shape) != (new_k.shape[0], new_k.shape[2]):
        raise ValueError("slots must be an int64 tensor of shape [B, S]")
    if slots.device != k_pages.device:
        raise ValueError("slots must be on the K/V pages' device")
    for pool in (k_pages, v_pages):
        if any(s == 0 and n > 1 for s, n in zip(pool.stride(), pool.shape)):
            raise ValueError("K/V pages must not be expanded views")


def pages_readable(k_pages, v_pages) -> bool:
    """Whether the decode kernel reads these pools in place."""
    return (k_pages.shape[2] % PAGE_GRANULE == 0 and k_pages.shape[3] % 8 == 0
            and gfx950_head_dim_ok(k_pages.shape[3])
            and _in_place(k_pages) and _in_place(v_pages))


def _in_place(t) -> bool:
    if not torch.compiler.is_compiling():
        return _hip.layout_ok(t)
    # There is no address under torch.compile; the op copies a pool that begins
    # off a 16-byte border.
    return t.stride(3) == 1 and not any(s % 8 for s in t.stride()[:3])


def sizes_ok(q, k_pages, v_pages, tables) -> bool:
    """Whether the decode kernel addresses these sizes (pools that pass
    ``pages_readable``). Under torch.compile it is left to the call."""
    return torch.compiler.is_compiling() or _hip.paged_decode_check(q, k_pages, v_pages, tables.shape[1]) == 0


def require_readable(q, k_pages, v_pages, tables) -> None:
    require_hip_tensors("paged attention", q, k_pages, v_pages)
    if k_pages.shape[2] % PAGE_GRANULE:
        raise ValueError(f"paged attention needs a page_size that is a multiple of {PAGE_GRANULE}")
    if not pages_readable(k_pages, v_pages):
        raise ValueError("paged attention needs head_dim a multiple of 8 in [8, 128] and "
                         "inner-contiguous, 16-byte aligned K/V pages")
    if not torch.compiler.is_compiling():
        _hip._check(_hip.paged_decode_check(q, k_pages, v_pages, tables.shape[1]), "kf_paged_decode")


def _written(*tensors) -> None:
    """Moves the tensors' version counters, as an in-place torch operation does."""
    torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def attention_paged(q, k_pages, v_pages, tables, lengths, *, causal: bool, scale: float,
                    with_lse: bool = False):
    """O (and LSE) of q over the pages (``kf_paged_decode``); the arguments
    have passed ``check_attention`` and ``require_readable``."""
    q, tables, lengths = _dense(q, tables, lengths)
    b, hq, sq, d = q.shape
    out = torch.empty((b, hq, sq, d), device=q.device, dtype=q.dtype)
    lse = torch.empty((b, hq, sq), device=q.device, dtype=torch.float32) if with_lse else None
    ws = _hip.workspace(q.device, _hip.paged_decode_workspace_bytes(b, hq, k_pages.shape[1], sq, d))
    _hip.paged_decode(q, k_pages, v_pages, out, lse, tables, lengths, scale=scale, causal=causal,
                      workspace=ws)
    return (out, lse) if with_lse else out


def _dense(q, tables, lengths):
    if not _hip.layout_ok(q):
        q = q.contiguous()
    if tables.stride(1) != 1 or (tables.shape[0] > 1 and tables.stride(0) < 0):
        tables = tables.contiguous()
    return q, tables, lengths if lengths.is_contiguous() else lengths.contiguous()


def step_fuses(k_pages, new_k, most: int = _hip.KF_PAGED_STEP_SLOTS) -> bool:
    """Whether the attention's launches can also store these new rows, at most
    ``most`` of them."""
    return (new_k.shape[2] <= _hip.KF_PAGED_STEP_TOKENS
            and new_k.shape[0] * new_k.shape[2] <= most
            and k_pages.shape[0] * k_pages.shape[2] < 2 ** 31)


def append_attention_paged(q, k_pages, v_pages, new_k, new_v, slots, tables, lengths, *,
                           causal: bool, scale: float):
    """O of q over the pages after the store of new_k/new_v at ``slots``, in
    the attention's launches (``kf_paged_append_decode``); the arguments have
    passed ``check_attention``, ``require_readable``, ``check_append`` and
    ``step_fuses``."""
    q, tables, lengths = _dense(q, tables, lengths)
    new_k, new_v = (t if _hip.layout_ok(t) else t.contiguous() for t in (new_k, new_v))
    if slots.stride(1) != 1:
        slots = slots.contiguous()
    b, hq, sq, d = q.shape
    out = torch.empty((b, hq, sq, d), device=q.device, dtype=q.dtype)
    ws = _hip.workspace(q.device, _hip.paged_decode_workspace_bytes(b, hq, k_pages.shape[1], sq, d))
    _hip.paged_append_decode(q, k_pages, v_pages, new_k, new_v, slots, out, None, tables, lengths,
                             scale=scale, causal=causal, workspace=ws)
    _written(k_pages, v_pages)
    return out


def append_paged(k_pages, v_pages, new_k, new_v, slots) -> None:
    """Stores new_k/new_v at their slots (``kf_paged_append``); the arguments
    have passed ``check_append``."""
    require_hip_tensors("paged append", k_pages, v_pages, new_k, new_v)
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise ValueError("K/V pages need a unit head_dim stride")
    if slots.stride(1) != 1:
        slots = slots.contiguous()
    _hip.paged_append(k_pages, v_pages, new_k, new_v, slots)
    _written(k_pages, v_pages)


def check_table(tables, lengths, free_pages, counters) -> None:
    """The state of a page table as the kernels address it."""
    if not isinstance(tables, torch.Tensor) or tables.ndim != 2 or min(tables.shape) == 0:
        raise ValueError("tables must be an int32 tensor of shape [B, columns]")
    device = tables.device
    _check_int32("tables", tables, tables.shape, device)
    _check_int32("lengths", lengths, (tables.shape[0],), device)
    if not isinstance(free_pages, torch.Tensor) or free_pages.ndim != 1 or free_pages.numel() == 0:
        raise ValueError("free_pages must be an int32 tensor of shape [pages]")
    _check_int32("free_pages", free_pages, free_pages.shape, device)
    _check_int32("counters", counters, (4,), device)
    if tables.stride(1) != 1 or not all(t.is_contiguous() for t in (lengths, free_pages, counters)):
        raise ValueError("a page table's state must be dense")
    if not _hip.is_gfx950(device):
        raise RuntimeError("page tables on the GPU require an AMD gfx950 (MI355X) device")


def _per_request(name: str, value, tables):
    if isinstance(value, torch.Tensor):
        _check_int32(name, value, (tables.shape[0],), tables.device)
        return value.contiguous()
    return value


def reserve_pages(tables, lengths, free_pages, counters, counts: Union[int, torch.Tensor],
                  width: int, page_size: int) -> torch.Tensor:
    """Slots of the new tokens (``kf_page_reserve``)."""
    check_table(tables, lengths, free_pages, counters)
    counts = _per_request("counts", counts, tables)
    slots = torch.empty((tables.shape[0], width), device=tables.device, dtype=torch.int64)
    _hip.page_reserve(tables, lengths, free_pages, counters, counts, slots, page_size=page_size)
    _written(tables, lengths, counters)
    return slots


def trim_pages(tables, lengths, free_pages, counters, new_lengths: Union[int, torch.Tensor],
               page_size: int) -> None:
    """Gives back the pages behind the new lengths (``kf_page_trim``)."""
    check_table(tables, lengths, free_pages, counters)
    new_lengths = _per_request("new_lengths", new_lengths, tables)
    _hip.page_trim(tables, lengths, free_pages, counters, new_lengths, page_size=page_size)
    _written(tables, lengths, free_pages, counters)
