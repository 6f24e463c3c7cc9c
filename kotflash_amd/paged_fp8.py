"""Paged K/V cache in 8 bits: half the memory, and half of what a decoding step
reads, of ``PagedKVCache`` behind the same ``PageTable``.

    table = PageTable(batch, max_len, num_pages=8192, device="cuda")
    caches = [PagedKVCacheFP8(table, kv_heads, head_dim, dtype=torch.bfloat16) for _ in layers]

    slots = table.reserve(prompt_lengths, width=n)
    for layer, cache in ...: cache.append(k, v, slots)      # quantises
    k, v = cache.read(n)                                    # what a prompt's next chunk attends to
    ...
    q, k = rotary(q, k, positions=table.lengths)
    slots = table.reserve(1)
    out = cache.append_and_attend(q, k, v, slots)

Keys and values are codes of e4m3 (4 significant bits, largest 448) times a
scale. 16 positions of a page, one head, share a scale for K and one for V: the
least power of two with which the largest fits. Powers of two make the product
exact, so that a value is rounded once, by at most 2^-4 of itself, or 2^-10 of
the scale if that is more: codes below 2^-6 have a step of 2^-9, and values
below 2^-10 of the scale (4.4e-6 of the largest it was made for) become zero. A
block takes its scale when its first position is stored; a later token that is
larger makes it grow (for good, though a draft that is trimmed may be the one),
and the rows that are there are divided by the ratio, which rounds what falls
below 2^-6 of the new scale again, by up to 2^-10 of it. Infinities are stored
as NaN.
Inference only. No counterpart in the reference (kotflash/cache.py:1-10).
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _hip
from .kernels import hip_paged_fp8
from .kernels.hip_paged_fp8 import BLOCK, FP8
from .paged import (
    _HALF, PageTable, _no_gradients, _on_gfx950, _options, _positive, _sdpa_paged,
)

STORE_BACKENDS = ("auto", "hip", "torch")


def _on_hip(backend: str, k_pages, v_pages, scales, dtype) -> bool:
    if backend not in STORE_BACKENDS:
        raise ValueError("backend must be one of: auto, hip, torch")
    if backend == "torch":
        return False
    if backend == "auto":
        return (_on_gfx950(k_pages) and dtype in _HALF
                and hip_paged_fp8.pages_in_place(k_pages, v_pages, scales))
    if not _on_gfx950(k_pages):
        raise RuntimeError("HIP backend requires an AMD MI355X (gfx950) GPU")
    return True


# ---------------------------------------------------------------------------
# Functions over plain tensors.

def fp8_append(k_pages, v_pages, scales, new_k, new_v, slots, *, backend: str = "auto") -> None:
    """Quantise new_k/new_v [B, Hkv, S, D] into the pools [pages, Hkv,
    page_size, D] (float8_e4m3fn) at ``slots`` (int64 [B, S]: page * page_size +
    row), with ``scales`` (float32 [pages, Hkv, page_size / 16, 2]; zeros before
    the first call). Slots outside the pool (-1 in the padding of ``reserve``)
    are skipped. Two tokens of a call must not share a slot, tokens of one
    block must follow one another in one request, with no skipped slot between
    (``reserve`` gives them so), and a pool takes one 16-bit type.

    ``auto`` takes ``hip`` for fp16 and bf16 on gfx950, for pools with a
    head_dim that is a multiple of 8 up to 128 and rows that begin at multiples
    of 16 bytes; ``torch`` takes any."""
    if backend in ("auto", "hip") and not torch.compiler.is_compiling() \
            and _hip.native().fp8_append(k_pages, v_pages, scales, new_k, new_v, slots) is None:
        return
    hip_paged_fp8.check_append(k_pages, v_pages, scales, new_k, new_v, slots)
    _no_gradients("8-bit append", scales, new_k, new_v)
    if not _on_hip(backend, k_pages, v_pages, scales, new_k.dtype):
        with torch.no_grad():
            _append(k_pages, v_pages, scales, new_k, new_v, slots)
    elif torch.compiler.is_compiling():
        from .ops import fp8_append_

        fp8_append_(k_pages, v_pages, scales, new_k, new_v, slots)
    else:
        hip_paged_fp8.append_fp8(k_pages, v_pages, scales, new_k, new_v, slots)


def fp8_read(k_pages, v_pages, scales, tables, lengths, width: int, *,
             start: Union[int, torch.Tensor] = 0, dtype: torch.dtype = torch.bfloat16,
             backend: str = "auto"):
    """K and V [B, Hkv, width, D] that the requests hold from position
    ``start`` on (an int, or int32 [B]), as ``paged_attention`` finds them
    through ``tables`` and ``lengths``; zeros behind a request's last position,
    and where its page number is outside the pool."""
    if backend in ("auto", "hip") and not torch.compiler.is_compiling():
        out = _hip.native().fp8_read(k_pages, v_pages, scales, tables, lengths, width, start,
                                     dtype == torch.float16, dtype in _HALF)
        if out is not NotImplemented:
            return out
    hip_paged_fp8.check_read(k_pages, v_pages, scales, tables, lengths, width, start, dtype)
    _no_gradients("8-bit read", scales)
    if not _on_hip(backend, k_pages, v_pages, scales, dtype):
        return _read(k_pages, v_pages, scales, tables, lengths, width, start, dtype)
    if torch.compiler.is_compiling():
        from .ops import fp8_read as op

        first = start if isinstance(start, torch.Tensor) else torch.full_like(lengths, start)
        return op(k_pages, v_pages, scales, tables, lengths, first, width, dtype)
    return hip_paged_fp8.read_fp8(k_pages, v_pages, scales, tables, lengths, width, start, dtype)


def fp8_attention(q, k_pages, v_pages, scales, tables, lengths, *, causal: bool = False,
                  scale: Optional[float] = None, return_lse: bool = False, backend: str = "auto"):
    """Attention of q [B, Hq, Sq, D] over each request's pages of codes, as
    they read back in q's type: ``paged_attention`` in every other respect.

    ``hip`` needs gfx950, q in fp16 or bf16 and pools as ``fp8_append``'s;
    ``auto`` takes it where these hold and ``sdpa`` (one call per request,
    lengths on the host) elsewhere."""
    if backend in ("auto", "hip", "triton") and not torch.compiler.is_compiling():
        out = _hip.native().fp8_attention(q, k_pages, v_pages, scales, tables, lengths, causal, scale,
                                          return_lse)
        if out is not NotImplemented:
            return out
    scale, on_hip = _attention_route(q, k_pages, v_pages, scales, tables, lengths, causal, scale, backend)
    if on_hip and torch.compiler.is_compiling():
        from .ops import fp8_decode

        both = fp8_decode(q, k_pages, v_pages, scales, tables, lengths, causal, scale)
        return both if return_lse else both[0]
    if on_hip:
        return hip_paged_fp8.attention_fp8(q, k_pages, v_pages, scales, tables, lengths, causal=causal,
                                           scale=scale, with_lse=return_lse)

    def rows_of(ids, rows):
        return (_values(pool, scales, i, ids, rows).to(q.dtype) for i, pool in enumerate((k_pages, v_pages)))

    return _sdpa_paged(q, k_pages, v_pages, tables, lengths, causal, scale, return_lse, rows_of)


def _attention_route(q, k_pages, v_pages, scales, tables, lengths, causal, scale, backend):
    """Every check of ``fp8_attention``; its scale, and whether the HIP kernel
    takes it."""
    hip_paged_fp8.check_attention(q, k_pages, v_pages, scales, tables, lengths)
    scale = _options(q, causal, scale, backend)
    _no_gradients("8-bit attention", q, scales)
    if backend == "sdpa":
        return scale, False
    if backend == "auto":
        return scale, (_on_gfx950(q) and q.dtype in _HALF
                       and hip_paged_fp8.pages_in_place(k_pages, v_pages, scales)
                       and hip_paged_fp8.sizes_ok(q, k_pages, v_pages, scales, tables))
    if not _on_gfx950(q):
        raise RuntimeError("HIP backend requires an AMD MI355X (gfx950) GPU")
    hip_paged_fp8.require_readable(q, k_pages, v_pages, scales, tables)
    return scale, True


def _values(pool, scales, which: int, ids, rows):
    """What rows of pages stand for, in fp32: [..., Hkv, D]."""
    return pool.view(torch.uint8)[ids, :, rows].view(FP8).float() * scales[ids, :, rows // BLOCK, which][..., None]


def _scale_for(largest):
    """The least power of two s >= 2^-126 with largest <= 448 s (fp32)."""
    mantissa, exponent = torch.frexp(largest)  # mantissa in [0.5, 1)
    exponent = torch.where(mantissa > 0.875, exponent + 1, exponent) - 9
    exponent = torch.where(largest > 0, exponent, -126).clamp(min=-126)
    return ((exponent + 127) << 23).view(torch.float32)


def _append(k_pages, v_pages, scales, new_k, new_v, slots) -> None:
    """``fp8_append`` in torch operations."""
    pages, hkv, page, _ = k_pages.shape
    blocks = page // BLOCK
    inside = (slots >= 0) & (slots < pages * page)
    at = slots[inside]
    if at.numel() == 0:
        return
    block, of = torch.unique(at // BLOCK, return_inverse=True)
    where, group = block // blocks, block % blocks
    begins = torch.zeros(len(block), dtype=torch.bool, device=at.device)
    begins[of[at % BLOCK == 0]] = True
    top = 16 if new_k.dtype == torch.float16 else 128
    for i, (pool, new) in enumerate(((k_pages, new_k), (v_pages, new_v))):
        x = new.transpose(1, 2)[inside].float()
        size = torch.where(x.isfinite(), x.abs(), 0).amax(-1)
        need = _scale_for(torch.zeros((len(block), hkv), device=at.device).scatter_reduce(
            0, of[:, None].expand(-1, hkv), size, "amax"))
        old = scales[where, :, group, i]
        grows = ~begins[:, None] & (need > old)
        scale = torch.where(begins[:, None] | grows, need, old)
        codes = pool.view(torch.uint8).unflatten(2, (blocks, BLOCK))
        there = codes[where, :, group]
        less = (there.view(FP8).float() * (old / scale)[..., None, None]).to(FP8).view(torch.uint8)
        codes[where, :, group] = torch.where(grows[..., None, None], less, there)
        # A code of 256 may stand for more than the type's largest value.
        limit = (0.9375 * 2.0 ** top / scale[of].double()).clamp(max=448).float()[..., None]
        y = (x / scale[of][..., None]).clamp(-limit, limit)
        y = torch.where(x.isfinite(), y, math.nan).to(FP8)
        codes[where[of], :, group[of], at % BLOCK] = y.view(torch.uint8)
        scales[where, :, group, i] = scale


def _read(k_pages, v_pages, scales, tables, lengths, width: int, start, dtype):
    """``fp8_read`` in torch operations."""
    pages, _, page, _ = k_pages.shape
    t = torch.arange(width, device=tables.device)
    first = start.long().clamp(min=0) if isinstance(start, torch.Tensor) else torch.full_like(lengths, start).long()
    at = first[:, None] + t
    column = at // page
    ids = tables.long().gather(1, column.clamp(max=tables.shape[1] - 1))
    there = (at < lengths[:, None]) & (column < tables.shape[1]) & (ids >= 0) & (ids < pages)
    ids, row = ids.clamp(0, pages - 1), at % page
    out = []
    for i, pool in enumerate((k_pages, v_pages)):
        x = _values(pool, scales, i, ids, row)
        out.append(torch.where(there[..., None, None], x, 0).to(dtype).transpose(1, 2).contiguous())
    return tuple(out)


# ---------------------------------------------------------------------------

class PagedKVCacheFP8:
    """One layer's K/V pages in 8 bits, behind a ``PageTable`` that several may
    share (with 16-bit caches too), whose page_size is a multiple of 16.

    ``k_pages`` and ``v_pages`` are float8_e4m3fn [num_pages, kv_heads,
    page_size, head_dim] (rows padded to 16 bytes), ``scales`` float32
    [num_pages, kv_heads, page_size / 16, 2] (K, V). ``dtype`` is that of the tensors it takes and gives.
    """

    def __init__(self, table: PageTable, kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        if not isinstance(table, PageTable):
            raise TypeError("table must be a PageTable")
        if table.page_size % BLOCK:
            raise ValueError(f"8-bit K/V pages need a page_size that is a multiple of {BLOCK}")
        if dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise ValueError("dtype must be float16, bfloat16 or float32")
        shape = (table.num_pages, _positive("kv_heads", kv_heads), table.page_size,
                 _positive("head_dim", head_dim))
        self.table, self.dtype = table, dtype
        device = table.tables.device
        # Rows in whole pieces of 16 bytes, as the kernels load them.
        wide = (*shape[:3], -(-head_dim // 16) * 16)
        self.k_pages, self.v_pages = (torch.empty(wide, device=device, dtype=FP8)[..., :head_dim]
                                      for _ in range(2))
        self.scales = torch.zeros((*shape[:2], table.page_size // BLOCK, 2), device=device)

    def append(self, new_k, new_v, slots, *, backend: str = "auto") -> None:
        """Quantise new_k/new_v [B, Hkv, S, D] into the slots that the table's
        ``reserve`` returned (``fp8_append``)."""
        if getattr(new_k, "dtype", self.dtype) != self.dtype:
            raise ValueError("new K/V dtype must match the cache's")
        fp8_append(self.k_pages, self.v_pages, self.scales, new_k, new_v, slots, backend=backend)

    def read(self, width: int, *, start: Union[int, torch.Tensor] = 0, backend: str = "auto"):
        """K and V [B, Hkv, width, D] of every request from position ``start``
        on, zeros behind its last (``fp8_read``)."""
        return fp8_read(self.k_pages, self.v_pages, self.scales, self.table.tables,
                        self.table.lengths, width, start=start, dtype=self.dtype, backend=backend)

    def attend(self, q, *, causal: bool = False, scale: Optional[float] = None,
               return_lse: bool = False, backend: str = "auto"):
        """Attention of q [B, Hq, Sq, D] over what each request holds
        (``fp8_attention``)."""
        if getattr(q, "dtype", self.dtype) != self.dtype:
            raise ValueError("q's dtype must match the cache's")
        return fp8_attention(q, self.k_pages, self.v_pages, self.scales, self.table.tables,
                             self.table.lengths, causal=causal, scale=scale, return_lse=return_lse,
                             backend=backend)

    def append_and_attend(self, q, new_k, new_v, slots, *, causal: bool = False,
                          append_backend: str = "auto", attention_backend: str = "auto"):
        """``append``, then ``attend``: a decoding step of this layer, after the
        table's ``reserve`` of the step."""
        pools = self.k_pages, self.v_pages, self.scales
        if append_backend in ("auto", "hip") and attention_backend in ("auto", "hip", "triton") \
                and not torch.compiler.is_compiling() and getattr(q, "dtype", None) == self.dtype:
            out = _hip.native().fp8_step(q, *pools, self.table.tables, self.table.lengths, causal, None,
                                         new_k, new_v, slots)
            if out is not NotImplemented:
                return out
        # Every check of the attention comes before the store writes anything.
        _attention_route(q, *pools, self.table.tables, self.table.lengths, causal, None, attention_backend)
        if q.dtype != self.dtype:
            raise ValueError("q's dtype must match the cache's")
        self.append(new_k, new_v, slots, backend=append_backend)
        return self.attend(q, causal=causal, backend=attention_backend)
