"""The HIP kernels as ``torch.library`` custom operators.

The reference wraps its Triton launchers in a ``torch.autograd.Function``
(kotflash/attention.py:203-220). Here the same launchers are registered as
custom ops in the ``kotflash_amd`` namespace, each with a fake (shape-only)
implementation and, for attention, a registered backward:

- ``kotflash_amd::attn_fwd(q, k, v, causal, scale) -> (out, lse)``
- ``kotflash_amd::attn_bwd(q, k, v, out, lse, grad_out, causal, scale) -> (dq, dk, dv)``
- ``kotflash_amd::decode(q, k, v, scale) -> out`` (split-KV decode over
  K/V views read in place, inference only)
- ``kotflash_amd::kv_append_(k_cache, v_cache, new_k, new_v, start) -> ()``
  (mutates both caches)
- ``kotflash_amd::append_decode_(q, k_cache, v_cache, new_k, new_v,
  past_length, scale) -> out`` (fused one-token append + split-KV decode,
  reference kotflash/kernels/triton_decode.py:302-386; mutates both caches)
- ``kotflash_amd::paged_decode(q, k_pages, v_pages, tables, lengths, causal,
  scale) -> (out, lse)``, ``kotflash_amd::paged_append_(k_pages, v_pages,
  new_k, new_v, slots) -> ()``, ``kotflash_amd::page_reserve_(tables, lengths,
  free_pages, counters, counts, page_size, width) -> slots`` and
  ``kotflash_amd::page_trim_(tables, lengths, free_pages, counters,
  new_lengths, page_size) -> ()`` (the paged cache of ``kotflash_amd.paged``,
  no reference counterpart; ``paged_append_`` mutates both pools, the last two
  the page table's state)
- ``kotflash_amd::fp8_append_(k_pages, v_pages, scales, new_k, new_v, slots) -> ()``,
  ``kotflash_amd::fp8_read(k_pages, v_pages, scales, tables, lengths, start,
  width, dtype) -> (k, v)`` and ``kotflash_amd::fp8_decode(q, k_pages, v_pages,
  scales, tables, lengths, causal, scale) -> (out, lse)`` (the 8-bit cache of ``kotflash_amd.paged_fp8``,
  no reference counterpart; the first mutates pools and scales)
- ``kotflash_amd::rotary(q, k, turns, positions, first, interleaved, inverse,
  amplitude) -> (q, k)`` (``kotflash_amd.rotary``, no reference counterpart;
  autograd differentiates it through itself, turned back)

``torch.compile`` traces through them without graph breaks: the fake
implementations give it output shapes, dtypes and strides, and autograd
differentiates ``attn_fwd`` through ``attn_bwd``. Outputs are always
fresh contiguous tensors, as the fake implementations state.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .kernels.hip_backward import attention_backward
from .kernels.hip_decode import attention_forward_strided_append, attention_forward_strided_decode
from .kernels.hip_forward import attention_forward
from .kernels.hip_paged import (
    append_paged, attention_paged, check_append, check_attention, require_readable, reserve_pages,
    trim_pages,
)

from .kernels import hip_paged_fp8
from .kernels.hip_rotary import check_rotary, rotate

__all__ = ["attn_fwd", "attn_bwd", "decode", "kv_append_", "append_decode_", "paged_decode",
           "paged_append_", "page_reserve_", "page_trim_", "fp8_append_", "fp8_read", "fp8_decode", "rotary"]


def _contig(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


@torch.library.custom_op("kotflash_amd::attn_fwd", mutates_args=())
def attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool,
             scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention forward (O in q's dtype, natural-log LSE in fp32)."""
    out, lse = attention_forward(q, k, v, causal=causal, scale=scale)
    return _contig(out), lse


@attn_fwd.register_fake
def _attn_fwd_fake(q, k, v, causal, scale):
    b, hq, sq, d = q.shape
    out = q.new_empty((b, hq, sq, d))
    lse = q.new_empty((b, hq, sq), dtype=torch.float32)
    return out, lse


@torch.library.custom_op("kotflash_amd::attn_bwd", mutates_args=())
def attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
             lse: torch.Tensor, grad_out: torch.Tensor, causal: bool,
             scale: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Attention backward: (dQ, dK, dV) in the inputs' dtypes, dK/dV summed
    over each GQA group."""
    dq, dk, dv = attention_backward(q, k, v, out, lse, grad_out, causal=causal, scale=scale)
    return _contig(dq), _contig(dk), _contig(dv)


@attn_bwd.register_fake
def _attn_bwd_fake(q, k, v, out, lse, grad_out, causal, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _attn_setup_context(ctx, inputs, output):
    q, k, v, causal, scale = inputs
    out, lse = output
    ctx.save_for_backward(q, k, v, out, lse)
    ctx.causal = causal
    ctx.scale = scale
    ctx.mark_non_differentiable(lse)


def _attn_backward(ctx, grad_out, grad_lse):
    q, k, v, out, lse = ctx.saved_tensors
    dq, dk, dv = attn_bwd(q, k, v, out, lse, _contig(grad_out), ctx.causal, ctx.scale)
    return dq, dk, dv, None, None


attn_fwd.register_autograd(_attn_backward, setup_context=_attn_setup_context)


@torch.library.custom_op("kotflash_amd::decode", mutates_args=())
def decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> torch.Tensor:
    """Split-KV decode (short non-causal query block against long K/V views);
    returns O."""
    return _contig(attention_forward_strided_decode(q, k, v, scale=scale))


@decode.register_fake
def _decode_fake(q, k, v, scale):
    return q.new_empty(q.shape)


@torch.library.custom_op("kotflash_amd::kv_append_", mutates_args=("k_cache", "v_cache"))
def kv_append_(k_cache: torch.Tensor, v_cache: torch.Tensor, new_k: torch.Tensor,
               new_v: torch.Tensor, start: int) -> None:
    """cache[:, :, start:start + n] = new for K and V (the reference's
    ``append_kv_`` pybind op, kotflash/csrc/kv_append.cpp:4-14, with its
    checks: matching 4-D shapes, fp16/bf16, unit head_dim stride, capacity)."""
    from . import _hip
    from .cache import _validate_kv_tensors
    from .kernels._layout import require_hip_tensors

    _validate_kv_tensors(k_cache, v_cache, new_k, new_v)
    require_hip_tensors("kv_append_", k_cache, v_cache, new_k, new_v)
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("K/V caches need a unit head_dim stride")
    if start < 0 or start + new_k.shape[2] > k_cache.shape[2]:
        raise ValueError("KV cache capacity exceeded")
    _hip.kv_append(k_cache, v_cache, new_k, new_v, start=start)


@kv_append_.register_fake
def _kv_append_fake(k_cache, v_cache, new_k, new_v, start):
    return None


@torch.library.custom_op("kotflash_amd::append_decode_", mutates_args=("k_cache", "v_cache"))
def append_decode_(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   new_k: torch.Tensor, new_v: torch.Tensor, past_length: int,
                   scale: float) -> torch.Tensor:
    """Store one new token at ``past_length`` of both caches and attend with
    q [B, Hq, 1, D] over the first past_length + 1 positions (the split kernel
    writes the token; two launches). Returns O."""
    return _contig(attention_forward_strided_append(q, k_cache, v_cache, new_k, new_v,
                                                    past_length=past_length, scale=scale))


@append_decode_.register_fake
def _append_decode_fake(q, k_cache, v_cache, new_k, new_v, past_length, scale):
    return q.new_empty(q.shape)


@torch.library.custom_op("kotflash_amd::paged_decode", mutates_args=())
def paged_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 tables: torch.Tensor, lengths: torch.Tensor, causal: bool,
                 scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention over the pages (``kotflash_amd.paged.paged_attention`` on the
    HIP kernels): O and LSE; inference only."""
    check_attention(q, k_pages, v_pages, tables, lengths)
    k_pages, v_pages = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (k_pages, v_pages))
    require_readable(q, k_pages, v_pages, tables)
    return attention_paged(q, k_pages, v_pages, tables, lengths, causal=causal, scale=scale,
                           with_lse=True)


@paged_decode.register_fake
def _paged_decode_fake(q, k_pages, v_pages, tables, lengths, causal, scale):
    b, hq, sq, d = q.shape
    return q.new_empty((b, hq, sq, d)), q.new_empty((b, hq, sq), dtype=torch.float32)


@torch.library.custom_op("kotflash_amd::paged_append_", mutates_args=("k_pages", "v_pages"))
def paged_append_(k_pages: torch.Tensor, v_pages: torch.Tensor, new_k: torch.Tensor,
                  new_v: torch.Tensor, slots: torch.Tensor) -> None:
    """new_k/new_v [B, Hkv, S, D] to their slots of the pools."""
    check_append(k_pages, v_pages, new_k, new_v, slots)
    append_paged(k_pages, v_pages, new_k, new_v, slots)


@paged_append_.register_fake
def _paged_append_fake(k_pages, v_pages, new_k, new_v, slots):
    return None


@torch.library.custom_op("kotflash_amd::page_reserve_", mutates_args=("tables", "lengths", "counters"))
def page_reserve_(tables: torch.Tensor, lengths: torch.Tensor, free_pages: torch.Tensor,
                  counters: torch.Tensor, counts: torch.Tensor, page_size: int,
                  width: int) -> torch.Tensor:
    """Pages and slots for counts[b] more tokens of every request
    (``PageTable.reserve``)."""
    return reserve_pages(tables, lengths, free_pages, counters, counts, width, page_size)


@page_reserve_.register_fake
def _page_reserve_fake(tables, lengths, free_pages, counters, counts, page_size, width):
    return tables.new_empty((tables.shape[0], width), dtype=torch.int64)


@torch.library.custom_op("kotflash_amd::page_trim_",
                         mutates_args=("tables", "lengths", "free_pages", "counters"))
def page_trim_(tables: torch.Tensor, lengths: torch.Tensor, free_pages: torch.Tensor,
               counters: torch.Tensor, new_lengths: torch.Tensor, page_size: int) -> None:
    """Back to new_lengths[b] tokens of every request (``PageTable.trim``)."""
    trim_pages(tables, lengths, free_pages, counters, new_lengths, page_size)


@page_trim_.register_fake
def _page_trim_fake(tables, lengths, free_pages, counters, new_lengths, page_size):
    return None


@torch.library.custom_op("kotflash_amd::fp8_append_", mutates_args=("k_pages", "v_pages", "scales"))
def fp8_append_(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, new_k: torch.Tensor,
                new_v: torch.Tensor, slots: torch.Tensor) -> None:
    """new_k/new_v [B, Hkv, S, D] quantised into their slots of the pools."""
    hip_paged_fp8.check_append(k_pages, v_pages, scales, new_k, new_v, slots)
    hip_paged_fp8.append_fp8(k_pages, v_pages, scales, new_k, new_v, slots)


@fp8_append_.register_fake
def _fp8_append_fake(k_pages, v_pages, scales, new_k, new_v, slots):
    return None


@torch.library.custom_op("kotflash_amd::fp8_read", mutates_args=())
def fp8_read(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, tables: torch.Tensor,
             lengths: torch.Tensor, start: torch.Tensor, width: int,
             dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V of every request from its start on
    (``kotflash_amd.paged_fp8.fp8_read`` on the HIP kernel)."""
    hip_paged_fp8.check_read(k_pages, v_pages, scales, tables, lengths, width, start, dtype)
    return hip_paged_fp8.read_fp8(k_pages, v_pages, scales, tables, lengths, width, start, dtype)


@fp8_read.register_fake
def _fp8_read_fake(k_pages, v_pages, scales, tables, lengths, start, width, dtype):
    shape = (tables.shape[0], k_pages.shape[1], width, k_pages.shape[3])
    return k_pages.new_empty(shape, dtype=dtype), k_pages.new_empty(shape, dtype=dtype)


@torch.library.custom_op("kotflash_amd::fp8_decode", mutates_args=())
def fp8_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor,
               tables: torch.Tensor, lengths: torch.Tensor, causal: bool,
               scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention over the pages (``kotflash_amd.paged_fp8.fp8_attention`` on
    the HIP kernels): O and LSE; inference only."""
    hip_paged_fp8.check_attention(q, k_pages, v_pages, scales, tables, lengths)
    hip_paged_fp8.require_readable(q, k_pages, v_pages, scales, tables)
    return hip_paged_fp8.attention_fp8(q, k_pages, v_pages, scales, tables, lengths, causal=causal,
                                       scale=scale, with_lse=True)


@fp8_decode.register_fake
def _fp8_decode_fake(q, k_pages, v_pages, scales, tables, lengths, causal, scale):
    b, hq, sq, d = q.shape
    return q.new_empty((b, hq, sq, d)), q.new_empty((b, hq, sq), dtype=torch.float32)


@torch.library.custom_op("kotflash_amd::rotary", mutates_args=())
def rotary(q: torch.Tensor, k: torch.Tensor, turns: torch.Tensor, positions: Optional[torch.Tensor],
           first: int, interleaved: bool, inverse: bool,
           amplitude: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """q and k (of no heads: none) turned by their positions
    (``kotflash_amd.rotary.Rotary`` on the HIP kernel)."""
    where = first if positions is None else positions
    keys = k if k.shape[1] else None
    check_rotary(q, keys, q.shape[3], where, turns.device)
    if turns.dtype != torch.int64 or turns.ndim != 1 or not 0 < 2 * turns.numel() <= q.shape[3]:
        raise ValueError("turns must be an int64 tensor of shape [rotary_dim / 2]")
    q_out, k_out = rotate(q, keys, turns.contiguous(), where, interleaved=interleaved,
                          inverse=inverse, amplitude=amplitude)
    return q_out, torch.empty_like(k) if k_out is None else k_out


@rotary.register_fake
def _rotary_fake(q, k, turns, positions, first, interleaved, inverse, amplitude):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _rotary_setup_context(ctx, inputs, output):
    q, k, turns, positions, first, interleaved, inverse, amplitude = inputs
    ctx.save_for_backward(turns, positions)
    ctx.rest = first, interleaved, inverse, amplitude


def _rotary_backward(ctx, dq, dk):
    turns, positions = ctx.saved_tensors
    first, interleaved, inverse, amplitude = ctx.rest
    dq, dk = rotary(dq, dk, turns, positions, first, interleaved, not inverse, amplitude)
    return dq, dk, None, None, None, None, None, None


rotary.register_autograd(_rotary_backward, setup_context=_rotary_setup_context)
