"""Paged K/V cache: requests hold their keys and values in pages of a pool.

``PreallocatedKVCache`` and ``RaggedKVCache`` give every sequence ``max_len``
positions of its own. A server whose requests come, grow and leave at their
own lengths keeps pages instead: ``PageTable`` says which pages of a common
pool each request holds, entirely on the GPU, and ``PagedKVCache`` is the pool
of one layer, stored to and attended over through the table. A model's layers
share one table:

    table = PageTable(batch, max_len, num_pages=4096, device="cuda")
    caches = [PagedKVCache(table, kv_heads, head_dim, dtype=torch.float16) for _ in layers]

    slots = table.reserve(prompt_lengths, width=n)        # room for the prompts
    for layer, cache in ...: cache.append(k, v, slots)    # [B, Hkv, n, D]
    ...
    slots = table.reserve(1)                              # one token each
    out = cache.append_and_attend(q, k, v, slots)         # per layer
    table.trim(kept)                                      # drop drafts, or a finished request

Lengths, tables and the free pages are device tensors that no call copies to
the host, so a step can be captured in a graph and replayed as requests grow.
Nothing here is thread-safe, and a table or cache is used on one stream at a
time (with events between streams). Inference only. An extension of the
reference, which has no paging (kotflash/cache.py:1-10).
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch
from torch.autograd import forward_ad

from . import _hip
from .attention import _sdpa
from .kernels import hip_paged

PAGED_BACKENDS = ("auto", "hip", "triton", "sdpa")
STORE_BACKENDS = ("auto", "hip", "cuda", "torch")

_HALF = (torch.float16, torch.bfloat16)


def _on_gfx950(t: torch.Tensor) -> bool:
    """Whether ``auto`` takes the HIP kernels for this device. A gfx950 without
    the library is a broken install: the launchers raise."""
    return t.is_cuda and _hip.is_gfx950(t.device)


def _no_gradients(what: str, *tensors) -> None:
    if (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)
            or not torch.compiler.is_compiling()
            and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)):
        raise RuntimeError(f"{what} is inference-only; disable gradients")


def _store_on_hip(backend: str, t: torch.Tensor, half: bool) -> bool:
    if backend not in STORE_BACKENDS:
        raise ValueError("append backend must be one of: auto, hip, cuda or torch")
    if backend == "auto":
        return _on_gfx950(t) and (not half or t.dtype in _HALF)
    if backend == "torch":
        return False
    if not _on_gfx950(t):
        raise RuntimeError("HIP backend requires an AMD MI355X (gfx950) GPU")
    return True


# ---------------------------------------------------------------------------
# Functions over plain tensors.

def paged_append(k_pages, v_pages, new_k, new_v, slots, *, backend: str = "auto") -> None:
    """Store new_k/new_v [B, Hkv, S, D] in the pools [pages, Hkv, page_size, D]
    at ``slots`` (int64 [B, S]: page * page_size + row): K and V bit-exact, in
    one launch. Slots outside the pool (-1 in the padding of ``reserve``) are
    skipped. Two tokens of a call must not share a slot (what it holds then is
    either's, or a mixture), and new_k/new_v must not lie in the pools.

    ``auto`` takes ``hip`` for fp16 and bf16 on gfx950, which needs pools with a
    unit head_dim stride and refuses others; ``torch`` takes any."""
    # The ordinary GPU call is checked and launched natively; anything else (and
    # every error) takes the checks below. So do the calls further down.
    if backend in ("auto", "hip", "cuda") and not torch.compiler.is_compiling() \
            and _hip.native().paged_append(k_pages, v_pages, new_k, new_v, slots) is None:
        return
    hip_paged.check_append(k_pages, v_pages, new_k, new_v, slots)
    _no_gradients("paged append", k_pages, v_pages, new_k, new_v)
    if _store_on_hip(backend, k_pages, half=True):
        if torch.compiler.is_compiling():
            from .ops import paged_append_

            paged_append_(k_pages, v_pages, new_k, new_v, slots)
            return
        hip_paged.append_paged(k_pages, v_pages, new_k, new_v, slots)
        return
    page = k_pages.shape[2]
    with torch.no_grad():
        inside = (slots >= 0) & (slots < k_pages.shape[0] * page)
        at = slots[inside]
        for pool, new in ((k_pages, new_k), (v_pages, new_v)):
            pool[at // page, :, at % page] = new.transpose(1, 2)[inside]


def paged_attention(q, k_pages, v_pages, tables, lengths, *, causal: bool = False,
                    scale: Optional[float] = None, return_lse: bool = False,
                    backend: str = "auto"):
    """Attention of q [B, Hq, Sq, D] over each request's pages.

    Position j of request b is row ``j % page_size`` of page ``tables[b, j //
    page_size]`` (int32 [B, columns]) of the pools [pages, Hkv, page_size, D];
    its rows see the first ``lengths[b]`` (int32 [B]) positions. With
    ``causal`` the Sq query tokens are the request's last ones (draft tokens,
    already stored): row i sees the first ``lengths[b] - Sq + 1 + i``, so a
    request with fewer new tokens than Sq has them in its last rows. A row that
    sees nothing gives zeros (LSE -inf), one that sees a score of NaN or
    +infinity NaN (LSE not finite); a position whose page number is outside the
    pool is not seen. MHA, GQA and MQA as in ``attention``.

    ``hip`` needs gfx950, fp16 or bf16, a head_dim that is a multiple of 8 up
    to 128, a page_size that is a multiple of 16 and tables of fewer than 2**31
    steps of 32 positions, over all requests and KV heads; ``auto`` takes it where
    these hold and ``sdpa`` (one call per request, lengths on the host)
    elsewhere. With ``return_lse``, returns (O, LSE), LSE in fp32 [B, Hq, Sq].
    """
    if backend in ("auto", "hip", "triton") and not torch.compiler.is_compiling():
        out = _hip.native().paged_attention(q, k_pages, v_pages, tables, lengths, causal, scale,
                                            return_lse)
        if out is not NotImplemented:
            return out
    scale, on_hip = _attention_route(q, k_pages, v_pages, tables, lengths, causal, scale, backend)
    if on_hip and torch.compiler.is_compiling():
        from .ops import paged_decode

        both = paged_decode(q, k_pages, v_pages, tables, lengths, causal, scale)
        return both if return_lse else both[0]
    if on_hip:
        return hip_paged.attention_paged(q, k_pages, v_pages, tables, lengths, causal=causal,
                                         scale=scale, with_lse=return_lse)
    return _sdpa_paged(q, k_pages, v_pages, tables, lengths, causal, scale, return_lse)


def _attention_route(q, k_pages, v_pages, tables, lengths, causal, scale, backend):
    """Every check of ``paged_attention``; its scale, and whether the HIP
    kernel takes it."""
    hip_paged.check_attention(q, k_pages, v_pages, tables, lengths)
    if not isinstance(causal, bool):
        raise TypeError("causal must be a bool")
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    else:
        try:
            scale = float(scale)
        except (TypeError, ValueError) as exc:
            raise TypeError("scale must be a finite real number or None") from exc
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
    if backend not in PAGED_BACKENDS:
        raise ValueError("backend must be one of: auto, hip, triton, sdpa")
    _no_gradients("paged attention", q, k_pages, v_pages)
    if backend == "sdpa":
        return scale, False
    if backend == "auto":
        return scale, (_on_gfx950(q) and q.dtype in _HALF
                       and hip_paged.pages_readable(k_pages, v_pages)
                       and hip_paged.sizes_ok(q, k_pages, v_pages, tables))
    if not _on_gfx950(q):
        raise RuntimeError("HIP backend requires an AMD MI355X (gfx950) GPU")
    hip_paged.require_readable(q, k_pages, v_pages, tables)
    return scale, True


def _sdpa_paged(q, k_pages, v_pages, tables, lengths, causal: bool, scale: float, return_lse: bool):
    b, hq, sq, d = q.shape
    pages, hkv, page, _ = k_pages.shape
    out = torch.zeros((b, hq, sq, d), device=q.device, dtype=q.dtype)
    lse = torch.full((b, hq, sq), -math.inf, device=q.device, dtype=torch.float32)
    for i, n in enumerate(lengths.tolist()):
        n = min(max(n, 0), tables.shape[1] * page)
        ids = tables[i, :-(-n // page)].long().repeat_interleave(page)[:n]
        position = torch.arange(n, device=q.device)
        inside = (ids >= 0) & (ids < pages)
        position, ids = position[inside], ids[inside]
        k, v = (pool[ids, :, position % page].transpose(0, 1)[None] for pool in (k_pages, v_pages))
        # Rows grouped by what they see: all of them alike, or (causal) one
        # group per row.
        for r in range(sq) if causal else [slice(None)]:
            m = int((position < n - (sq - 1 - r)).sum()) if causal else position.numel()
            if m == 0:
                continue
            rows = q[i:i + 1, :, r:r + 1] if causal else q[i:i + 1]
            o = _sdpa(rows, k[:, :, :m], v[:, :, :m], causal=False, scale=scale)
            out[i, :, r] = o[0, :, 0] if causal else o[0]
            if return_lse:
                ke = k[0, :, :m].float().repeat_interleave(hq // hkv, 0)
                s = torch.matmul(rows[0].float(), ke.transpose(-2, -1).contiguous()) * scale
                ls = torch.logsumexp(s, -1)
                lse[i, :, r] = ls[:, 0] if causal else ls
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------

def _positive(name: str, value) -> int:
    if isinstance(value, bool) or not isinstance(value, int) or value <= 0:
        raise ValueError(f"{name} must be a positive integer")
    return value


class PageTable:
    """The pages of every request of a batch, and the free ones, on the GPU.

    ``tables`` (int32 [batch, columns], -1 where a request has no page),
    ``lengths`` (int32 [batch]), ``free_pages`` (int32 [num_pages], a stack)
    with its height ``free_count`` (int32 [1]), and ``refused`` (int32 [1]): the
    requests that the last ``reserve`` left as they were. They may be read, and
    written between calls, by any work on the stream in use; nothing copies
    them to the host except ``num_free`` and ``check``.
    """

    def __init__(self, batch: int, max_len: int, *, num_pages: int, page_size: int = 16,
                 device: Union[torch.device, str] = "cuda") -> None:
        self.batch = _positive("batch", batch)
        self.max_len = _positive("max_len", max_len)
        self.num_pages = _positive("num_pages", num_pages)
        self.page_size = _positive("page_size", page_size)
        columns = -(-max_len // page_size)
        if columns * page_size >= 2 ** 30 or batch * columns >= 2 ** 31 or num_pages >= 2 ** 30:
            raise ValueError("page tables address positions and pages with 32 bits")
        self.tables = torch.full((batch, columns), -1, device=device, dtype=torch.int32)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        # The lowest page is on top.
        self.free_pages = torch.arange(num_pages - 1, -1, -1, device=device, dtype=torch.int32)
        self.counters = torch.tensor([num_pages, 0, 0, 0], device=device, dtype=torch.int32)
        self._views()

    def _views(self) -> None:
        self.free_count = self.counters[0:1]
        self.refused = self.counters[1:2]

    # A copy's or a pickle's views are of its own counters.
    def __getstate__(self) -> dict:
        return {k: v for k, v in self.__dict__.items() if k not in ("free_count", "refused")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._views()

    def num_free(self) -> int:
        """Free pages (waits for the device)."""
        return int(self.free_count)

    def check(self) -> None:
        """RuntimeError if the last ``reserve`` refused a request (waits for
        the device)."""
        if int(self.refused):
            raise RuntimeError(f"page table full: {int(self.refused)} requests found no room "
                               f"({self.num_free()} of {self.num_pages} pages free)")

    def _per_request(self, name: str, value):
        if isinstance(value, torch.Tensor):
            hip_paged._check_int32(name, value, (self.batch,), self.tables.device)
            return value if value.is_contiguous() else value.contiguous()
        if isinstance(value, bool) or not isinstance(value, int):
            raise TypeError(f"{name} must be an int or a device int32 tensor")
        if not 0 <= value < 2 ** 30:
            raise ValueError(f"{name} must be in [0, 2**30)")
        return value

    def _tensor_of(self, value) -> torch.Tensor:
        return value if isinstance(value, torch.Tensor) else torch.full_like(self.lengths, value)

    def reserve(self, counts: Union[int, torch.Tensor], *, width: Optional[int] = None,
                backend: str = "auto") -> torch.Tensor:
        """Room for ``counts`` more tokens (an int for every request, or int32
        [batch] on the device); returns their slots, int64 [batch, width], -1
        behind each request's own. ``lengths`` grow by the counts.

        Requests are served in order. One is refused, and left as it was, when
        its count is outside [0, width], its table has too few columns, or the
        pages asked for by the requests up to it are more than the free ones:
        its slots are all -1 and ``refused`` counts it.
        """
        if backend in ("auto", "hip", "cuda") and not torch.compiler.is_compiling():
            slots = _hip.native().page_reserve(
                self.tables, self.lengths, self.free_pages, self.counters, counts, self.page_size,
                max(counts, 1) if width is None and type(counts) is int else width)
            if slots is not NotImplemented:
                return slots
        counts = self._per_request("counts", counts)
        if width is None:
            if isinstance(counts, torch.Tensor):
                raise ValueError("width is needed with per-request counts")
            width = max(counts, 1)
        width = _positive("width", width)
        if width >= 2 ** 30:
            raise ValueError("width must be below 2**30")
        if not isinstance(counts, torch.Tensor) and counts > width:
            raise ValueError("counts must not exceed width")
        state = (self.tables, self.lengths, self.free_pages, self.counters)
        if _store_on_hip(backend, self.tables, half=False):
            if torch.compiler.is_compiling():
                from .ops import page_reserve_

                return page_reserve_(*state, self._tensor_of(counts), self.page_size, width)
            return hip_paged.reserve_pages(*state, counts, width, self.page_size)
        return _reserve(*state, counts, width, self.page_size)

    def trim(self, lengths: Union[int, torch.Tensor], *, backend: str = "auto") -> None:
        """Every request keeps its first ``lengths`` tokens (an int, or int32
        [batch] on the device; longer than it is: all of them). The pages
        behind go back to the stack, so that the ``reserve`` that took them
        would take the same again."""
        if backend in ("auto", "hip", "cuda") and not torch.compiler.is_compiling() \
                and _hip.native().page_trim(self.tables, self.lengths, self.free_pages, self.counters,
                                            lengths, self.page_size) is None:
            return
        lengths = self._per_request("lengths", lengths)
        state = (self.tables, self.lengths, self.free_pages, self.counters)
        if _store_on_hip(backend, self.tables, half=False):
            if torch.compiler.is_compiling():
                from .ops import page_trim_

                page_trim_(*state, self._tensor_of(lengths), self.page_size)
                return
            hip_paged.trim_pages(*state, lengths, self.page_size)
        else:
            _trim(*state, lengths, self.page_size)


def _bounded(tables, lengths, free_pages, counters, page: int):
    """The stack's height and the requests' lengths as far as they can be true,
    as the kernels bound them."""
    return (counters[0].long().clamp(0, free_pages.numel()),
            lengths.long().clamp(0, tables.shape[1] * page))


def _reserve(tables, lengths, free_pages, counters, counts, width: int, page: int) -> torch.Tensor:
    """``PageTable.reserve`` in torch operations."""
    columns = tables.shape[1]
    height, held = _bounded(tables, lengths, free_pages, counters, page)
    counts = torch.as_tensor(counts, device=tables.device).long().expand_as(held)
    first = (held + page - 1) // page
    fits = (counts >= 0) & (counts <= width) & (held + counts <= columns * page)
    need = torch.where(fits, (held + counts + page - 1) // page - first, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= height))
    need = torch.where(served, need, 0)
    upto = need.cumsum(0)
    column = torch.arange(columns, device=tables.device)
    fresh = (column >= first[:, None]) & (column < (first + need)[:, None])
    place = height - 1 - (upto - need)[:, None] - (column - first[:, None])
    tables[fresh] = free_pages[place[fresh]]
    t = torch.arange(width, device=tables.device)
    position = held[:, None] + t
    ids = tables.long().gather(1, (position // page).clamp(max=columns - 1))
    given = served[:, None] & (t < counts[:, None]) & (ids >= 0) & (ids < free_pages.numel())
    slots = torch.where(given, ids * page + position % page, -1)
    lengths.copy_(torch.where(served, held + counts, lengths))
    counters[0] = height - need.sum()
    counters[1] = (~served).sum()
    return slots


def _trim(tables, lengths, free_pages, counters, new_lengths, page: int) -> None:
    """``PageTable.trim`` in torch operations."""
    height, held = _bounded(tables, lengths, free_pages, counters, page)
    keep = torch.as_tensor(new_lengths, device=tables.device).long().clamp(min=0).minimum(held)
    first, end = (keep + page - 1) // page, (held + page - 1) // page
    freed = end - first
    column = torch.arange(tables.shape[1], device=tables.device)
    gone = (column >= first[:, None]) & (column < end[:, None])
    place = height + freed.sum() - 1 - (freed.cumsum(0) - freed)[:, None] - (column - first[:, None])
    back = gone & (place < free_pages.numel())
    free_pages[place[back]] = tables[back]
    tables.masked_fill_(gone, -1)
    lengths.copy_(keep)
    counters[0] = (height + freed.sum()).clamp(max=free_pages.numel())


class PagedKVCache:
    """One layer's K/V pages, behind a ``PageTable`` that several may share.

    ``k_pages`` and ``v_pages`` are [num_pages, kv_heads, page_size, head_dim].
    The pages hold whatever was there: only rows that were stored are read.
    """

    def __init__(self, table: PageTable, kv_heads: int, head_dim: int, *, dtype: torch.dtype) -> None:
        if not isinstance(table, PageTable):
            raise TypeError("table must be a PageTable")
        shape = (table.num_pages, _positive("kv_heads", kv_heads), table.page_size,
                 _positive("head_dim", head_dim))
        self.table = table
        self.k_pages = torch.empty(shape, device=table.tables.device, dtype=dtype)
        self.v_pages = torch.empty_like(self.k_pages)

    def append(self, new_k, new_v, slots, *, backend: str = "auto") -> None:
        """Store new_k/new_v [B, Hkv, S, D] at the slots that the table's
        ``reserve`` returned (``paged_append``)."""
        paged_append(self.k_pages, self.v_pages, new_k, new_v, slots, backend=backend)

    def attend(self, q, *, causal: bool = False, scale: Optional[float] = None,
               return_lse: bool = False, backend: str = "auto"):
        """Attention of q [B, Hq, Sq, D] over what each request holds
        (``paged_attention``)."""
        return paged_attention(q, self.k_pages, self.v_pages, self.table.tables, self.table.lengths,
                               causal=causal, scale=scale, return_lse=return_lse, backend=backend)

    def append_and_attend(self, q, new_k, new_v, slots, *, causal: bool = False,
                          append_backend: str = "auto", attention_backend: str = "auto"):
        """``append``, then ``attend``: a decoding step of this layer, after
        the table's ``reserve`` of the step.

        ``append_backend="fused"`` stores the new rows from inside the
        attention's launches, to the same effect (HIP attention, up to 16 tokens
        a request and 256 in all); ``"auto"`` takes it for up to 64. The others
        store first, in a launch of their own.
        """
        if append_backend in ("auto", "fused", "hip", "cuda") and attention_backend in ("auto", "hip", "triton") \
                and not torch.compiler.is_compiling():
            how = 2 if append_backend == "fused" else 1 if append_backend == "auto" else 0
            out = _hip.native().paged_step(q, self.k_pages, self.v_pages, self.table.tables,
                                           self.table.lengths, causal, None, new_k, new_v, slots, how)
            if out is not NotImplemented:
                return out
        if append_backend not in STORE_BACKENDS + ("fused",):
            raise ValueError("append backend must be one of: auto, hip, cuda, torch or fused")
        # Every check of the attention comes before the store writes anything.
        scale, on_hip = _attention_route(q, self.k_pages, self.v_pages, self.table.tables,
                                         self.table.lengths, causal, None, attention_backend)
        if append_backend in ("auto", "fused") and on_hip:
            hip_paged.check_append(self.k_pages, self.v_pages, new_k, new_v, slots)
            _no_gradients("paged append", new_k, new_v)
            most = _hip.KF_PAGED_STEP_SLOTS if append_backend == "fused" else hip_paged.FUSED_STEP_ROWS
            if slots.shape[0] == q.shape[0] and hip_paged.step_fuses(self.k_pages, new_k, most):
                if not torch.compiler.is_compiling():
                    return hip_paged.append_attention_paged(
                        q, self.k_pages, self.v_pages, new_k, new_v, slots, self.table.tables,
                        self.table.lengths, causal=causal, scale=scale)
                append_backend = "hip"  # two ops: none stores and attends
        if append_backend == "fused":
            raise ValueError("append_backend='fused' needs HIP attention, up to "
                             f"{_hip.KF_PAGED_STEP_TOKENS} new tokens per request, "
                             f"{_hip.KF_PAGED_STEP_SLOTS} in all, and a pool of fewer than 2**31 slots")
        self.append(new_k, new_v, slots, backend=append_backend)
        return self.attend(q, causal=causal, backend=attention_backend)
