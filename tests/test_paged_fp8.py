"""The 8-bit paged cache on the CPU: the torch path against the definition,
and what is refused."""
import copy
import math

import pytest
import torch

from kotflash_amd.paged import PagedKVCache, PageTable
from kotflash_amd.paged_fp8 import PagedKVCacheFP8, fp8_append, fp8_attention, fp8_read
from tests.fp8_oracle import Cache, assert_attention, make_cache, round_e4m3, scale_of

F16, BF16, F32, FP8 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _randn(*shape, dtype=F16, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _cache(batch=2, hkv=2, d=32, page=32, dtype=F16, max_len=200):
    table = PageTable(batch, max_len, num_pages=batch * -(-max_len // page), page_size=page, device="cpu")
    return PagedKVCacheFP8(table, hkv, d, dtype=dtype)


def test_oracle_rounds_as_torch():
    x = torch.arange(0, 0x7c00, dtype=torch.int32).to(torch.int16).view(F16)
    x = torch.cat((x, -x)).double()
    x = x[x.abs() <= 448]
    assert torch.equal(round_e4m3(x), x.float().to(FP8).double())
    for a, s in ((448, 1), (449, 2), (1, 2.0 ** -8), (0, 2.0 ** -126), (3.3e38, 2.0 ** 120)):
        assert scale_of(a) == s


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_append_and_read(dtype):
    """Prompts, then single tokens and drafts that make blocks grow, through
    the table; every state against the definition."""
    cache = _cache(dtype=dtype)
    table = cache.table
    ref = Cache(cache.k_pages, cache.v_pages, cache.scales)
    rows = torch.zeros(0, dtype=torch.int64)
    for step, (counts, width) in enumerate((((21, 40), 40), ((1, 1), 1), ((3, 0), 4), ((1, 1), 1), ((30, 7), 30))):
        k, v = (_randn(2, 2, width, 32, dtype=dtype, seed=10 * step + i, scale=3.0 ** step) for i in range(2))
        slots = table.reserve(torch.tensor(counts, dtype=torch.int32), width=width)
        cache.append(k, v, slots)
        ref.append(k, v, slots)
        rows = torch.cat((rows, slots[slots >= 0]))
        ref.assert_matches(cache.k_pages, cache.v_pages, cache.scales, rows)
    for width, start in ((70, 0), (5, 17), (100, torch.tensor([50, -3], dtype=torch.int32)), (4, 190), (3, 2 ** 29)):
        starts = start.tolist() if isinstance(start, torch.Tensor) else [start] * 2
        got = cache.read(width, start=start)
        want = ref.read(table.tables, table.lengths, width, starts, dtype)
        for g, w in zip(got, want):
            assert g.dtype == dtype and g.is_contiguous() and torch.equal(g.double(), w)


def test_rounding_error():
    """A value is off by at most 2^-4 of itself, or half the smallest step."""
    cache = _cache(batch=1)
    k = _randn(1, 2, 64, 32, scale=5.0)
    cache.append(k, k, cache.table.reserve(64))
    got = cache.read(64)[0]
    step = cache.scales[0, 0, 0, 0].item() * 2.0 ** -10
    assert bool(((got - k).float().abs() <= k.float().abs() / 16 + 4 * step).all())


def test_new_request_does_not_see_the_old_scale():
    """A block that begins anew has the scale of what comes in."""
    cache = _cache(batch=1)
    big, small = _randn(1, 2, 20, 32, scale=1000.0), _randn(1, 2, 20, 32, seed=1)
    cache.append(big, big, cache.table.reserve(20))
    cache.table.trim(0)
    cache.append(small, small, cache.table.reserve(20))
    other = _cache(batch=1)
    other.append(small, small, other.table.reserve(20))
    assert torch.equal(cache.read(20)[0], other.read(20)[0])


def test_special_values():
    k = torch.zeros(1, 1, 3, 16, dtype=F16)
    k[0, 0, 0, :6] = torch.tensor([math.inf, -math.inf, math.nan, 65504, -65504, 1])
    k[0, 0, 2, 0] = math.inf
    cache = _cache(batch=1, hkv=1, d=16)
    slots = cache.table.reserve(3)
    cache.append(k, k, slots)
    ref = Cache(torch.zeros_like(cache.k_pages), torch.zeros_like(cache.v_pages), torch.zeros_like(cache.scales))
    ref.append(k, k, slots)
    ref.assert_matches(cache.k_pages, cache.v_pages, cache.scales, slots.flatten())
    got = cache.read(3)[0][0, 0]
    assert got[0, :3].isnan().all() and got[0, 3:6].tolist() == [61440, -61440, 1] and bool(got[1].eq(0).all())
    b = torch.full((1, 1, 1, 16), torch.finfo(BF16).max, dtype=BF16)
    cache = _cache(batch=1, hkv=1, d=16, dtype=BF16)
    cache.append(b, -b, cache.table.reserve(1))
    assert float(cache.read(1)[0].max()) == 240 * 2.0 ** 120 and float(cache.read(1)[1].min()) == -240 * 2.0 ** 120


def test_foreign_slots_leave_pools_alone():
    cache = _cache()
    before = cache.k_pages.view(torch.uint8).clone()
    k = _randn(2, 2, 3, 32)
    n = cache.k_pages.shape[0] * 32
    cache.append(k, k, torch.tensor([[-1, n, -2 ** 40], [2 ** 62, -5, n + 7]]))
    assert torch.equal(cache.k_pages.view(torch.uint8), before) and not cache.scales.any()


def test_copies():
    cache = _cache()
    cache.append(_randn(2, 2, 3, 32), _randn(2, 2, 3, 32, seed=1), cache.table.reserve(3))
    other = copy.deepcopy(cache)
    assert all(torch.equal(a, b) for a, b in zip(other.read(3), cache.read(3)))


def test_layers_share_a_table():
    table = PageTable(2, 64, num_pages=8, page_size=16, device="cpu")
    eight, sixteen = PagedKVCacheFP8(table, 2, 32, dtype=F16), PagedKVCache(table, 2, 32, dtype=F16)
    k, v = _randn(2, 2, 5, 32), _randn(2, 2, 5, 32, seed=1)
    slots = table.reserve(5)
    eight.append(k, v, slots)
    sixteen.append(k, v, slots)
    assert (eight.read(5)[0] - k).abs().max() < 0.25


def test_constructor_refusals():
    table = PageTable(1, 64, num_pages=8, page_size=16, device="cpu")
    for args, kw, error, match in [
        ((None, 2, 32), {}, TypeError, "PageTable"), ((table, 0, 32), {}, ValueError, "kv_heads"),
        ((table, 2, 0), {}, ValueError, "head_dim"), ((table, 2, 32), dict(dtype=torch.float64), ValueError, "dtype"),
        ((PageTable(1, 64, num_pages=8, page_size=24, device="cpu"), 2, 32), {}, ValueError, "multiple of 16"),
    ]:
        with pytest.raises(error, match=match):
            PagedKVCacheFP8(*args, **kw)


@pytest.mark.parametrize("change,error,match", [
    (dict(k=1), TypeError, "torch.Tensor"), (dict(k=torch.zeros(4, 2, 16)), ValueError, "matching"),
    (dict(v=torch.zeros(4, 2, 32, 32).to(FP8)), ValueError, "matching"),
    (dict(k=torch.zeros(4, 2, 16, 32)), ValueError, "float8_e4m3fn"),
    (dict(k=torch.zeros(0, 2, 16, 32).to(FP8), v=torch.zeros(0, 2, 16, 32).to(FP8)), ValueError, "non-empty"),
    (dict(k=torch.zeros(4, 2, 24, 32).to(FP8), v=torch.zeros(4, 2, 24, 32).to(FP8)), ValueError, "multiple of 16"),
    (dict(scales=torch.zeros(4, 2, 1)), ValueError, "scales"), (dict(scales=torch.zeros(4, 2, 1, 2).half()), ValueError, "scales"),
    (dict(scales=torch.zeros(1, 1, 1, 2).expand(4, 2, 1, 2)), ValueError, "expanded"),
    (dict(nk=None), TypeError, "new_k"), (dict(nk=torch.zeros(2, 2, 32)), ValueError, "matching"),
    (dict(nk=torch.zeros(2, 2, 0, 32).half(), nv=torch.zeros(2, 2, 0, 32).half()), ValueError, "empty"),
    (dict(nk=torch.zeros(2, 1, 3, 32).half(), nv=torch.zeros(2, 1, 3, 32).half()), ValueError, "heads"),
    (dict(nv=torch.zeros(2, 2, 3, 32)), ValueError, "one dtype"),
    (dict(nk=torch.zeros(2, 2, 3, 32).double(), nv=torch.zeros(2, 2, 3, 32).double()), ValueError, "one dtype"),
    (dict(slots=[[0]]), TypeError, "slots"), (dict(slots=torch.zeros(2, 3, dtype=torch.int32)), ValueError, "slots"),
    (dict(slots=torch.zeros(2, 2, dtype=torch.int64)), ValueError, "slots"), (dict(backend="cuda"), ValueError, "backend"),
    (dict(backend="hip"), RuntimeError, "gfx950"), (dict(nk=torch.zeros(2, 2, 3, 32).half().requires_grad_()), RuntimeError, "inference"),
])
def test_append_refusals(change, error, match):
    a = dict(k=torch.zeros(4, 2, 16, 32).to(FP8), v=torch.zeros(4, 2, 16, 32).to(FP8), scales=torch.zeros(4, 2, 1, 2),
             nk=torch.zeros(2, 2, 3, 32).half(), nv=torch.zeros(2, 2, 3, 32).half(),
             slots=torch.zeros(2, 3, dtype=torch.int64), backend="auto")
    a.update(change)
    backend = a.pop("backend")
    with pytest.raises(error, match=match):
        fp8_append(*a.values(), backend=backend)


@pytest.mark.parametrize("change,error,match", [
    (dict(tables=torch.zeros(2, 2)), ValueError, "int32"), (dict(tables=torch.zeros(2, dtype=torch.int32)), ValueError, "columns"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError, "lengths"), (dict(width=0), ValueError, "width"),
    (dict(width=2 ** 30), ValueError, "width"), (dict(width=True), TypeError, "width"), (dict(width=1.0), TypeError, "width"),
    (dict(start=-1), ValueError, "start"), (dict(start=0.5), TypeError, "start"),
    (dict(start=torch.zeros(2)), ValueError, "start"), (dict(dtype=torch.float64), ValueError, "dtype"),
    (dict(backend="sdpa"), ValueError, "backend"), (dict(backend="hip"), RuntimeError, "gfx950"),
])
def test_read_refusals(change, error, match):
    k, v, scales, tables, lengths = make_cache(2, 2, 32, 16, [3, 20], dtype=F16, seed=0)
    a = dict(tables=tables, lengths=lengths, width=4, start=0, dtype=F16, backend="auto")
    a.update(change)
    with pytest.raises(error, match=match):
        fp8_read(k, v, scales, a["tables"], a["lengths"], a["width"], start=a["start"], dtype=a["dtype"],
                 backend=a["backend"])


def test_cache_takes_its_own_type():
    cache = _cache(dtype=BF16)
    k = _randn(2, 2, 1, 32)
    with pytest.raises(ValueError, match="cache's"):
        cache.append(k, k, cache.table.reserve(1))


def test_tables_that_name_no_page():
    """Positions of a page outside the pool read as zeros; lengths beyond the
    table count as what it holds."""
    k, v, scales, tables, lengths = make_cache(2, 2, 32, 16, [40, 20], dtype=F16, seed=4)
    tables[0, 1], tables[1, 0] = 10 ** 6, -7
    lengths[0] = 1000
    ref = Cache(k, v, scales)
    got = fp8_read(k, v, scales, tables, lengths, 80, dtype=F16)
    want = ref.read(tables, lengths, 80, [0, 0], F16)
    for g, w in zip(got, want):
        assert torch.equal(g.double().nan_to_num(7), w.nan_to_num(7))


@pytest.mark.parametrize("causal", [False, True])
def test_attention(causal):
    """The torch path against the definition, with its bound."""
    k8, v8, scales, tables, lens = make_cache(3, 2, 32, 16, [0, 5, 70], dtype=F16, seed=1, wild=False)
    q = _randn(3, 4, 3, 32)
    k, v = Cache(k8, v8, scales).held(F32)
    o, lse = fp8_attention(q.float(), k8, v8, scales, tables, lens, causal=causal, return_lse=True)
    assert_attention(o, q.float(), k, v, tables, lens, lse=lse, causal=causal)


def test_append_and_attend():
    cache = _cache(dtype=F32, d=32)
    ref = Cache(cache.k_pages, cache.v_pages, cache.scales)
    for step, n in enumerate((20, 1, 3)):
        q, k, v = (_randn(2, h, n, 32, dtype=F32, seed=10 * step + h) for h in (4, 2, 2))
        slots = cache.table.reserve(n)
        o = cache.append_and_attend(q, k, v, slots, causal=True)
        ref.append(k, v, slots)
        assert_attention(o, q, *ref.held(F32), cache.table.tables, cache.table.lengths, causal=True)


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(2, 4, 32)), ValueError, "layout"), (dict(q=torch.zeros(2, 4, 0, 32)), ValueError, "non-empty"),
    (dict(q=torch.zeros(2, 4, 1, 16)), ValueError, "head dimension"), (dict(q=torch.zeros(2, 3, 1, 32)), ValueError, "divisible"),
    (dict(q=torch.zeros(2, 4, 1, 32).double()), ValueError, "float16"), (dict(q=torch.zeros(3, 4, 1, 32)), ValueError, "tables"),
    (dict(causal=1), TypeError, "causal"), (dict(scale="x"), TypeError, "scale"), (dict(scale=math.inf), ValueError, "finite"),
    (dict(backend="torch"), ValueError, "backend"), (dict(backend="hip"), RuntimeError, "gfx950"),
    (dict(q=torch.zeros(2, 4, 1, 32).requires_grad_()), RuntimeError, "inference"),
])
def test_attention_refusals(change, error, match):
    k, v, scales, tables, lengths = make_cache(2, 2, 32, 16, [3, 20], dtype=F16, seed=0)
    a = dict(q=torch.zeros(2, 4, 1, 32))
    a.update(change)
    with pytest.raises(error, match=match):
        fp8_attention(a.pop("q"), k, v, scales, tables, lengths, **a)


def test_step_refuses_before_it_stores():
    cache = _cache()
    slots = cache.table.reserve(1)
    q, k = _randn(2, 4, 1, 32), _randn(2, 2, 1, 32)
    for args, kw in (((q.float(), k, k, slots), {}), ((q, k.float(), k.float(), slots), {}), ((q, k, k, slots), dict(causal=2)),
                     ((q, k, k, slots), dict(append_backend="fused"))):
        with pytest.raises((ValueError, TypeError)):
            cache.append_and_attend(*args, **kw)
        assert not cache.scales.any()
