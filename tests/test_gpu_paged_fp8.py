"""The 8-bit paged cache's kernels on the GPU, against the definition."""
import math

import pytest
import torch

import kotflash_amd.ops  # noqa: F401
from kotflash_amd.kernels import hip_paged_fp8
from kotflash_amd.paged import PageTable
from kotflash_amd.paged_fp8 import PagedKVCacheFP8, fp8_append, fp8_attention, fp8_read
from kotflash_amd.rotary import Rotary
from tests.fp8_oracle import Cache, assert_attention, make_cache

pytestmark = pytest.mark.gpu
F16, BF16, FP8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _randn(*shape, dtype=F16, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _cache(batch, hkv, d, page, max_len, dtype=F16, seed=0):
    table = PageTable(batch, max_len, num_pages=batch * -(-max_len // page) + 2, page_size=page, device="cuda")
    order = torch.randperm(table.num_pages, generator=torch.Generator().manual_seed(seed))
    table.free_pages.copy_(order.to(torch.int32))
    return PagedKVCacheFP8(table, hkv, d, dtype=dtype)


def _same(a, b):
    return torch.equal(a.double().nan_to_num(7), b.to(a.device).double().nan_to_num(7))


# --- store -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 48, 56, 64, 72, 80, 88, 96, 104, 112, 120, 128])
def test_append_dims(dtype, d):
    """Prompts, tokens and drafts that make blocks grow."""
    cache = _cache(3, 2, d, 32, 160, dtype, seed=d)
    table = cache.table
    ref = Cache(cache.k_pages, cache.v_pages, cache.scales)
    rows = torch.zeros(0, dtype=torch.int64)
    for step, (counts, width) in enumerate((((37, 1, 0), 37), ((1, 1, 1), 1), ((2, 5, 0), 5), ((1, 1, 1), 1),
                                            ((40, 17, 33), 40), ((1, 1, 1), 1))):
        k, v = (_randn(3, 2, width, d, dtype=dtype, seed=10 * step + i, scale=2.5 ** step) for i in range(2))
        slots = table.reserve(torch.tensor(counts, dtype=torch.int32, device="cuda"), width=width)
        cache.append(k, v, slots, backend="hip")
        ref.append(k, v, slots)
        rows = torch.cat((rows, slots[slots >= 0].cpu()))
        ref.assert_matches(cache.k_pages, cache.v_pages, cache.scales, rows)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 100])
@pytest.mark.parametrize("first", [0, 1, 15, 16, 21])
def test_append_lengths(n, first):
    """Runs that begin and end anywhere in a block and in a window."""
    cache = _cache(2, 3, 64, 16, 160, BF16, seed=n)
    ref = Cache(cache.k_pages, cache.v_pages, cache.scales)
    rows = []
    for i, width in enumerate((first, n)):
        if width:
            k, v = (_randn(2, 3, width, 64, dtype=BF16, seed=i + j, scale=10.0 ** i) for j in range(2))
            slots = cache.table.reserve(width)
            cache.append(k, v, slots, backend="hip")
            ref.append(k, v, slots)
            rows.append(slots.flatten().cpu())
    ref.assert_matches(cache.k_pages, cache.v_pages, cache.scales, torch.cat(rows))


def test_append_any_slots():
    """Single tokens and runs at any slots of different blocks, slots outside
    the pool among them; everything else stays as it was."""
    k8, v8, scales, _, _ = make_cache(1, 4, 128, 48, [48 * 40], dtype=F16, seed=3, device="cuda")
    ref = Cache(k8, v8, scales)
    places = k8.shape[0] * 48
    g = torch.Generator().manual_seed(1)
    blocks = torch.randperm(places // 16, generator=g)[:90].view(6, 15)
    slots = blocks * 16 + torch.randint(0, 16, blocks.shape, generator=g)
    slots[0, ::4], slots[1, 3], slots[2, 0], slots[3, 14] = -1, places, -2 ** 40, 2 ** 62
    slots[4, 4:9] = int(blocks[4, 4]) * 16 + torch.tensor([7, 3, 12, 0, 9])  # a run in no order
    k, v = _randn(6, 4, 15, 128, scale=30.0), _randn(6, 4, 15, 128, seed=1, scale=0.01)
    fp8_append(k8, v8, scales, k, v, slots.cuda(), backend="hip")
    ref.append(k, v, slots)
    ref.assert_matches(k8, v8, scales)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_special_values(dtype):
    k = torch.zeros(2, 1, 18, 64, dtype=dtype)
    k[0, 0, 0, :8] = torch.tensor([math.inf, -math.inf, math.nan, torch.finfo(dtype).max, -torch.finfo(dtype).max, 1,
                                   torch.finfo(dtype).smallest_normal, -0.0])
    k[0, 0, 17, 3] = math.inf
    k[1, 0, 0] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps * torch.arange(-32, 32)
    k[1, 0, 16] = torch.linspace(-448, 448, 64)
    k[1, 0, 17] = 448.5
    v = k.flip(3)
    cache = _cache(2, 1, 64, 16, 64, dtype)
    slots = cache.table.reserve(18)
    ref = Cache(cache.k_pages, cache.v_pages, cache.scales)
    cache.append(k.cuda(), v.cuda(), slots, backend="hip")
    ref.append(k, v, slots)
    ref.assert_matches(cache.k_pages, cache.v_pages, cache.scales, slots.flatten().cpu())
    # A grown block with NaN in it, and one that nothing was stored to.
    for n, scale in ((1, 300.0), (1, 0.0)):
        k = (_randn(2, 1, n, 64, dtype=dtype) * scale).nan_to_num(0, 1, 1)
        slots = torch.cat((slots, cache.table.reserve(n)), 1)
        cache.append(k, k, slots[:, -n:], backend="hip")
        ref.append(k, k, slots[:, -n:])
        ref.assert_matches(cache.k_pages, cache.v_pages, cache.scales, slots.flatten().cpu())


def test_append_layouts():
    """Transposed views, rows off 16-byte borders, strided pools and slots."""
    shape = (6, 2, 32, 64)
    wide = torch.zeros(6, 2, 2, 32, 128, dtype=torch.uint8, device="cuda").view(FP8)
    k8, v8 = wide[:, 0, :, :, :64], wide[:, 1, :, :, 64:]
    scales = torch.zeros(6, 3, 2, 2, 2, device="cuda")[:, 1]
    assert k8.shape == shape and not k8.is_contiguous()
    ref = Cache(k8, v8, scales)
    k, v = _randn(3, 20, 2, 64).transpose(1, 2), _randn(3, 2, 20, 68, seed=1)[..., 4:]
    slots = torch.arange(0, 60, device="cuda").view(3, 20) + torch.tensor([[0], [12 + 32], [24 + 64]], device="cuda")
    other = torch.stack((slots, slots), 2)[..., 0]
    fp8_append(k8, v8, scales, k, v, other, backend="hip")
    ref.append(k, v, slots)
    ref.assert_matches(k8, v8, scales)
    beside = wide.view(torch.uint8).clone()
    beside[:, 0, :, :, :64] = beside[:, 1, :, :, 64:] = 0
    assert not beside.any()


# --- read --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,page", [(8, 16), (16, 16), (40, 48), (48, 48), (64, 16), (72, 16), (80, 32), (128, 16), (128, 256)])
def test_read(dtype, d, page):
    lengths = [0, 1, 15, 16, 17, 100, 300]
    k8, v8, scales, tables, lens = make_cache(7, 2, d, page, lengths, dtype=dtype, seed=d, device="cuda")
    tables[5, 0] = -3
    tables[6, 0] = 10 ** 6
    ref = Cache(k8, v8, scales)
    starts = torch.tensor([0, -5, 3, 16, 10 ** 9, 41, 250], dtype=torch.int32, device="cuda")
    for width, start in ((1, 0), (37, 0), (300, 0), (40, 90), (64, starts), (5, 2 ** 29)):
        first = starts.tolist() if isinstance(start, torch.Tensor) else [start] * 7
        got = fp8_read(k8, v8, scales, tables, lens, width, start=start, dtype=dtype, backend="hip")
        want = ref.read(tables.cpu(), lens, width, first, dtype)
        for g, w in zip(got, want):
            assert g.dtype == dtype and g.is_contiguous() and _same(w, g.cpu())


def test_read_codes_and_scales():
    """Every code, scales from end to end of the type."""
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 16, 16).expand(31, 1, 16, 16).contiguous().cuda().view(FP8)
    for dtype, low, high in ((F16, -33, 8), (BF16, -126, 120)):
        scales = torch.exp2(torch.linspace(low, high, 31).round()).view(31, 1, 1, 1).expand(31, 1, 1, 2).contiguous().cuda()
        tables = torch.arange(31, dtype=torch.int32, device="cuda")[None]
        lens = torch.tensor([31 * 16], dtype=torch.int32, device="cuda")
        k, v = fp8_read(codes, codes, scales, tables, lens, 31 * 16, dtype=dtype, backend="hip")
        want = (codes.cpu().float().double() * scales.cpu().double()[..., :1]).to(dtype)
        assert _same(want.view(496, 16), k[0, 0].cpu()) and torch.equal(k.view(torch.int16), v.view(torch.int16))


def test_paths_agree():
    """The native call, the ctypes one, the op and torch.compile."""
    args = make_cache(3, 2, 64, 32, [40, 7, 90], dtype=F16, seed=2, device="cuda")
    want = fp8_read(*args, 90, dtype=F16)
    pools, start = args[:3], torch.zeros(3, dtype=torch.int32, device="cuda")
    for got in (hip_paged_fp8.read_fp8(*args, 90, 0, F16), hip_paged_fp8.read_fp8(*args, 90, start, F16),
                torch.ops.kotflash_amd.fp8_read(*args, start, 90, F16),
                torch.compile(lambda *a: fp8_read(*a, 90, dtype=F16), fullgraph=True, backend="aot_eager")(*args)):
        assert all(_same(a, b) for a, b in zip(want, got))
    k, v = _randn(3, 2, 4, 64), _randn(3, 2, 4, 64, seed=1)
    slots = (torch.arange(12, device="cuda") * 16 + 5).view(3, 4)
    results = []
    for store in (fp8_append, hip_paged_fp8.append_fp8, torch.ops.kotflash_amd.fp8_append_,
                  torch.compile(fp8_append, fullgraph=True, backend="aot_eager")):
        mine = [t.clone() for t in pools]
        store(*mine, k, v, slots)
        results.append([mine[0].view(torch.uint8), mine[1].view(torch.uint8), mine[2]])
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], r))


def test_versions_and_refusals():
    k8, v8, scales, tables, lens = make_cache(2, 2, 64, 16, [5, 20], dtype=F16, seed=2, device="cuda")
    k, slots = _randn(2, 2, 1, 64), torch.tensor([[0], [16]], device="cuda")
    before = [t._version for t in (k8, v8, scales)]
    fp8_append(k8, v8, scales, k, k, slots)
    assert all(t._version > n for t, n in zip((k8, v8, scales), before))
    # Rows of 24 bytes without their padding, and at the end of the storage.
    with pytest.raises(ValueError, match="16-byte aligned"):
        odd = [torch.zeros(2, 1, 16, 24, device="cuda").to(FP8) for _ in range(2)]
        fp8_read(*odd, torch.zeros(2, 1, 1, 2, device="cuda"), tables, lens, 4, dtype=F16, backend="hip")
    with pytest.raises(TypeError, match="float16 and bfloat16"):
        fp8_read(k8, v8, scales, tables, lens, 4, dtype=torch.float32, backend="hip")
    with pytest.raises(RuntimeError, match="inference"):
        fp8_append(k8, v8, scales, k.clone().requires_grad_(), k, slots)
    with pytest.raises(ValueError, match="device"):
        fp8_append(k8, v8, scales, k, k, slots.cpu())
    with pytest.raises(ValueError, match="16-byte aligned"):
        short = torch.zeros(2 * 16 * 32 - 8, dtype=torch.uint8, device="cuda").view(FP8)
        odd = [short.as_strided((2, 1, 16, 24), (512, 512, 32, 1)) for _ in range(2)]
        fp8_read(*odd, torch.zeros(2, 1, 1, 2, device="cuda"), tables, lens, 4, dtype=F16, backend="hip")
    # What the kernels do not take, auto runs in torch.
    odd = [torch.zeros(2, 1, 16, 24, device="cuda").to(FP8) for _ in range(2)]
    sc = torch.zeros(2, 1, 1, 2, device="cuda")
    new = _randn(2, 1, 1, 24)
    ref = Cache(*odd, sc)
    fp8_append(*odd, sc, new, new, slots)
    ref.append(new, new, slots)
    ref.assert_matches(*odd, sc)


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GiB: pages at its far end."""
    pages = (5 << 30) // (2 * 16 * 128)
    k8 = torch.empty(pages, 2, 16, 128, dtype=torch.uint8, device="cuda").view(FP8)
    v8 = torch.empty_like(k8)
    scales = torch.zeros(pages, 2, 1, 2, device="cuda")
    tables = torch.tensor([[pages - 1, 3, pages - 7]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([43], dtype=torch.int32, device="cuda")
    t = torch.arange(43, device="cuda")
    slots = (tables[0].long()[t // 16] * 16 + t % 16)[None]
    k, v = _randn(1, 2, 43, 128), _randn(1, 2, 43, 128, seed=1)
    fp8_append(k8, v8, scales, k, v, slots, backend="hip")
    small = [torch.zeros(3, 2, 16, 128, device="cuda").to(FP8) for _ in range(2)]
    ss = torch.zeros(3, 2, 1, 2, device="cuda")
    fp8_append(*small, ss, k, v, t[None], backend="torch")
    got = fp8_read(k8, v8, scales, tables, lens, 43, dtype=F16, backend="hip")
    want = fp8_read(*small, ss, torch.arange(3, dtype=torch.int32, device="cuda")[None], lens, 43, dtype=F16, backend="torch")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph_replays():
    """A captured reserve, append and read follows the requests as they grow."""
    cache = _cache(2, 2, 64, 16, 200)
    table = cache.table
    k, v = _randn(2, 2, 3, 64), _randn(2, 2, 3, 64, seed=1)

    def call():
        slots = table.reserve(3)
        cache.append(k, v, slots)
        return cache.read(32)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    table.trim(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    ref = _cache(2, 2, 64, 16, 200)
    for step in range(6):
        k.copy_(_randn(2, 2, 3, 64, seed=step, scale=1.5 ** step))
        v.copy_(_randn(2, 2, 3, 64, seed=step + 50))
        graph.replay()
        torch.cuda.synchronize()
        slots = ref.table.reserve(3)
        ref.append(k, v, slots)
        want = ref.read(32)
        assert all(torch.equal(a, b) for a, b in zip(held, want))


# --- attention ---------------------------------------------------------------

def _case(batch, hq, hkv, sq, d, page, lengths, *, dtype, seed, wild=False):
    pools = make_cache(batch, hkv, d, page, lengths, dtype=dtype, seed=seed, device="cuda", wild=wild)
    return (_randn(batch, hq, sq, d, dtype=dtype, seed=seed + 1), *pools)


def _check(case, causal=False, scale=None, **kw):
    q, k8, v8, scales, tables, lens = case
    o, lse = fp8_attention(*case, causal=causal, scale=scale, return_lse=True, backend="hip", **kw)
    k, v = Cache(k8, v8, scales).held(q.dtype)
    assert_attention(o, q, k, v, tables, lens, lse=lse, causal=causal, scale=scale)
    return o, lse


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 88, 96, 104, 112, 120, 128])
@pytest.mark.parametrize("wild", [False, True])
def test_attention_dims(dtype, d, wild):
    _check(_case(4, 8, 2, 1, d, 16, [1, 70, 333, 1000], dtype=dtype, seed=d, wild=wild))


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 79, 80, 127, 128, 129, 257])
@pytest.mark.parametrize("page", [16, 48])
def test_attention_lengths(length, page):
    """One request alone, and beside others."""
    _check(_case(1, 4, 2, 1, 64, page, [length], dtype=F16, seed=length))
    _check(_case(5, 4, 2, 1, 128, page, [length, 0, 40, length, 0], dtype=BF16, seed=length))


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 112, 256, 1024])
def test_attention_page_sizes(page):
    _check(_case(3, 8, 4, 1, 64, page, [page - 1, page, 3 * page + 5], dtype=F16, seed=page))


@pytest.mark.parametrize("hq,hkv,sq", [(1, 1, 1), (16, 1, 1), (17, 1, 1), (28, 4, 1), (33, 1, 1), (64, 1, 1),
                                       (65, 1, 1), (8, 8, 3), (8, 2, 5), (16, 2, 4), (32, 2, 16), (4, 1, 40)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_rows(hq, hkv, sq, causal, d):
    """1 to 256 packed rows per KV head: one, two and four waves, and several
    row groups; causal rows of which the first see nothing."""
    _check(_case(4, hq, hkv, sq, d, 16, [3, 0, 100, 259], dtype=F16, seed=hq + sq), causal=causal)


@pytest.mark.parametrize("batch", [63, 64, 65, 200])
def test_attention_batches(batch):
    """Runs of units over many requests, empty ones among them."""
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 300, (batch,), generator=g).tolist()
    lengths[::7] = [0] * len(lengths[::7])
    _check(_case(batch, 4, 2, 1, 64, 32, lengths, dtype=BF16, seed=batch))


@pytest.mark.parametrize("hq,hkv,d,n", [(8, 8, 128, 70000), (16, 1, 64, 200000), (32, 1, 96, 40000)])
def test_attention_long(hq, hkv, d, n):
    """Runs of many units: one request over all workers, and beside a short."""
    _check(_case(2, hq, hkv, 1, d, 64, [n, 100], dtype=BF16, seed=n))


@pytest.mark.parametrize("sq", [2, 4, 16])
@pytest.mark.parametrize("rest", [0, 1, 15, 16, 17, 40, 63])
def test_attention_drafts(sq, rest):
    """Causal limits anywhere in a step of 64 positions."""
    _check(_case(3, 8, 2, sq, 128, 16, [128 + rest, 64 + rest, rest], dtype=F16, seed=sq + rest), causal=True)


def test_attention_scales():
    case = _case(2, 4, 2, 1, 64, 16, [70, 200], dtype=F16, seed=5)
    for scale in (0.0, 1.0, -0.5, 1e-4):
        _check(case, scale=scale)


def test_attention_empty_batch_and_rows():
    o, lse = _check(_case(3, 4, 2, 2, 64, 16, [0, 0, 0], dtype=F16, seed=1), causal=True)
    assert not o.any() and bool((lse == -math.inf).all())


def test_attention_junk_is_not_read():
    """NaN codes behind a request's last row, pages of nobody, page numbers
    outside the pool, and lengths beyond the table or below zero."""
    q, k8, v8, scales, tables, lens = _case(4, 8, 2, 1, 64, 32, [100, 40, 64, 7], dtype=F16, seed=3)
    scales[k8.view(torch.uint8).eq(127).all(-1).all(-1).all(-1)] = math.nan
    tables[0, 1], tables[1, 0] = 10 ** 6, -2 ** 31
    lens[2], lens[3] = 10 ** 6, -5
    tables[2, 2:] = -1
    o, lse = fp8_attention(q, k8, v8, scales, tables, lens, return_lse=True, backend="hip")
    k, v = Cache(k8, v8, scales.nan_to_num(1)).held(F16)
    assert_attention(o, q, k, v, tables, lens, lse=lse)


@pytest.mark.parametrize("where", ["key", "value"])
def test_attention_nan_in_sight(where):
    """A NaN that a row sees makes it NaN; causal rows in front of it, and the
    other requests and heads, stay as they are."""
    q, k8, v8, scales, tables, lens = _case(2, 4, 2, 4, 128, 16, [90, 90], dtype=F16, seed=9)
    clean, clean_lse = fp8_attention(q, k8, v8, scales, tables, lens, causal=True, return_lse=True, backend="hip")
    pool = (k8 if where == "key" else v8).view(torch.uint8)
    pool[int(tables[0, 88 // 16]), 1, 88 % 16, 5] = 0x7f
    o, lse = fp8_attention(q, k8, v8, scales, tables, lens, causal=True, return_lse=True, backend="hip")
    assert torch.equal(o[1], clean[1]) and torch.equal(o[0, :2], clean[0, :2])
    assert torch.equal(o[0, 2:, :2], clean[0, 2:, :2])  # rows that see up to 86 and 87
    if where == "key":
        assert o[0, 2:, 2:].isnan().all() and not lse[0, 2:, 2:].isfinite().any()
    else:
        assert o[0, 2:, 2:, 5].isnan().all() and o[0, 2:, 2:, 6:].isfinite().all()


def test_attention_repeats_bit_for_bit():
    case = _case(5, 32, 4, 1, 128, 16, [4000, 1, 900, 0, 2500], dtype=BF16, seed=2)
    first = fp8_attention(*case, return_lse=True)
    for _ in range(5):
        again = fp8_attention(*case, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_attention_layouts():
    """Strided queries, tables and pools."""
    q, k8, v8, scales, tables, lens = _case(3, 8, 2, 2, 64, 16, [50, 130, 9], dtype=F16, seed=4)
    want = fp8_attention(q, k8, v8, scales, tables, lens, return_lse=True, backend="hip")
    q2 = q.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.stack((k8.view(torch.uint8), v8.view(torch.uint8)), 1).view(FP8)
    sc2 = torch.stack((scales, scales), 1)[:, 1]
    t2 = torch.stack((tables, tables), 2)[..., 0]
    l2 = torch.stack((lens, lens), 1)[:, 0]
    for args in ((q2, wide[:, 0], wide[:, 1], sc2, tables, lens), (q, k8, v8, scales, t2, l2),
                 (torch.cat((q, q), 3)[..., :64], k8, v8, scales, tables, lens)):
        got = fp8_attention(*args, return_lse=True, backend="hip")
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_attention_paths_agree():
    case = _case(3, 8, 2, 2, 64, 16, [50, 130, 9], dtype=F16, seed=4)
    want = fp8_attention(*case, causal=True, return_lse=True)
    got = hip_paged_fp8.attention_fp8(*case, causal=True, scale=0.125, with_lse=True)
    op = torch.ops.kotflash_amd.fp8_decode(*case, True, 0.125)
    compiled = torch.compile(lambda *a: fp8_attention(*a, causal=True, return_lse=True), fullgraph=True,
                             backend="aot_eager")(*case)
    for other in (got, op, compiled):
        assert all(torch.equal(a, b) for a, b in zip(want, other))
    sdpa = fp8_attention(*case, causal=True, return_lse=True, backend="sdpa")
    assert (sdpa[0] - want[0]).abs().max() < 4e-3 and (sdpa[1] - want[1]).abs().max() < 2e-3
    # What the kernels do not take, auto runs there.
    odd = make_cache(2, 1, 24, 16, [5, 30], dtype=F16, seed=1, device="cuda")
    odd = (*(t.view(torch.uint8).contiguous().view(FP8) for t in odd[:2]), *odd[2:])
    out = fp8_attention(_randn(2, 4, 1, 24), *odd)
    assert_attention(out, _randn(2, 4, 1, 24), *Cache(*odd[:3]).held(F16), *odd[3:])
    with pytest.raises(ValueError, match="16-byte aligned"):
        fp8_attention(_randn(2, 4, 1, 24), *odd, backend="hip")
    # Pools of different strides: attention needs them alike.
    q, k8, v8, scales, tables, lens = case
    other = torch.cat((v8.view(torch.uint8),) * 2, 3).view(FP8)[..., :64]
    got = fp8_attention(q, k8, other, scales, tables, lens, causal=True, return_lse=True)
    assert (got[0] - want[0]).abs().max() < 4e-3
    with pytest.raises(RuntimeError, match="same strides"):
        fp8_attention(q, k8, other, scales, tables, lens, backend="hip")


def test_attention_beyond_32_bits():
    """Pages at the far end of a pool of more than 4 GiB."""
    pages = (5 << 30) // (2 * 16 * 128)
    k8 = torch.empty(pages, 2, 16, 128, dtype=torch.uint8, device="cuda").view(FP8)
    v8 = torch.empty_like(k8)
    scales = torch.empty(pages, 2, 1, 2, device="cuda")
    q, ks, vs, sc, tables, lens = _case(1, 4, 2, 1, 128, 16, [70], dtype=F16, seed=1)
    far = tables.clone()
    for c in range(5):
        p, to = int(tables[0, c]), pages - 1 - 3 * c
        far[0, c] = to
        for pool, small in ((k8, ks), (v8, vs)):
            pool.view(torch.uint8)[to] = small.view(torch.uint8)[p]
        scales[to] = sc[p]
    assert torch.equal(fp8_attention(q, k8, v8, scales, far, lens), fp8_attention(q, ks, vs, sc, tables, lens))


# --- a step ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
def test_steps_of_a_server(dtype):
    """Rotary positions, room, store and attention together, as requests come,
    grow and leave; against the definition over what the cache holds."""
    batch, hq, hkv, d = 3, 8, 2, 64
    cache = _cache(batch, hkv, d, 32, 300, dtype)
    rot = Rotary(d, base=500.0)
    ref = Cache(cache.k_pages, cache.v_pages, cache.scales)
    table = cache.table
    for step, (counts, width) in enumerate((((70, 100, 0), 100), ((1, 1, 1), 1), ((4, 2, 3), 4), ((1, 1, 1), 1), ((0, 0, 90), 90),
                                            ((1, 1, 1), 1))):
        if step == 3:
            table.trim(torch.tensor([73, 102, 0], dtype=torch.int32, device="cuda"))
        if step == 4:
            table.trim(torch.tensor([0, 2 ** 20, 1], dtype=torch.int32, device="cuda"))
        q, k, v = (_randn(batch, h, width, d, dtype=dtype, seed=10 * step + i) for i, h in enumerate((hq, hkv, hkv)))
        q, k = rot(q, k, positions=table.lengths)
        slots = table.reserve(torch.tensor(counts, dtype=torch.int32, device="cuda"), width=width)
        o = cache.append_and_attend(q, k, v, slots)
        ref.append(k, v, slots)
        kd, vd = ref.held(dtype)
        assert_attention(o, q, kd, vd, table.tables, table.lengths)
        apart = cache.attend(q, return_lse=True)
        assert torch.equal(o, apart[0])


def test_step_refuses_before_it_stores():
    cache = _cache(2, 2, 64, 16, 100)
    slots = cache.table.reserve(1)
    before = cache.scales.clone()
    q, k = _randn(2, 4, 1, 64), _randn(2, 2, 1, 64)
    for bad, error in ((dict(q=q.float()), ValueError), (dict(q=q[:, :3]), ValueError), (dict(causal=1), TypeError),
                       (dict(attention_backend="x"), ValueError), (dict(append_backend="fused"), ValueError),
                       (dict(new_k=k.bfloat16(), new_v=k.bfloat16()), ValueError), (dict(slots=slots.int()), ValueError)):
        args = {"q": q, "new_k": k, "new_v": k, "slots": slots, **bad}
        with pytest.raises(error):
            cache.append_and_attend(args.pop("q"), args.pop("new_k"), args.pop("new_v"), args.pop("slots"), **args)
        assert torch.equal(cache.scales, before)


def test_step_graph_replays():
    """A captured step follows the requests as they grow."""
    cache, plain = (_cache(2, 2, 64, 16, 300) for _ in range(2))
    rot = Rotary(64)
    q0, k0, v0 = _randn(2, 8, 1, 64), _randn(2, 2, 1, 64, seed=1), _randn(2, 2, 1, 64, seed=2)

    def step(c):
        q, k = rot(q0, k0, positions=c.table.lengths)
        slots = c.table.reserve(1)
        return c.append_and_attend(q, k, v0, slots)

    for c in (cache, plain):
        k = _randn(2, 2, 120, 64, seed=7)
        c.append(k, k, c.table.reserve(120))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(cache)
    torch.cuda.current_stream().wait_stream(stream)
    cache.table.trim(120)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(cache)
    for i in range(20):
        for t, s in ((q0, 0), (k0, 1), (v0, 2)):
            t.copy_(_randn(*t.shape, seed=100 * i + s))
        graph.replay()
        torch.cuda.synchronize()
        want = step(plain)
        assert torch.equal(held, want), i


def test_step_under_compile():
    """A step is one graph of its ops, to the same bits."""
    caches = [_cache(2, 2, 64, 16, 300) for _ in range(2)]
    rot = Rotary(64)
    q, k, v = _randn(2, 8, 1, 64), _randn(2, 2, 1, 64, seed=1), _randn(2, 2, 1, 64, seed=2)

    def step(c, q, k, v):
        q, k = rot(q, k, positions=c.table.lengths)
        return c.append_and_attend(q, k, v, c.table.reserve(1))

    compiled = torch.compile(lambda *a: step(caches[0], *a), fullgraph=True, backend="aot_eager")
    for c in caches:
        old = _randn(2, 2, 90, 64, seed=7)
        c.append(old, old, c.table.reserve(90))
    with torch.no_grad():
        for _ in range(3):
            assert torch.equal(compiled(q, k, v), step(caches[1], q, k, v))
    assert torch.equal(caches[0].scales, caches[1].scales)


def test_tables_made_in_inference_mode():
    with torch.inference_mode():
        cache = _cache(2, 2, 64, 16, 100)
        k = _randn(2, 2, 20, 64)
        cache.append(k, k, cache.table.reserve(20))
        out = cache.append_and_attend(_randn(2, 4, 1, 64), k[:, :, :1], k[:, :, :1], cache.table.reserve(1))
    assert out.isfinite().all()


def test_calls_on_two_streams():
    """Caches of their own, on streams of their own, at the same time."""
    caches = [_cache(4, 2, 128, 16, 3000, BF16, seed=i) for i in range(2)]
    q = [_randn(4, 8, 1, 128, dtype=BF16, seed=i) for i in range(2)]
    for i, c in enumerate(caches):
        k = _randn(4, 2, 2900, 128, dtype=BF16, seed=10 + i)
        c.append(k, k, c.table.reserve(2900))
    want = [c.attend(x) for c, x in zip(caches, q)]
    streams = [torch.cuda.Stream() for _ in caches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(caches[i].attend(q[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(got, want) for o in os)


@pytest.mark.parametrize("seed", range(12))
def test_random_shapes(seed):
    import random

    rng = random.Random(seed)
    dtype = rng.choice([F16, BF16])
    d, page = 8 * rng.randint(1, 16), 16 * rng.choice([1, 2, 3, 5, 8])
    hkv = rng.choice([1, 2, 3, 8])
    hq, sq = hkv * rng.choice([1, 2, 5, 8, 16]), rng.choice([1, 1, 2, 3, 7])
    lengths = [rng.choice([0, 1, rng.randint(1, 100), rng.randint(1, 2000)]) for _ in range(rng.randint(1, 9))]
    print(dtype, d, page, hkv, hq, sq, lengths, flush=True)
    _check(_case(len(lengths), hq, hkv, sq, d, page, lengths, dtype=dtype, seed=seed), causal=rng.random() < 0.5)
