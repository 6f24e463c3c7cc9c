"""The paged cache's kernels on the GPU, against the definition in 64 bits."""
import math
import random

import pytest
import torch

from kotflash_amd import _hip
from kotflash_amd.paged import PagedKVCache, PageTable, paged_append, paged_attention
from tests.paged_oracle import Pages, assert_attention, make_case

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _attend(*args, **kw):
    return paged_attention(*args, backend="hip", return_lse=True, **kw)


def _check(case, **kw):
    o, lse = _attend(*case, **kw)
    assert_attention(o, *case, lse=lse, **kw)
    return o, lse


# --- attention ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 80, 96, 104, 128])
def test_head_dims(dtype, d):
    _check(make_case(4, 8, 2, 1, d, 16, [1, 70, 333, 1000], dtype=dtype, seed=d, device="cuda"))


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 127, 128, 129, 257])
@pytest.mark.parametrize("page", [16, 48])
def test_lengths(length, page):
    """One request alone, and beside others."""
    _check(make_case(1, 4, 2, 1, 64, page, [length], dtype=F16, seed=length, device="cuda"))
    _check(make_case(5, 4, 2, 1, 128, page, [length, 0, 40, length, 0], dtype=BF16, seed=length, device="cuda"))


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 256, 1024])
def test_page_sizes(page):
    _check(make_case(3, 8, 4, 1, 64, page, [page - 1, page, 3 * page + 5], dtype=F16, seed=page, device="cuda"))


@pytest.mark.parametrize("hq,hkv,sq", [(1, 1, 1), (16, 1, 1), (17, 1, 1), (28, 4, 1), (33, 1, 1), (64, 1, 1),
                                       (65, 1, 1), (8, 8, 3), (8, 2, 5), (16, 2, 4), (32, 2, 16), (4, 1, 40)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_rows(hq, hkv, sq, causal, d):
    """1 to 256 packed rows per KV head: one to four row blocks, and several
    row groups; causal rows of which the first see nothing."""
    _check(make_case(4, hq, hkv, sq, d, 16, [3, 0, 100, 259], dtype=F16, seed=hq + sq, device="cuda"), causal=causal)


@pytest.mark.parametrize("batch", [63, 64, 65, 200])
def test_batches(batch):
    """Runs of units over many requests, empty ones among them."""
    rng = random.Random(batch)
    lengths = [rng.choice([0, 0, 1, rng.randint(1, 400)]) for _ in range(batch)]
    _check(make_case(batch, 4, 2, 1, 64, 16, lengths, dtype=F16, seed=batch, device="cuda"))
    _check(make_case(batch, 2, 1, 1, 32, 16, [0] * batch, dtype=BF16, seed=batch, device="cuda"))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_long(dtype):
    """Runs of several steps per worker, requests cut anywhere."""
    _check(make_case(3, 4, 1, 1, 128, 16, [40000, 7, 29999], dtype=dtype, seed=8, device="cuda"))


def test_runs_over_many_segments():
    """More steps than workers, and many short requests: a run holds whole
    requests between two parts of others."""
    rng = random.Random(5)
    lengths = [rng.randint(0, 90) for _ in range(700)]
    lengths[300] = 20000
    _check(make_case(700, 8, 8, 1, 32, 16, lengths, dtype=F16, seed=5, device="cuda"))


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-3])
def test_scales(scale):
    _check(make_case(2, 4, 2, 2, 64, 16, [50, 333], dtype=F16, seed=2, device="cuda"), scale=scale, causal=True)


def test_large_scores():
    """Scores of several hundred, growing along the keys: the running maximum
    moves at every step."""
    q, k, v, tables, lengths = make_case(1, 4, 2, 1, 64, 16, [640], dtype=F16, seed=2, device="cuda", values=2.0)
    for c in range(40):
        k[tables[0, c]] *= 0.2 * c
    _check((q, k, v, tables, lengths), scale=0.5)


def test_small_probabilities_of_a_long_tail():
    """One key far above thousands of equal ones, whose P lie below the
    smallest fp16 number: together they still count."""
    q, k, v, tables, lengths = make_case(1, 1, 1, 1, 64, 16, [30000], dtype=F16, seed=2, device="cuda")
    q.fill_(1.0)
    k.zero_()
    v.fill_(1.0)
    first = int(tables[0, 0])
    k[first, 0, 0] = 18.0 / 64
    v[first, 0, 0] = 0.0
    # exp(-18) = 2^-26 each: 30000 of them are 4.6e-4 of the sum.
    o, lse = _check((q, k, v, tables, lengths), scale=1.0)
    assert (o > 3e-4).all()


def test_what_lies_behind_is_not_read():
    """NaN, infinities and the type's lowest value behind every request's end
    and in the pages of nobody change no bit."""
    for causal in (False, True):
        got = []
        for junk in (0.0, math.nan, math.inf, torch.finfo(BF16).min):
            case = make_case(3, 8, 2, 2, 96, 32, [5, 64, 201], dtype=BF16, seed=6, device="cuda", junk=junk)
            got.append(_attend(*case, causal=causal))
        for o, lse in got[1:]:
            assert torch.equal(o, got[0][0]) and torch.equal(lse, got[0][1])


def test_nan_and_infinity_in_sight():
    """A visible NaN reaches its request's rows and no others; a value that is
    infinite reaches its column."""
    q, k, v, tables, lengths = make_case(3, 4, 2, 1, 64, 16, [100, 100, 100], dtype=F16, seed=6, device="cuda")
    k[tables[1, 2], 0, 3, 5] = math.nan
    v[tables[2, 0], 1, 0, 7] = math.inf
    o = _attend(q, k, v, tables, lengths)[0]
    assert torch.isnan(o[1, :2]).all()
    assert torch.isinf(o[2, 2:, 0, 7]).all()
    rest = o.clone()
    rest[1, :2] = 0
    rest[2, 2:, 0, 7] = 0
    assert torch.isfinite(rest).all()


def test_pages_outside_the_pool():
    q, k, v, tables, lengths = make_case(4, 4, 2, 1, 64, 16, [100, 16, 500, 31], dtype=F16, seed=4, device="cuda")
    tables[0, 1], tables[1, 0], tables[2, 31] = k.shape[0], -1, 2 ** 31 - 1
    tables[2, 3:9] = -2 ** 31
    tables[3, 1] = -7
    o, lse = _check((q, k, v, tables, lengths))
    assert (o[1] == 0).all() and (lse[1] == -math.inf).all()


def test_lengths_outside_the_table():
    q, k, v, tables, lengths = make_case(3, 4, 2, 1, 64, 16, [96, 20, 33], dtype=F16, seed=5, device="cuda")
    tables = tables[:, :6]
    for bad, worth in ((2 ** 31 - 1, 96), (-2 ** 31, 0), (-1, 0), (97, 96)):
        lengths[0] = bad
        o, lse = _attend(q, k, v, tables, lengths)
        fixed = lengths.clone()
        fixed[0] = worth
        assert_attention(o, q, k, v, tables, fixed, lse=lse)


def test_layouts():
    """Pools cut from one tensor, head next to row, tables and lengths that
    are views, queries of any order."""
    q, k, v, tables, lengths = make_case(3, 8, 2, 2, 64, 32, [40, 0, 150], dtype=F16, seed=7, device="cuda")
    ref, ref_lse = _attend(q, k, v, tables, lengths, causal=True)
    pages, hkv, page, d = k.shape
    both = torch.full((pages, 2, hkv, page, d), math.nan, dtype=F16, device="cuda")
    both[:, 0], both[:, 1] = k, v
    rows = torch.full((pages, page, 2, hkv, d + 8), math.nan, dtype=F16, device="cuda")
    rows[:, :, 0, :, :d], rows[:, :, 1, :, :d] = k.transpose(1, 2), v.transpose(1, 2)
    wide = torch.full((3, tables.shape[1] + 5), -9, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + tables.shape[1]] = tables
    spaced = torch.zeros(6, dtype=torch.int32, device="cuda")
    spaced[::2] = lengths
    for kp, vp in ((both[:, 0], both[:, 1]),
                   (rows[:, :, 0, :, :d].transpose(1, 2), rows[:, :, 1, :, :d].transpose(1, 2))):
        for qq in (q, q.transpose(1, 2).contiguous().transpose(1, 2), q.transpose(2, 3).contiguous().transpose(2, 3),
                   torch.cat((q, q), 3)[..., 64:]):
            for tt in (tables, wide[:, 2:2 + tables.shape[1]], tables.t().contiguous().t()):
                o, lse = _attend(qq, kp, vp, tt, spaced[::2], causal=True)
                assert torch.equal(o, ref) and torch.equal(lse, ref_lse)


def test_shared_pages():
    """Requests may hold the same pages (a common prompt): reading them is no
    matter of whose they are."""
    q, k, v, tables, lengths = make_case(3, 4, 2, 1, 64, 16, [200, 0, 0], dtype=F16, seed=4, device="cuda")
    tables[1], tables[2] = tables[0], tables[0]
    lengths[1], lengths[2] = 200, 64
    _check((q, k, v, tables, lengths))


def test_pool_beyond_32_bits():
    """Element and byte offsets of the last pages pass 2^31 and 2^32."""
    hkv, page, d = 4, 64, 128
    pages = 2 ** 32 // (hkv * page * d * 2) + 9 + 2 ** 31 // (hkv * page * d)
    q, ks, vs, tables, lengths = make_case(2, 8, hkv, 1, d, page, [130, 300], dtype=F16, seed=4)
    k = torch.empty((pages, hkv, page, d), dtype=F16, device="cuda")
    v = torch.empty_like(k)
    k[-len(ks):], v[-len(ks):] = ks.cuda(), vs.cuda()
    inside = (tables >= 0) & (tables < len(ks))
    far = torch.where(inside, tables + pages - len(ks), tables)
    far = torch.where(~inside & (tables >= 0), -1, far)
    o, lse = _attend(q.cuda(), k, v, far.cuda(), lengths.cuda())
    tables = torch.where(inside, tables, -1)
    assert_attention(o, q, ks, vs, tables, lengths, lse=lse)
    # And the store at the last slots.
    slots = torch.tensor([[pages * page - 1, pages * page, (pages - 3) * page]], device="cuda")
    nk, nv = torch.randn(2, 1, hkv, 3, d, device="cuda").to(F16)
    paged_append(k, v, nk, nv, slots)
    for pool, new in ((k, nk), (v, nv)):
        assert torch.equal(pool[-1, :, -1], new[0, :, 0]) and torch.equal(pool[-3, :, 0], new[0, :, 2])
    del k, v
    torch.cuda.empty_cache()


def test_same_bits_every_time():
    case = make_case(5, 32, 8, 1, 128, 16, [4000, 17, 900, 2500, 1], dtype=BF16, seed=4, device="cuda")
    o, lse = _attend(*case)
    for _ in range(20):
        again = _attend(*case)
        assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    # The rest of the batch does not change what a row sums, only where it is
    # cut: alone, it agrees within the bound.
    alone = tuple(t[:1] if i in (0, 3, 4) else t for i, t in enumerate(case))
    assert_attention(_attend(*alone)[0], *alone)


def test_auto_takes_the_kernels(monkeypatch):
    case = make_case(2, 4, 2, 1, 64, 16, [50, 100], dtype=F16, seed=4, device="cuda")
    import kotflash_amd.paged as paged
    expected = _attend(*case)[0]
    monkeypatch.setattr(paged, "_sdpa_paged", None)
    assert torch.equal(paged_attention(*case), expected)
    assert torch.equal(paged_attention(*case, backend="triton"), expected)


def test_what_the_kernels_do_not_take():
    """auto takes sdpa for these, hip refuses them."""
    for dtype, d, page in ((torch.float32, 64, 16), (F16, 20, 16), (F16, 64, 24), (F16, 136, 16)):
        case = make_case(2, 4, 2, 1, d, page, [30, 50], dtype=dtype, seed=4, device="cuda")
        o, lse = paged_attention(*case, return_lse=True)
        assert_attention(o, *case, lse=lse)
        with pytest.raises((ValueError, TypeError)):
            paged_attention(*case, backend="hip")
    q, k, v, tables, lengths = make_case(2, 4, 2, 1, 64, 16, [30, 50], dtype=F16, seed=4, device="cuda")
    with pytest.raises(ValueError, match="same device"):
        paged_attention(q, k, v, tables.cpu(), lengths)
    with pytest.raises(RuntimeError, match="inference-only"):
        paged_attention(q.requires_grad_(), k, v, tables, lengths)


# --- tables ------------------------------------------------------------------

def _counts(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("seed", range(10))
def test_table_follows_the_definition(seed):
    rng = random.Random(seed)
    batch, page = rng.choice([1, 2, 63, 300, 1023, 1025, 2500]), rng.choice([1, 3, 16, 64, 1000])
    columns = rng.randint(1, 70)
    pages = rng.randint(1, batch * columns + 5)
    table = PageTable(batch, columns * page, num_pages=pages, page_size=page)
    ref = Pages(batch, columns, pages, page)
    for _ in range(8):
        if rng.random() < 0.6:
            width = rng.choice([1, 1, rng.randint(1, 3 * page), rng.randint(1, min(2000, columns * page))])
            if rng.random() < 0.3:
                counts = rng.randint(0, width)
                assert table.reserve(counts, width=width).tolist() == ref.reserve([counts] * batch, width)
            else:
                counts = [rng.choice([-1, width + 1, -2 ** 31, 2 ** 31 - 1]) if rng.random() < 0.02
                          else rng.randint(0, width) for _ in range(batch)]
                assert table.reserve(_counts(counts), width=width).tolist() == ref.reserve(counts, width)
        else:
            keep = [rng.choice([-2 ** 31, 2 ** 31 - 1, rng.randint(0, columns * page)]) for _ in range(batch)]
            table.trim(_counts(keep))
            ref.trim(keep)
        ref.assert_matches(table)
    table.trim(0)
    ref.trim([0] * batch)
    ref.assert_matches(table)
    assert sorted(table.free_pages.tolist()) == list(range(pages))


def test_torch_and_hip_tables_agree():
    tables = [PageTable(40, 500, num_pages=300, page_size=16) for _ in range(2)]
    rng = random.Random(1)
    for _ in range(10):
        counts = _counts([rng.randint(0, 90) for _ in range(40)])
        keep = _counts([rng.randint(0, 400) for _ in range(40)])
        slots = [t.reserve(counts, width=90, backend=b) for t, b in zip(tables, ("hip", "torch"))]
        assert torch.equal(*slots)
        for t, b in zip(tables, ("torch", "hip")):
            t.trim(keep, backend=b)
        for name in ("tables", "lengths", "free_pages", "counters"):
            assert torch.equal(getattr(tables[0], name), getattr(tables[1], name)), name


def test_broken_state_stays_inside():
    """Lengths, tables and counts that no allocator leaves behind: nothing is
    written outside the table, and slots name places of the pool or -1."""
    for height, length, entry in ((10 ** 9, 5, 3), (-4, 10 ** 9, -1), (2, -50, 10 ** 9), (8, 2 ** 31 - 1, -2 ** 31)):
        guard = torch.full((4 + 4, 6 + 2), 77, dtype=torch.int32, device="cuda")
        table = PageTable(4, 96, num_pages=8, page_size=16)
        table.tables = guard[2:6, 1:7]
        table.tables.fill_(entry)
        table.lengths.fill_(length)
        table.free_count.fill_(height)
        for _ in range(2):
            slots = table.reserve(20)
            assert slots.shape == (4, 20)
            table.trim(3)
        inner = torch.zeros_like(guard, dtype=torch.bool)
        inner[2:6, 1:7] = True
        assert (guard[~inner] == 77).all()
        assert 0 <= table.num_free() <= 8


# --- store -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("b,hkv,n,d,page", [(1, 1, 1, 8, 16), (3, 2, 7, 64, 16), (64, 8, 1, 128, 16), (2, 3, 33, 20, 5),
                                            (5, 4, 130, 96, 48), (2, 16, 9, 128, 1)])
@pytest.mark.parametrize("layout", ["bhsd", "bshd", "odd"])
def test_store_is_exact(dtype, b, hkv, n, d, page, layout):
    g = torch.Generator().manual_seed(n)
    pages = -(-b * n // page) + 3
    k = torch.full((pages, hkv, page, d), math.nan, dtype=dtype, device="cuda")
    v = k.clone()
    slots = torch.randperm(pages * page, generator=g)[:b * n].reshape(b, n)
    skip = torch.rand(b, n, generator=g) < 0.2
    slots[skip] = torch.tensor([-1, pages * page, 2 ** 62, -2 ** 62])[torch.arange(int(skip.sum())) % 4]
    new = torch.randn(2, b, hkv, n, d, generator=g).to(dtype).cuda()
    if layout == "bshd":
        nk, nv = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in new)
    elif layout == "odd":
        nk, nv = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in new)
    else:
        nk, nv = new
    paged_append(k, v, nk, nv, slots.cuda(), backend="hip")
    ek = torch.full((pages, hkv, page, d), math.nan, dtype=dtype, device="cuda")
    ev = ek.clone()
    paged_append(ek, ev, *new, slots.cuda(), backend="torch")
    for got, want in ((k, ek), (v, ev)):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_store_layouts_of_pool_and_slots():
    """Pools interleaved in one tensor, offsets that rule out 16-byte rows,
    slots read from a view."""
    both = torch.zeros(4, 16, 2, 2, 68, dtype=F16, device="cuda")
    nk, nv = torch.randn(2, 2, 2, 5, 64, device="cuda").to(F16)
    wide = torch.randperm(64, device="cuda")[:20].reshape(2, 10)
    for lo in (0, 2):
        kp, vp = (both[:, :, i, :, lo:lo + 64].transpose(1, 2) for i in range(2))
        both.zero_()
        paged_append(kp, vp, nk, nv, wide[:, ::2], backend="hip")
        for b in range(2):
            for t in range(5):
                s = int(wide[b, 2 * t])
                assert torch.equal(both[s // 16, s % 16, 0, :, lo:lo + 64], nk[b, :, t])
                assert torch.equal(both[s // 16, s % 16, 1, :, lo:lo + 64], nv[b, :, t])
        assert int((both != 0).sum()) <= 2 * 2 * 5 * 2 * 64
    with pytest.raises(ValueError, match="unit head_dim"):
        t = torch.zeros(4, 2, 64, 16, dtype=F16, device="cuda").transpose(2, 3)
        paged_append(t, t.clone(), nk, nv, wide[:, ::2])


# --- together ----------------------------------------------------------------

def _serve(table, caches, hq, dtype, steps, seed):
    """Prompts, steps, drafts of which some are dropped, requests that leave
    and others that come: checked against each request's own tokens."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    batch = table.batch
    d, hkv = caches[0].k_pages.shape[3], caches[0].k_pages.shape[1]
    own = [[torch.zeros(2, hkv, 0, d, dtype=dtype) for _ in range(batch)] for _ in caches]
    lens = [0] * batch
    for step in range(steps):
        kind = "prompt" if step == 0 else rng.choice(["one", "one", "drafts", "leave"])
        if kind == "leave":
            keep = [0 if rng.random() < 0.3 else n for n in lens]
        elif kind == "one":
            keep = lens
        else:
            keep = [max(0, n - rng.randint(0, 3)) for n in lens]
        if keep != lens:
            table.trim(_counts(keep))
            own = [[x[:, :, :m] for x, m in zip(layer, keep)] for layer in own]
        n = {"prompt": 70, "leave": 50, "one": 1, "drafts": 4}[kind]
        counts = [n if kind in ("one", "drafts") else rng.randint(0, n) * (m == 0) for m in keep]
        slots = table.reserve(_counts(counts), width=n)
        for cache, layer in zip(caches, own):
            q = torch.randn(batch, hq, n, d, generator=g).to(dtype)
            new = torch.randn(2, batch, n, hkv, d, generator=g).to(dtype)
            nk, nv = (x.cuda().transpose(1, 2) for x in new)
            if kind in ("one", "drafts"):
                out = cache.append_and_attend(q.cuda(), nk, nv, slots, causal=kind == "drafts")
            else:
                cache.append(nk, nv, slots)
            for b, c in enumerate(counts):
                layer[b] = torch.cat((layer[b], new[:, b, :c].transpose(1, 2)), 2)
            if kind in ("one", "drafts"):
                most = max(x.shape[2] for x in layer)
                pools = [torch.zeros(batch, hkv, most, d, dtype=dtype) for _ in range(2)]
                for b, x in enumerate(layer):
                    for i in range(2):
                        pools[i][b, :, :x.shape[2]] = x[i]
                ids = torch.arange(batch, dtype=torch.int32)[:, None]
                assert_attention(out, q, *pools, ids, _counts([x.shape[2] for x in layer]).cpu(),
                                 causal=kind == "drafts")
        lens = [a + c for a, c in zip(keep, counts)]
        assert table.lengths.tolist() == lens
        table.check()


@pytest.mark.parametrize("dtype,d,page", [(F16, 64, 16), (BF16, 128, 32), (F16, 80, 48)])
def test_a_server_s_run(dtype, d, page):
    table = PageTable(6, 400, num_pages=150, page_size=page)
    caches = [PagedKVCache(table, 2, d, dtype=dtype) for _ in range(2)]
    for c in caches:
        c.k_pages.fill_(math.nan)
        c.v_pages.fill_(math.nan)
    _serve(table, caches, 8, dtype, 14, page)


def test_captured_steps_grow():
    """One captured step, replayed as the requests grow over page borders,
    with eager work between the replays; each replay against eager calls on
    a copy."""
    batch, hq, hkv, d, page = 3, 8, 2, 64, 16
    both = []
    for _ in range(2):
        table = PageTable(batch, 256, num_pages=40, page_size=page)
        cache = PagedKVCache(table, hkv, d, dtype=F16)
        cache.k_pages.zero_()
        cache.v_pages.zero_()
        g = torch.Generator(device="cuda").manual_seed(3)
        slots = table.reserve(_counts([14, 0, 31]), width=31)
        cache.append(*torch.randn(2, batch, hkv, 31, d, device="cuda", generator=g).to(F16), slots)
        both.append((table, cache))
    (table, cache), (table2, cache2) = both
    q = torch.zeros(batch, hq, 1, d, device="cuda", dtype=F16)
    nk, nv = torch.zeros(2, batch, hkv, 1, d, device="cuda", dtype=F16)
    counts = _counts([1, 1, 1])
    keep = table.lengths.clone()

    def step(table, cache):
        table.trim(keep)
        slots = table.reserve(counts, width=1)
        return cache.append_and_attend(q, nk, nv, slots)

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step(table, cache)  # warm-up; the trim in the step takes it back
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = step(table, cache)
    torch.cuda.synchronize()
    for r in range(6):
        q.copy_(torch.randn(q.shape, device="cuda"))
        nk.copy_(torch.randn(nk.shape, device="cuda"))
        nv.copy_(torch.randn(nv.shape, device="cuda"))
        counts.copy_(_counts([1, r % 2, 1]))
        torch.cuda.synchronize()
        graph.replay()
        expected = step(table2, cache2)
        torch.cuda.synchronize()
        assert torch.equal(out, expected), r
        for name in ("tables", "lengths", "free_pages", "counters"):
            assert torch.equal(getattr(table, name), getattr(table2, name)), (r, name)
        assert torch.equal(cache.k_pages, cache2.k_pages) and torch.equal(cache.v_pages, cache2.v_pages)
        keep.copy_(table.lengths)
        torch.zeros(1 << 20, device="cuda").sum().item()


def test_two_streams_and_a_graph():
    """Calls on two streams, and a graph replayed beside them, share no
    scratch memory."""
    cases = [make_case(4, 16, 4, 1, 128, 16, [3000, 10, 700, 1], dtype=F16, seed=s, device="cuda") for s in (1, 2)]
    want = [_attend(*c) for c in cases]
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(sa):
        _attend(*cases[0])
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=sa):
            captured = _attend(*cases[0])
    torch.cuda.synchronize()
    for r in range(4):
        with torch.cuda.stream(sb):
            graph.replay()
        with torch.cuda.stream(sa):
            eager = [_attend(*cases[1]) for _ in range(3)]
        torch.cuda.synchronize()
        for got, w in [(captured, want[0])] + [(e, want[1]) for e in eager]:
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1]), r


# --- the C ABI ---------------------------------------------------------------

def test_library_refuses_a_small_workspace():
    q, k, v, tables, lengths = make_case(2, 4, 2, 1, 64, 16, [50, 100], dtype=F16, seed=4, device="cuda")
    need = _hip.paged_decode_workspace_bytes(2, 4, 2, 1, 64)
    out = torch.full_like(q, 5.0)
    with pytest.raises(RuntimeError, match="workspace"):
        _hip.paged_decode(q, k, v, out, None, tables, lengths, scale=0.1, causal=False,
                          workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    assert (out == 5).all()
    _hip.paged_decode(q, k, v, out, None, tables, lengths, scale=0.125, causal=False,
                      workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    assert_attention(out, q, k, v, tables, lengths, scale=0.125)


# --- launch paths ------------------------------------------------------------

def test_python_and_native_paths_agree(monkeypatch):
    """Without the native module every call runs the same kernels through the
    Python path; a native call that it does not take changes nothing first."""
    case = make_case(3, 8, 2, 4, 64, 16, [50, 0, 333], dtype=F16, seed=4, device="cuda")
    new = torch.randn(2, 3, 2, 4, 64, device="cuda").to(F16)
    spare = torch.arange(64, 76, device="cuda").reshape(3, 4)

    def run():
        table = PageTable(3, 400, num_pages=40)
        slots = [table.reserve(9), table.reserve(_counts([3, 0, 30]), width=30)]
        table.trim(_counts([4, 10, 25]))
        table.trim(24)
        pools = [t.clone() for t in case[1:3]]
        paged_append(*pools, *new, spare % (case[1].shape[0] * 16))
        cache = PagedKVCache(table, 2, 64, dtype=F16)
        cache.k_pages.zero_()
        cache.v_pages.zero_()
        step = cache.append_and_attend(case[0], *new, table.reserve(4), causal=True)
        return [*slots, table.tables, table.lengths, table.free_pages, table.counters, *pools, step,
                paged_attention(*case, causal=True), *paged_attention(*case, causal=True, return_lse=True),
                paged_attention(*case, scale=0.3)]

    native = run()
    monkeypatch.setattr(_hip, "_NATIVE", _hip._NoNative())
    for i, (a, b) in enumerate(zip(native, run())):
        assert a.dtype == b.dtype and a.shape == b.shape
        assert torch.equal(a.nan_to_num(-7.0) if a.is_floating_point() else a,
                           b.nan_to_num(-7.0) if b.is_floating_point() else b), i


def test_inference_tensors():
    with torch.inference_mode():
        table = PageTable(2, 64, num_pages=8)
        cache = PagedKVCache(table, 2, 64, dtype=F16)
        new = torch.ones(2, 2, 1, 64, device="cuda", dtype=F16)
        q = torch.ones(2, 4, 1, 64, device="cuda", dtype=F16)
        out = cache.append_and_attend(q, new, new, table.reserve(1))
        table.trim(0)
    assert (out == 1).all() and table.num_free() == 8


def test_tables_change_their_version():
    table = PageTable(2, 64, num_pages=8)
    before = [t._version for t in (table.tables, table.lengths, table.counters)]
    table.reserve(1)
    assert all(t._version > v for t, v in zip((table.tables, table.lengths, table.counters), before))


def test_ops_compile_without_graph_breaks():
    import kotflash_amd.ops  # noqa: F401

    ns = torch.ops.kotflash_amd
    q, k, v, tables, lengths = make_case(2, 4, 2, 1, 64, 16, [50, 100], dtype=F16, seed=4, device="cuda", junk=0.0)
    state = [PageTable(2, 256, num_pages=20) for _ in range(2)]
    new = torch.randn(2, 2, 2, 1, 64, device="cuda").to(F16)
    counts = _counts([1, 1])

    def step(q, k, v, nk, nv, tables, lengths, free, counters, counts, keep):
        ns.page_trim_(tables, lengths, free, counters, keep, 16)
        slots = ns.page_reserve_(tables, lengths, free, counters, counts, 16, 1)
        ns.paged_append_(k, v, nk, nv, slots)
        return ns.paged_decode(q, k, v, tables, lengths, False, 0.125)[0] * 2

    results = []
    for fn, t in zip((step, torch.compile(step, backend="aot_eager", fullgraph=True)), state):
        pools = [torch.zeros(20, 2, 16, 64, device="cuda", dtype=F16) for _ in range(2)]
        for r in range(18):
            out = fn(q, *pools, new[0] + r, new[1] - r, t.tables, t.lengths, t.free_pages, t.counters, counts,
                     _counts([100, 100]))
        results.append([out, *pools, t.tables, t.lengths, t.free_pages, t.counters])
    assert results[0][4].tolist() == [18, 18]
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_cache_under_torch_compile():
    table = PageTable(2, 64, num_pages=8)
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    new = torch.ones(2, 2, 1, 64, device="cuda", dtype=F16)
    q = torch.randn(2, 4, 1, 64, device="cuda").to(F16)
    fn = torch.compile(lambda q, n, s: cache.append_and_attend(q, n, n, s), backend="aot_eager")
    for _ in range(3):
        out = fn(q, new, table.reserve(1))
    assert (out == 1).all() and table.lengths.tolist() == [3, 3]


def test_calls_on_a_side_stream():
    """Inputs made on one stream, used on another with an event between."""
    side = torch.cuda.Stream()
    table = PageTable(2, 512, num_pages=64)
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    big = torch.randn(2, 2, 300, 64, device="cuda").to(F16)
    q = torch.randn(2, 4, 1, 64, device="cuda").to(F16)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        slots = table.reserve(_counts([300, 200]), width=300)
        out = cache.append_and_attend(q, big, big, slots)
    torch.cuda.current_stream().wait_stream(side)
    ids = torch.arange(2, dtype=torch.int32)[:, None]
    assert_attention(out, q, big, big, ids, torch.tensor([300, 200], dtype=torch.int32))


def test_every_request_its_own_worker_and_none():
    """Sizes around the number of workers: units one short of it, equal, one
    more, twice, and with a last worker that has one unit."""
    for d, per_request in ((64, 1), (128, 1), (128, 4)):
        for steps in (1023, 1024, 1025, 2047, 2048, 2049, 4100):
            batch = -(-steps // per_request)
            lengths = [32 * per_request] * (batch - 1) + [32 * (steps - per_request * (batch - 1))]
            case = make_case(batch, 2, 1, 1, d, 32, lengths, dtype=F16, seed=steps, device="cuda")
            o = _attend(*case)[0]
            pick = torch.tensor([0, 1, batch // 2, batch - 2, batch - 1])
            few = tuple(t[pick.to(t.device)] if i in (0, 3, 4) else t for i, t in enumerate(case))
            assert_attention(o[pick.cuda()], *few)
            assert torch.isfinite(o).all()


# --- the step that stores and attends in one launch --------------------------

@pytest.mark.parametrize("n", [1, 2, 4, 5, 16])
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 64, 16), (4, 4, 128, 32), (16, 2, 72, 48), (32, 1, 96, 16), (80, 1, 40, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_fused_step_matches_two_launches(n, hq, hkv, d, page, dtype):
    """Requests whose new tokens end or begin a page or a step, cross them, or
    are their first; with fewer new tokens than slots, and none."""
    before = [0, 0, 1, 15, 16, 31, 32, 33, page - 1, page, 2 * page - 2, 200, 1000, 64 - n, 7]
    counts = [n, 0, n, n, 1, n, n, n, n, n, n, max(1, n - 1), n, n, n // 2]
    g = torch.Generator(device="cuda").manual_seed(n + d)
    results = []
    b = len(before)
    q = torch.randn(b, hq, n, d, device="cuda", generator=g).to(dtype)
    new = torch.randn(2, b, n, hkv, d, device="cuda", generator=g).to(dtype).transpose(2, 3)
    old = torch.randn(2, b, hkv, max(before), d, device="cuda", generator=g).to(dtype)
    for how in ("fused", "hip", "auto"):
        table = PageTable(b, 1100, num_pages=400, page_size=page)
        cache = PagedKVCache(table, hkv, d, dtype=dtype)
        cache.k_pages.fill_(math.nan)
        cache.v_pages.fill_(math.nan)
        cache.append(*old, table.reserve(_counts(before), width=max(before)))
        slots = table.reserve(_counts(counts), width=n)
        out = cache.append_and_attend(q, *new, slots, causal=True, append_backend=how)
        results.append((out, cache.k_pages, cache.v_pages))
    for other in results[1:]:
        for a, b_ in zip(results[0], other):
            assert torch.equal(a.view(torch.int16), b_.view(torch.int16))
    lens = [x + c for x, c in zip(before, counts)]
    whole = [torch.cat((old[i], torch.zeros_like(new[i])), 2) for i in range(2)]
    for i in range(2):
        for r, (x, c) in enumerate(zip(before, counts)):
            whole[i][r, :, x:x + c] = new[i][r, :, :c]
    ids = torch.arange(b, dtype=torch.int32)[:, None]
    pick = [0, 1, 2, 5, 8, 11, 13, 14]
    assert_attention(results[0][0][pick], q[pick], *whole, ids[pick], torch.tensor(lens, dtype=torch.int32)[pick],
                     causal=True)


def test_fused_step_leaves_other_slots():
    """Slots outside the pool, and holes between named ones, store nothing."""
    table = PageTable(2, 64, num_pages=8)
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    cache.k_pages.zero_()
    cache.v_pages.zero_()
    slots = table.reserve(_counts([3, 0]), width=5)
    holes = torch.full_like(slots, -1)
    holes[0, 0], holes[0, 2], holes[0, 4] = slots[0, 0], slots[0, 1], slots[0, 2]
    holes[0, 1], holes[0, 3], holes[1, 0] = 8 * 16, 2 ** 40, -2 ** 62
    new = torch.randn(2, 2, 2, 5, 64, device="cuda").to(F16)
    q = torch.randn(2, 4, 1, 64, device="cuda").to(F16)
    out = cache.append_and_attend(q, *new, holes, append_backend="fused")
    page = int(table.tables[0, 0])
    for pool, x in ((cache.k_pages, new[0]), (cache.v_pages, new[1])):
        assert torch.equal(pool[page, :, :3], x[0][:, [0, 2, 4]])
        assert int((pool != 0).sum()) <= 2 * 3 * 64
    assert (out[1] == 0).all()
    assert_attention(out[:1], q[:1], new[0][:1][:, :, [0, 2, 4]].contiguous(), new[1][:1][:, :, [0, 2, 4]].contiguous(),
                     torch.zeros(1, 1, dtype=torch.int32), torch.tensor([3], dtype=torch.int32))


def test_fused_step_refusals():
    table = PageTable(2, 64, num_pages=8)
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    cache.k_pages.zero_()
    slots = table.reserve(17)
    new = torch.ones(2, 2, 17, 64, device="cuda", dtype=F16)
    q = torch.ones(2, 4, 1, 64, device="cuda", dtype=F16)
    with pytest.raises(ValueError, match="up to 16 new tokens"):
        cache.append_and_attend(q, new, new, slots, append_backend="fused")
    with pytest.raises(ValueError, match="HIP attention"):
        cache.append_and_attend(q, new[:, :, :1], new[:, :, :1], slots[:, :1], append_backend="fused",
                                attention_backend="sdpa")
    with pytest.raises(ValueError, match="slots"):
        cache.append_and_attend(q, new[:1, :, :1], new[:1, :, :1], slots[:, :1])
    assert (cache.k_pages == 0).all()
    assert (cache.append_and_attend(q, new, new, slots) == 1).all()


def test_fused_step_python_path(monkeypatch):
    monkeypatch.setattr(_hip, "_NATIVE", _hip._NoNative())
    table = PageTable(2, 64, num_pages=8)
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    new = torch.randn(2, 2, 2, 3, 64, device="cuda").to(F16)
    q = torch.randn(2, 4, 3, 64, device="cuda").to(F16)
    calls = []
    real = _hip.paged_append_decode
    monkeypatch.setattr(_hip, "paged_append_decode", lambda *a, **k: (calls.append(1), real(*a, **k)))
    out = cache.append_and_attend(q, *new.transpose(3, 4).contiguous().transpose(3, 4), table.reserve(3), causal=True)
    assert calls == [1]
    ids = torch.arange(2, dtype=torch.int32)[:, None]
    assert_attention(out, q, *new, ids, torch.tensor([3, 3], dtype=torch.int32), causal=True)


@pytest.mark.parametrize("dtype,d,hq,hkv", [(F16, 64, 8, 2), (BF16, 128, 4, 1), (BF16, 96, 24, 1), (F16, 32, 48, 1),
                                            (F16, 128, 16, 1)])
@pytest.mark.parametrize("length", [4, 33, 37, 66, 259])
def test_what_a_row_does_not_see_yet(dtype, d, hq, hkv, length):
    """K and V of later draft tokens that are NaN or infinite do not reach the
    rows in front of them; they do reach those that see them."""
    sq = 4
    for seed, value in enumerate((math.nan, math.inf, -math.inf)):
        q, k, v, tables, lengths = make_case(3, hq, hkv, sq, d, 16, [length, 500, length], dtype=dtype, seed=seed,
                                             device="cuda")
        clean = _attend(q, k, v, tables, lengths, causal=True)
        at = length - 2  # seen by the last two rows only
        page, row = int(tables[0, at // 16]), at % 16
        bad_k, bad_v = k.clone(), v.clone()
        bad_v[page, :, row, 3] = value
        o, lse = _attend(q, k, bad_v, tables, lengths, causal=True)
        assert torch.equal(lse, clean[1])
        tol = 2 * torch.finfo(dtype).eps * clean[0].abs() + 2.0 ** -20  # rows summed apart: the order differs
        assert bool(((o - clean[0]).abs() <= tol)[:, :, :2].all()) and torch.equal(o[1:], clean[0][1:])
        assert not torch.isfinite(o[0, :, 2:, 3]).any()
        rest = [i for i in range(d) if i != 3]
        assert bool(((o - clean[0]).abs() <= tol)[0][..., rest].all())
        bad_k[page, :, row, 3] = value
        o, lse = _attend(q, bad_k, v, tables, lengths, causal=True)
        assert torch.equal(o[:, :, :2], clean[0][:, :, :2]) and torch.equal(lse[:, :, :2], clean[1][:, :, :2])
        if math.isnan(value):
            assert torch.isnan(o[0, :, 2:]).all()


def test_gradients_are_refused():
    q, k, v, tables, lengths = make_case(2, 4, 2, 1, 64, 16, [30, 50], dtype=F16, seed=4, device="cuda", junk=0.0)
    table = PageTable(2, 64, num_pages=k.shape[0])
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    cache.k_pages.zero_()
    slots = table.reserve(1)
    new = torch.ones(2, 2, 1, 64, device="cuda", dtype=F16, requires_grad=True)
    for call in (lambda: cache.append(new, new, slots), lambda: cache.append_and_attend(q, new, new, slots)):
        with pytest.raises(RuntimeError, match="inference-only"):
            call()
        assert (cache.k_pages == 0).all()
    with torch.no_grad():
        cache.append_and_attend(q, new, new, slots)
    assert (cache.k_pages != 0).any()


@pytest.mark.parametrize("batch,hq,hkv,d,longest", [(40, 16, 1, 64, 20000), (40, 16, 1, 128, 9000), (1, 16, 1, 64, 40000),
                                                    (2, 8, 8, 96, 9000), (300, 16, 1, 128, 700)])
def test_rows_with_many_partials(batch, hq, hkv, d, longest):
    """One long request among short ones: few and many rows, few and many
    partials of a row."""
    lengths = [longest] + [(7 * i) % 90 for i in range(1, batch)]
    _check(make_case(batch, hq, hkv, 1, d, 16, lengths, dtype=F16, seed=d, device="cuda"))


def test_tables_of_inference_mode_take_the_native_path(monkeypatch):
    """A server that makes its cache under inference_mode gets the same launches."""
    import kotflash_amd.kernels.hip_paged as hip_paged

    def refuse(*args, **kw):
        raise AssertionError("the Python path ran")

    for name in ("reserve_pages", "trim_pages", "attention_paged", "append_attention_paged"):
        monkeypatch.setattr(hip_paged, name, refuse)
    with torch.inference_mode():
        table = PageTable(2, 64, num_pages=8)
        cache = PagedKVCache(table, 2, 64, dtype=F16)
        new = torch.randn(2, 2, 2, 1, 64, device="cuda").to(F16)
        q = torch.randn(2, 4, 1, 64, device="cuda").to(F16)
        out = cache.append_and_attend(q, *new, table.reserve(1))
        assert table.lengths.tolist() == [1, 1]
        table.trim(0)
    assert torch.equal(out, new[1].repeat_interleave(2, 1))
    assert table.num_free() == 8 and table.lengths.tolist() == [0, 0]


def test_a_whole_step_under_torch_compile():
    """Tables, store and attention compiled together, over page borders,
    against the same calls without."""
    results = []
    for compiled in (False, True):
        torch.manual_seed(5)
        table = PageTable(2, 128, num_pages=16)
        cache = PagedKVCache(table, 2, 64, dtype=F16)
        cache.k_pages.zero_()
        cache.v_pages.zero_()
        most = _counts([20, 100])

        def step(q, n):
            table.trim(most)
            slots = table.reserve(1)
            return cache.append_and_attend(q, n, n, slots, append_backend="hip")

        fn = torch.compile(step, backend="aot_eager") if compiled else step
        outs = []
        for _ in range(36):
            n = torch.randn(2, 2, 1, 64, device="cuda").to(F16)
            q = torch.randn(2, 4, 1, 64, device="cuda").to(F16)
            outs.append(fn(q, n))
        results.append([torch.stack(outs), table.tables, table.lengths, table.free_pages, table.counters,
                        cache.k_pages, cache.v_pages])
    assert results[0][2].tolist() == [21, 36]
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("how", ["fused", "hip"])
def test_drafts_of_their_own_number(how):
    """Requests with fewer drafts than rows: theirs are the last rows of q, in
    whatever columns their new rows and slots stand."""
    n, counts, before = 4, [4, 1, 3, 0, 2], [30, 0, 15, 20, 64]
    b = len(counts)
    g = torch.Generator(device="cuda").manual_seed(9)
    table = PageTable(b, 128, num_pages=40)
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    cache.k_pages.fill_(math.nan)
    cache.v_pages.fill_(math.nan)
    old = torch.randn(2, b, 2, max(before), 64, device="cuda", generator=g).to(F16)
    cache.append(*old, table.reserve(_counts(before), width=max(before)))
    slots = table.reserve(_counts(counts), width=n)
    new = torch.randn(2, b, 2, n, 64, device="cuda", generator=g).to(F16)
    q = torch.randn(b, 8, n, 64, device="cuda", generator=g).to(F16)
    # Right-aligned, as the rows of q are.
    last = torch.stack([s.roll(n - c) for s, c in zip(slots, counts)])
    out = cache.append_and_attend(q, *new, last, causal=True, append_backend=how)
    own = [torch.cat((old[i], torch.zeros_like(new[i])), 2) for i in range(2)]
    for i in range(2):
        for r, (x, c) in enumerate(zip(before, counts)):
            own[i][r, :, x:x + c] = new[i][r, :, n - c:]
    ids = torch.arange(b, dtype=torch.int32)[:, None]
    assert_attention(out, q, *own, ids, torch.tensor([x + c for x, c in zip(before, counts)], dtype=torch.int32),
                     causal=True)
    # The token of the request with one draft sees itself alone, in the last row.
    assert torch.equal(out[1, :, -1], new[1][1, :, -1].repeat_interleave(4, 0))
    assert (out[1, :, :-1] == 0).all()


def _step_state(dtype=F16, batch=4, hkv=2, d=64, page=16):
    """A cache whose requests hold 900, 40, 0 and 333 tokens (and so on), and
    the tokens that they get next."""
    g = torch.Generator(device="cuda").manual_seed(3)
    table = PageTable(batch, 1200, num_pages=80 * batch, page_size=page)
    cache = PagedKVCache(table, hkv, d, dtype=dtype)
    cache.k_pages.fill_(math.nan)
    cache.v_pages.fill_(math.nan)
    held = [(900, 40, 0, 333)[b % 4] for b in range(batch)]
    old = torch.randn(2, batch, hkv, 900, d, device="cuda", generator=g).to(dtype)
    cache.append(*old, table.reserve(_counts(held), width=900))
    return table, cache, g


def _steps_agree(prepare, n, *, how="fused", hq=8, **kw):
    """A step that stores and attends in one launch, against two launches: the
    output and both pools to the bit. ``prepare(table, cache)`` gives slots."""
    got = []
    for backend in (how, "hip"):
        table, cache, g = _step_state(**kw)
        slots = prepare(table, cache)
        b, hkv, d = table.batch, cache.k_pages.shape[1], cache.k_pages.shape[3]
        new = torch.randn(2, b, hkv, n, d, device="cuda", generator=g).to(cache.k_pages.dtype)
        q = torch.randn(b, hq, 1, d, device="cuda", generator=g).to(cache.k_pages.dtype)
        out = cache.append_and_attend(q, *new, slots, append_backend=backend)
        got.append((out, cache.k_pages, cache.v_pages))
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    return got[0]


@pytest.mark.parametrize("how", ["fused", "auto"])
@pytest.mark.parametrize("kw", [dict(), dict(dtype=BF16, d=128, page=32), dict(hq=64, hkv=1, d=96, page=48),
                                dict(hq=80, hkv=1, d=40), dict(hq=20, hkv=1, d=128)])
def test_a_step_with_a_part_of_the_slots(how, kw):
    """The first of more slots than the step brings tokens: the new rows are
    not the requests' last ones, and units in front of the last read them."""
    def some(first):
        def prepare(table, cache):
            slots = table.reserve(80)
            cache.append(*torch.ones(2, table.batch, cache.k_pages.shape[1], 80, cache.k_pages.shape[3], device="cuda",
                                     dtype=cache.k_pages.dtype), slots)
            return slots[:, first:first + 4]
        return prepare

    for first in (0, 5, 40, 76):
        _steps_agree(some(first), 4, how=how, **kw)


@pytest.mark.parametrize("how", ["fused", "auto"])
def test_a_step_over_pages_of_several_requests(how):
    """Requests that hold the same pages all see what one of them stores."""
    def prepare(table, cache):
        slots = table.reserve(2)
        table.tables[1:] = table.tables[0]
        table.lengths[1:] = table.lengths[0] - torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32)
        slots[1:] = -1
        return slots

    out, k, v = _steps_agree(prepare, 2, how=how)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("how", ["fused", "auto"])
def test_a_step_whose_rows_nobody_sees(how):
    """New rows behind the lengths, in pages of no request, and of requests
    that hold nothing are stored."""
    def shorter(table, cache):
        slots = table.reserve(3)
        table.lengths.copy_(_counts([880, 0, 0, 334]))
        return slots

    def elsewhere(table, cache):
        slots = table.reserve(3)
        spare = int(table.free_pages[0])
        slots[1] = spare * 16 + torch.tensor([15, 0, 7], device="cuda")
        slots[2] = -1
        return slots

    def nothing(table, cache):
        slots = table.reserve(3)
        table.lengths.zero_()
        return slots

    for prepare in (shorter, elsewhere, nothing):
        _, k, v = _steps_agree(prepare, 3, how=how)
    assert int(torch.isfinite(k).all(-1).sum()) == 2 * (900 + 40 + 0 + 333 + 4 * 3)


def test_a_step_of_many_rows():
    """Up to 256 new rows are stored by the attention, more in front of it."""
    for batch, n in ((64, 4), (256, 1), (65, 1), (16, 16)):
        _steps_agree(lambda table, cache: table.reserve(n), n, batch=batch)
    table, cache, g = _step_state(batch=86)
    slots = table.reserve(3)
    new = torch.randn(2, 86, 2, 3, 64, device="cuda").to(F16)
    q = torch.randn(86, 4, 1, 64, device="cuda").to(F16)
    with pytest.raises(ValueError, match="256 in all"):
        cache.append_and_attend(q, *new, slots, append_backend="fused")
    assert torch.isnan(cache.k_pages[slots // 16, :, slots % 16]).all()
    _steps_agree(lambda table, cache: table.reserve(3), 3, batch=86, how="auto")


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("lengths", [[100, 100, 100], [30000, 500, 30000]])
@pytest.mark.parametrize("sq", [1, 8])
def test_lse_of_rows_that_see_a_nan(dtype, d, lengths, sq):
    """A NaN score, or one of +infinity, leaves a row with an LSE that is not
    finite and not that of an empty row, whether one worker wrote the row or
    several; the rows of others, and those where the score is -infinity, keep
    theirs."""
    q, k, v, tables, lens = make_case(3, 16, 2, sq, d, 16, lengths, dtype=dtype, seed=6, device="cuda")
    clean, clean_lse = _attend(q, k, v, tables, lens)
    for at in (0, lengths[0] // 2, lengths[0] - 1):
        for value in (math.nan, math.inf):
            bad = k.clone()
            bad[tables[0, at // 16], 0, at % 16, 3] = value
            o, lse = _attend(q, bad, v, tables, lens)
            hit = torch.zeros_like(lse, dtype=torch.bool)
            hit[0, :8] = True if math.isnan(value) else q[0, :8, :, 3] > 0
            assert torch.isnan(o[hit]).all()
            assert (torch.isnan(lse[hit]) | (lse[hit] == math.inf)).all()
            assert torch.isfinite(o[~hit]).all() and torch.isfinite(lse[~hit]).all()
            hit[0, :8] = True
            assert torch.equal(o[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
            want = paged_attention(q[:1], bad, v, tables[:1], lens[:1], return_lse=True, backend="sdpa")
            assert torch.equal(torch.isfinite(want[1]), torch.isfinite(lse[:1]))


def test_reserve_refuses_a_width_beyond_64_bits():
    table = PageTable(2, 64, num_pages=8)
    for width in (2 ** 64, 2 ** 63, 2 ** 40, 2 ** 30, -2 ** 64):
        with pytest.raises(ValueError, match="width"):
            table.reserve(1, width=width)
    assert table.lengths.tolist() == [0, 0] and table.num_free() == 8


def test_slots_of_a_broken_state_name_places_of_the_pool():
    """Page numbers outside the pool, in tables and on the stack, give -1."""
    for width, counts in ((20, 20), (1, 1), (1500, 40)):
        for entry in (-1, 7, 8, 9, 2 ** 31 - 1, -2 ** 31):
            table = PageTable(4, 1600, num_pages=8, page_size=16)
            table.tables.fill_(entry)
            table.free_pages[::2] = entry
            table.lengths.copy_(_counts([5, 16, 0, 31]))
            slots = table.reserve(counts, width=width)
            assert ((slots >= -1) & (slots < 8 * 16)).all(), (width, entry)
            assert (slots[0, 0] == 7 * 16 + 5) if entry == 7 else (slots[0, 0] == -1)


def test_torch_and_hip_tables_agree_on_broken_states():
    for height, length, entry in ((10 ** 9, 5, 3), (-4, 10 ** 9, -1), (2, -50, 10 ** 9), (8, 2 ** 31 - 1, -2 ** 31)):
        tables = [PageTable(4, 96, num_pages=8, page_size=16) for _ in range(2)]
        for t in tables:
            t.tables.fill_(entry)
            t.lengths.copy_(_counts([length, 7, 96, length]))
            t.free_count.fill_(height)
        for _ in range(3):
            slots = [t.reserve(20, backend=b) for t, b in zip(tables, ("hip", "torch"))]
            assert torch.equal(*slots)
            for name in ("tables", "lengths", "free_pages", "counters"):
                assert torch.equal(getattr(tables[0], name), getattr(tables[1], name)), name
            for t, b in zip(tables, ("hip", "torch")):
                t.trim(3, backend=b)
            for name in ("tables", "lengths", "free_pages", "counters"):
                assert torch.equal(getattr(tables[0], name), getattr(tables[1], name)), name


def test_forward_mode_gradients_are_refused():
    import torch.autograd.forward_ad as fwd

    q, k, v, tables, lengths = make_case(2, 4, 2, 1, 64, 16, [30, 50], dtype=F16, seed=4, device="cuda", junk=0.0)
    table = PageTable(2, 64, num_pages=k.shape[0])
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    cache.k_pages.zero_()
    slots = table.reserve(1)
    new = torch.ones(2, 2, 1, 64, device="cuda", dtype=F16)
    with fwd.dual_level():
        dual = [fwd.make_dual(t, torch.ones_like(t)) for t in (q, k, new)]
        for call in (lambda: paged_attention(dual[0], k, v, tables, lengths),
                     lambda: paged_attention(q, dual[1], v, tables, lengths, backend="sdpa"),
                     lambda: cache.append(dual[2], new, slots),
                     lambda: cache.append(dual[2], new, slots, backend="torch"),
                     lambda: cache.append_and_attend(q, new, dual[2], slots),
                     lambda: cache.append_and_attend(dual[0], new, new, slots, append_backend="hip")):
            with pytest.raises(RuntimeError, match="inference-only"):
                call()
        assert (cache.k_pages == 0).all()
    cache.append_and_attend(q, new, new, slots)


@pytest.mark.parametrize("native", [True, False])
def test_what_is_written_changes_its_version(native, monkeypatch):
    """Autograd sees stores and table calls as it sees in-place operations."""
    if not native:
        monkeypatch.setattr(_hip, "_NATIVE", _hip._NoNative())
    table = PageTable(2, 64, num_pages=8)
    cache = PagedKVCache(table, 2, 64, dtype=F16)
    cache.k_pages.zero_()
    new = torch.ones(2, 2, 1, 64, device="cuda", dtype=F16)
    q = torch.ones(2, 4, 1, 64, device="cuda", dtype=F16)
    x = torch.ones(64, device="cuda", dtype=F16, requires_grad=True)
    slots = table.reserve(1)

    def moves(tensors, call):
        before = [t._version for t in tensors]
        call()
        return all(t._version > v for t, v in zip(tensors, before))

    pools, state = (cache.k_pages, cache.v_pages), (table.tables, table.lengths, table.counters)
    assert moves(pools, lambda: cache.append(new, new, slots))
    for how in ("fused", "hip", "torch"):
        assert moves(pools, lambda: cache.append_and_attend(q, new, new, slots, append_backend=how))
    assert moves(state, lambda: table.reserve(1)) and moves(state + (table.free_pages,), lambda: table.trim(0))
    product = (cache.k_pages[0, 0, 0] * x).sum()
    cache.append(new, new, slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


@pytest.mark.parametrize("native", [True, False])
def test_sizes_beyond_the_kernels(native, monkeypatch):
    """Tables whose steps pass 32-bit numbers: auto takes sdpa, hip refuses, a
    step before it stores anything."""
    if not native:
        monkeypatch.setattr(_hip, "_NATIVE", _hip._NoNative())
    b, hkv, page, d = 16, 8, 2 ** 20, 8
    k = torch.zeros(2, hkv, page, d, dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(3)
    few = torch.randn(2, hkv, 40, d, generator=g).to(F16)
    k[1, :, :40], v[1, :, :40] = few[0].cuda(), few[1].cuda()
    tables = torch.full((b, 512), -1, dtype=torch.int32, device="cuda")
    tables[:, 0] = 1
    lengths = (torch.arange(b, dtype=torch.int32) * 2 + 1).cuda()
    q = torch.randn(b, hkv, 1, d, generator=g).to(F16).cuda()
    o, lse = paged_attention(q, k, v, tables, lengths, return_lse=True)
    small = torch.zeros(b, 1, dtype=torch.int32)
    assert_attention(o, q, few[0][None], few[1][None], small, lengths, lse=lse)
    with pytest.raises(RuntimeError, match="32-bit step numbers"):
        paged_attention(q, k, v, tables, lengths, backend="hip")
    table = PageTable(b, 64, num_pages=2)
    cache = PagedKVCache(table, hkv, d, dtype=F16)
    cache.k_pages, cache.v_pages = k, v
    table.tables, table.lengths = tables, lengths
    new = torch.ones(b, hkv, 1, d, dtype=F16, device="cuda")
    slots = torch.arange(b, device="cuda")[:, None] + 50
    for how in ("hip", "auto", "fused"):
        with pytest.raises(RuntimeError, match="32-bit step numbers"):
            cache.append_and_attend(q, new, new, slots, append_backend=how, attention_backend="hip")
    assert (k[0, :, :100] == 0).all()
    with pytest.raises(ValueError, match="fused"):
        cache.append_and_attend(q, new, new, slots, append_backend="fused")
    assert (k[0, :, :100] == 0).all()
    out = cache.append_and_attend(q, new, new, slots)
    assert torch.equal(out, o) and (k[0, :, 50:50 + b] == 1).all() and int((k[0] != 0).sum()) == b * hkv * d
    del k, v, cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("how", ["auto", "fused", "hip"])
@pytest.mark.parametrize("offset", [0, 4])
def test_a_compiled_step_is_one_graph_of_the_ops(how, offset):
    """Compiled with fullgraph, random keys and values, causal drafts over page
    borders, pools off a 16-byte border too: each step against eager calls."""
    from torch._dynamo.backends.registry import lookup_backend

    seen = []

    def backend(gm, inputs):
        seen.append([str(n.target).split(".")[1] for n in gm.graph.nodes if "kotflash_amd" in str(n.target)])
        return lookup_backend("aot_eager")(gm, inputs)

    results = []
    for compiled in (False, True):
        torch.manual_seed(5)
        table = PageTable(2, 128, num_pages=16)
        cache = PagedKVCache(table, 2, 64, dtype=F16)
        if compiled and offset:
            n = cache.k_pages.numel()
            cache.k_pages, cache.v_pages = (torch.empty(n + 8, device="cuda", dtype=F16)[offset:offset + n].view(16, 2, 16, 64)
                                            for _ in range(2))
        cache.k_pages.zero_()
        cache.v_pages.zero_()
        most = _counts([21, 100])

        def step(q, k, v):
            table.trim(most)
            return cache.append_and_attend(q, k, v, table.reserve(3), causal=True, append_backend=how)

        torch._dynamo.reset()
        fn = torch.compile(step, backend=backend, fullgraph=True) if compiled else step
        outs = []
        for _ in range(20):
            k, v = torch.randn(2, 2, 2, 3, 64, device="cuda").to(F16)
            outs.append(fn(torch.randn(2, 4, 3, 64, device="cuda").to(F16), k, v))
        results.append([torch.stack(outs), table.tables, table.lengths, table.free_pages, table.counters,
                        cache.k_pages, cache.v_pages])
    assert seen == [["page_trim_", "page_reserve_", "paged_append_", "paged_decode"]]
    assert results[0][2].tolist() == [24, 60]
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_library_trims_to_lengths_beyond_32_bits():
    table = PageTable(2, 64, num_pages=8)
    table.reserve(40)
    state = (table.tables, table.lengths, table.free_pages, table.counters)
    before = [t.clone() for t in state]
    for length in (2 ** 30, 2 ** 31, 2 ** 32 + 3, 2 ** 62):
        _hip.page_trim(*state, length, page_size=16)
        for t, b in zip(state, before):
            assert torch.equal(t, b), length
    _hip.page_trim(*state, 20, page_size=16)
    assert table.lengths.tolist() == [20, 20] and table.num_free() == 4
