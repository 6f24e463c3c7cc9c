"""The paged cache on the CPU: allocator, stores and attention against their
definition, and every refusal."""
import math
import random

import pytest
import torch

from kotflash_amd.paged import PagedKVCache, PageTable, paged_append, paged_attention
from tests.paged_oracle import Pages, assert_attention, attention64, make_case

F32 = torch.float32


def _table(batch=3, max_len=64, num_pages=8, page=16):
    return PageTable(batch, max_len, num_pages=num_pages, page_size=page, device="cpu")


@pytest.mark.parametrize("seed", range(12))
def test_table_follows_the_definition(seed):
    rng = random.Random(seed)
    batch, page = rng.choice([1, 2, 7, 30]), rng.choice([1, 3, 16, 64])
    columns, pages = rng.randint(1, 9), rng.randint(1, 90)
    table = _table(batch, columns * page, pages, page)
    ref = Pages(batch, columns, pages, page)
    for _ in range(25):
        if rng.random() < 0.6:
            width = rng.randint(1, 3 * page)
            if rng.random() < 0.3:
                counts = rng.randint(0, width)
                assert table.reserve(counts, width=width).tolist() == ref.reserve([counts] * batch, width)
            else:
                counts = [rng.randint(-1, width + 1) if rng.random() < 0.2 else rng.randint(0, width)
                          for _ in range(batch)]
                got = table.reserve(torch.tensor(counts, dtype=torch.int32), width=width)
                assert got.tolist() == ref.reserve(counts, width)
        else:
            keep = [rng.randint(-2, columns * page + 2) for _ in range(batch)]
            table.trim(torch.tensor(keep, dtype=torch.int32))
            ref.trim(keep)
        ref.assert_matches(table)
    table.trim(0)
    ref.trim([0] * batch)
    ref.assert_matches(table)
    assert sorted(table.free_pages.tolist()) == list(range(pages))


def test_trim_undoes_reserve():
    table = _table(4, 200, 40)
    table.reserve(torch.tensor([30, 0, 17, 100], dtype=torch.int32), width=100)
    before = [t.clone() for t in (table.tables, table.lengths, table.free_pages, table.counters)]
    kept = table.lengths.clone()
    table.reserve(torch.tensor([5, 40, 16, 1], dtype=torch.int32), width=40)
    table.trim(kept)
    for x, y in zip(before, (table.tables, table.lengths, table.free_pages, table.counters)):
        assert torch.equal(x, y)


def test_requests_behind_a_refused_one():
    """Once one does not fit, none that needs a page is served; those that
    need none are."""
    table = _table(4, 64, 3)
    table.reserve(torch.tensor([8, 0, 0, 8], dtype=torch.int32), width=8)  # 2 of 3 pages
    slots = table.reserve(torch.tensor([8, 17, 1, 8], dtype=torch.int32), width=17)
    assert table.lengths.tolist() == [16, 0, 0, 16]
    assert int(table.refused) == 2 and table.num_free() == 1
    assert (slots[1:3] == -1).all() and (slots[0, :8] >= 0).all() and (slots[0, 8:] == -1).all()
    with pytest.raises(RuntimeError, match="2 requests found no room"):
        table.check()
    table.reserve(torch.tensor([0, 0, 1, 0], dtype=torch.int32), width=1)
    table.check()
    assert table.num_free() == 0


@pytest.mark.parametrize("page,hq,hkv,sq,causal", [(16, 4, 2, 1, False), (5, 3, 3, 2, True),
                                                   (16, 4, 1, 20, True), (32, 2, 2, 3, False)])
def test_attention_follows_the_definition(page, hq, hkv, sq, causal):
    lengths = [0, 1, 7, 16, 33, 64]
    args = make_case(6, hq, hkv, sq, 24, page, lengths, dtype=F32, seed=page + sq)
    o, lse = paged_attention(*args, causal=causal, return_lse=True)
    # fp32 throughout: torch's own sums, within the 64-bit bound of that type.
    assert_attention(o, *args, causal=causal, lse=lse)
    assert torch.equal(o, paged_attention(*args, causal=causal))
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all()


def test_pages_outside_the_pool_are_not_seen():
    q, k, v, tables, lengths = make_case(3, 2, 1, 1, 16, 16, [40, 16, 33], dtype=F32, seed=4)
    tables[0, 1] = k.shape[0]
    tables[1, 0] = -1
    tables[2, 2] = -2 ** 31
    o, lse = paged_attention(q, k, v, tables, lengths, return_lse=True)
    assert_attention(o, q, k, v, tables, lengths, lse=lse)
    assert (o[1] == 0).all() and (lse[1] == -math.inf).all()
    # Request 2 lost only its last position's page.
    assert_attention(o[2:], q[2:], k, v, tables[2:], torch.tensor([32], dtype=torch.int32))


def test_lengths_beyond_the_table():
    q, k, v, tables, lengths = make_case(2, 2, 1, 1, 16, 16, [32, 20], dtype=F32, seed=5)
    tables = tables[:, :2].contiguous()
    for bad in (10 ** 9, 2 ** 31 - 1):
        lengths[0] = bad
        assert_attention(paged_attention(q, k, v, tables, lengths), q, k, v, tables,
                         torch.tensor([32, 20], dtype=torch.int32))
    lengths[0] = -5
    assert (paged_attention(q, k, v, tables, lengths)[0] == 0).all()


def test_a_run_of_steps_matches_contiguous_attention():
    """Prompts, steps and drafts through table and cache, as a server runs
    them, against attention over each request's own tokens."""
    g = torch.Generator().manual_seed(9)
    hq, hkv, d, page = 4, 2, 16, 16
    table = _table(3, 128, 12, page)
    cache = PagedKVCache(table, hkv, d, dtype=F32)
    kept = [torch.zeros(2, hkv, 0, d) for _ in range(3)]

    def add(counts, n, causal):
        slots = table.reserve(torch.tensor(counts, dtype=torch.int32), width=n)
        q = torch.randn(3, hq, n, d, generator=g)
        nk, nv = (torch.randn(3, n, hkv, d, generator=g).transpose(1, 2) for _ in range(2))
        out = cache.append_and_attend(q, nk, nv, slots, causal=causal)
        for b, c in enumerate(counts):
            kept[b] = torch.cat((kept[b], torch.stack((nk[b, :, :c], nv[b, :, :c]))), 2)
        return q, out

    add([20, 3, 0], 20, False)
    for _ in range(20):
        q, out = add([1, 1, 1], 1, False)
    table.trim(torch.tensor([30, 100, 21], dtype=torch.int32))
    kept[0] = kept[0][:, :, :30]
    q, out = add([4, 4, 4], 4, True)
    for b in range(3):
        n = kept[b].shape[2]
        assert table.lengths[b] == n
        for r in range(4):
            m = n - 3 + r
            k, v = (kept[b][i, :, :m].repeat_interleave(hq // hkv, 0) for i in range(2))
            ref = torch.nn.functional.scaled_dot_product_attention(q[b, :, r:r + 1], k, v)
            torch.testing.assert_close(out[b, :, r:r + 1], ref, atol=1e-5, rtol=1e-5)
    table.check()


def test_append_skips_slots_outside_the_pool():
    k = torch.zeros(2, 1, 4, 8)
    v = torch.zeros(2, 1, 4, 8)
    new = torch.arange(1, 6, dtype=F32)[None, None, :, None].expand(1, 1, 5, 8)
    paged_append(k, v, new, -new, torch.tensor([[-1, 7, 8, 0, 2 ** 62]]))
    assert k[1, 0, 3, 0] == 2 and k[0, 0, 0, 0] == 4 and k.sum() == 48
    assert torch.equal(v, -k)


def _attention_args(**change):
    q, k, v, tables, lengths = make_case(2, 4, 2, 1, 16, 16, [20, 3], dtype=F32, seed=1)
    args = dict(q=q, k_pages=k, v_pages=v, tables=tables, lengths=lengths)
    args.update({name: f(args) for name, f in change.items()})
    return args


@pytest.mark.parametrize("change,kw,error,match", [
    (dict(q=lambda a: a["q"][0]), {}, ValueError, "q must use"),
    (dict(q=lambda a: a["q"][..., :8]), {}, ValueError, "head dimension"),
    (dict(q=lambda a: a["q"][:, :3]), {}, ValueError, "divisible"),
    (dict(q=lambda a: a["q"][:, :, :0]), {}, ValueError, "non-empty"),
    (dict(q=lambda a: a["q"].double()), {}, ValueError, "dtype"),
    (dict(k_pages=lambda a: None), {}, TypeError, "torch.Tensor"),
    (dict(v_pages=lambda a: a["v_pages"][1:]), {}, ValueError, "matching"),
    (dict(v_pages=lambda a: a["v_pages"].half()), {}, ValueError, "same dtype"),
    (dict(tables=lambda a: a["tables"].long()), {}, ValueError, "int32"),
    (dict(tables=lambda a: a["tables"][:1]), {}, ValueError, "tables"),
    (dict(tables=lambda a: a["tables"][0]), {}, ValueError, "tables"),
    (dict(tables=lambda a: a["tables"][:, :0]), {}, ValueError, "tables"),
    (dict(lengths=lambda a: a["lengths"].long()), {}, ValueError, "lengths"),
    (dict(lengths=lambda a: [20, 3]), {}, TypeError, "lengths"),
    (dict(q=lambda a: a["q"].requires_grad_()), {}, RuntimeError, "inference-only"),
    ({}, dict(causal=1), TypeError, "causal"),
    ({}, dict(scale=math.inf), ValueError, "finite"),
    ({}, dict(scale="x"), TypeError, "scale"),
    ({}, dict(backend="cuda"), ValueError, "backend"),
    ({}, dict(backend="hip"), RuntimeError, "gfx950"),
])
def test_attention_refusals(change, kw, error, match):
    with pytest.raises(error, match=match):
        paged_attention(**_attention_args(**change), **kw)


@pytest.mark.parametrize("change,error,match", [
    (dict(new_k=lambda a: a["new_k"][:, :, :0], new_v=lambda a: a["new_v"][:, :, :0]), ValueError, "empty"),
    (dict(new_v=lambda a: a["new_v"][:1]), ValueError, "matching"),
    (dict(new_k=lambda a: a["new_k"][:, :1], new_v=lambda a: a["new_v"][:, :1]), ValueError, "heads"),
    (dict(new_v=lambda a: a["new_v"].double()), ValueError, "dtype"),
    (dict(slots=lambda a: a["slots"].int()), ValueError, "slots"),
    (dict(slots=lambda a: a["slots"][:, :2]), ValueError, "slots"),
    (dict(slots=lambda a: [0]), TypeError, "slots"),
    (dict(k_pages=lambda a: a["k_pages"][:1].expand(4, -1, -1, -1)), ValueError, "expanded"),
    (dict(backend=lambda a: "sdpa"), ValueError, "append backend"),
    (dict(backend=lambda a: "hip"), RuntimeError, "gfx950"),
])
def test_append_refusals(change, error, match):
    args = dict(k_pages=torch.zeros(4, 2, 16, 8), v_pages=torch.zeros(4, 2, 16, 8),
                new_k=torch.zeros(2, 2, 3, 8), new_v=torch.zeros(2, 2, 3, 8),
                slots=torch.full((2, 3), -1))
    args.update({name: f(args) for name, f in change.items()})
    with pytest.raises(error, match=match):
        paged_append(**args)


@pytest.mark.parametrize("kw", [dict(batch=0), dict(max_len=True), dict(num_pages=-1), dict(page=0),
                                dict(max_len=2 ** 31), dict(num_pages=2 ** 30)])
def test_table_sizes(kw):
    with pytest.raises(ValueError):
        _table(**kw)


@pytest.mark.parametrize("counts,width,error", [
    (torch.zeros(3), 1, ValueError), (torch.zeros(2, dtype=torch.int32), 1, ValueError),
    (torch.zeros(3, dtype=torch.int32), None, ValueError), (1.0, 1, TypeError), (True, 1, TypeError),
    (-1, 1, ValueError), (5, 4, ValueError), (1, 0, ValueError),
])
def test_reserve_refusals(counts, width, error):
    table = _table()
    with pytest.raises(error):
        table.reserve(counts, width=width)
    assert table.lengths.tolist() == [0, 0, 0] and table.num_free() == 8


def test_trim_and_cache_refusals():
    table = _table()
    with pytest.raises(ValueError):
        table.trim(-1)
    with pytest.raises(TypeError):
        table.trim([1, 2, 3])
    with pytest.raises(ValueError, match="append backend"):
        table.trim(0, backend="sdpa")
    with pytest.raises(RuntimeError, match="gfx950"):
        table.reserve(1, backend="hip")
    with pytest.raises(TypeError):
        PagedKVCache(None, 1, 8, dtype=F32)
    with pytest.raises(ValueError):
        PagedKVCache(table, 0, 8, dtype=F32)


def test_a_refused_step_stores_nothing():
    table = _table()
    cache = PagedKVCache(table, 2, 8, dtype=F32)
    cache.k_pages.zero_()
    cache.v_pages.zero_()
    slots = table.reserve(1)
    new = torch.ones(3, 2, 1, 8)
    q = torch.ones(3, 4, 1, 8)
    for kw, error in ((dict(attention_backend="hip"), RuntimeError), (dict(causal=None), TypeError),
                      (dict(append_backend="x"), ValueError)):
        with pytest.raises(error):
            cache.append_and_attend(q, new, new, slots, **kw)
    with pytest.raises(RuntimeError, match="inference-only"):
        cache.append_and_attend(q.requires_grad_(), new, new, slots)
    assert (cache.k_pages == 0).all() and (cache.v_pages == 0).all()


def test_oracle_bound_is_not_loose():
    """The bound that GPU results are held to rejects one missing key in a
    hundred. (It does not reject a result rounded to bf16 once: the rounding of
    P alone may cost 2 u sum w |v|, more than that where values cancel.)"""
    args = make_case(1, 2, 1, 1, 64, 16, [100], dtype=torch.float16, seed=3)
    o, _, tol, _ = attention64(*args)
    short = attention64(*args[:4], torch.tensor([99], dtype=torch.int32))[0]
    assert bool(((short - o).abs() > tol).any())


def test_fused_needs_the_kernels():
    table = _table()
    cache = PagedKVCache(table, 2, 8, dtype=F32)
    cache.k_pages.zero_()
    new = torch.ones(3, 2, 1, 8)
    with pytest.raises(ValueError, match="fused"):
        cache.append_and_attend(torch.ones(3, 4, 1, 8), new, new, table.reserve(1), append_backend="fused")
    assert (cache.k_pages == 0).all()


def test_reserve_refuses_a_width_beyond_30_bits():
    table = _table()
    for width in (2 ** 64, 2 ** 63, 2 ** 30, -2 ** 64):
        with pytest.raises(ValueError, match="width"):
            table.reserve(1, width=width)
    assert table.lengths.tolist() == [0, 0, 0] and table.num_free() == 8


def test_broken_state_stays_inside():
    """Lengths, tables, counts and stacks that no allocator leaves behind: slots
    name places of the pool or -1, and a refused request is left as it was."""
    for height, length, entry in ((10 ** 9, 5, 3), (-4, 10 ** 9, -1), (2, -50, 10 ** 9), (8, 2 ** 31 - 1, -2 ** 31)):
        table = _table(4, 96, 8)
        table.tables.fill_(entry)
        table.free_pages[::2] = entry
        table.lengths.fill_(length)
        table.free_count.fill_(height)
        slots = table.reserve(20)
        assert ((slots >= -1) & (slots < 8 * 16)).all()
        if length > 96:
            assert (table.lengths == length).all() and int(table.refused) == 4
        table.trim(3)
        assert 0 <= table.num_free() <= 8 and (table.lengths <= 3).all() and (table.lengths >= 0).all()


def test_forward_mode_gradients_are_refused():
    import torch.autograd.forward_ad as fwd

    args = _attention_args()
    table = _table()
    cache = PagedKVCache(table, 2, 8, dtype=F32)
    cache.k_pages.zero_()
    cache.v_pages.zero_()
    slots, new = table.reserve(1), torch.ones(3, 2, 1, 8)
    with fwd.dual_level():
        dual = fwd.make_dual(new, torch.ones_like(new))
        for name in ("q", "k_pages", "v_pages"):
            with pytest.raises(RuntimeError, match="inference-only"):
                paged_attention(**dict(args, **{name: fwd.make_dual(args[name], torch.ones_like(args[name]))}))
        for k, v in ((dual, new), (new, dual)):
            for call in (cache.append, lambda *a: cache.append_and_attend(torch.ones(3, 4, 1, 8), *a)):
                with pytest.raises(RuntimeError, match="inference-only"):
                    call(k, v, slots)
        assert (cache.k_pages == 0).all() and (cache.v_pages == 0).all()
        paged_attention(**args)
    with pytest.raises(RuntimeError, match="inference-only"):
        torch.func.jvp(lambda q: paged_attention(**dict(args, q=q)), (args["q"],), (args["q"],))
