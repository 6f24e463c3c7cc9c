"""Attention over 8-bit pools in memory orders other than page after page."""
import pytest
import torch

from kotflash_amd import _hip
from kotflash_amd.paged_fp8 import fp8_append, fp8_attention, fp8_read
from tests.fp8_oracle import Cache, make_cache
from tests.paged_oracle import attention64

pytestmark = pytest.mark.gpu
F16, FP8 = torch.float16, torch.float8_e4m3fn


def _q(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).half().cuda()


def _assert_close(o, q, k, v, tables, lens):
    """``attention64``'s bound, half the output's smallest step (2^-24 / 2 in
    fp16), and what rounding P to fp16 adds where P is below the type's smallest
    normal value, which relative half steps leave out: P = 2^(s - m + 7), m at
    most the row's maximum, so the largest P, and the denominator, are at
    least 2^7. A P below 2^-14 becomes a multiple of 2^-24, off by at most 2^-25:
    2^-32 |v_j| of the output per key, and 2^-32 |O| per key by the denominator.
    It shows where a row's weight lies on tiny values and V holds far larger."""
    want, _, tol, _ = attention64(q, k, v, tables, lens)
    page, group = k.shape[2], q.shape[1] // k.shape[1]
    tol = tol + 2.0 ** -25
    for b, n in enumerate(lens.tolist()):
        pos = torch.arange(n)
        rows = v[tables[b].cpu().long()[pos // page], :, pos % page]  # [n, Hkv, D]
        more = rows.abs().sum(0).repeat_interleave(group, 0)[:, None]
        tol[b] += 2.0 ** -32 * (more + n * want[b].abs())
    err = (o.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("order", [(2, 0, 1, 3), (1, 2, 0, 3), (2, 1, 0, 3), (0, 2, 1, 3)])
def test_orders(order):
    """Positions, heads or pages outermost: the bits of contiguous pools."""
    q, pools = _q(3, 8, 2, 64), make_cache(3, 2, 64, 48, [50, 200, 9], dtype=F16, seed=4, device="cuda")
    want = fp8_attention(q, *pools, return_lse=True, backend="hip")
    back = [order.index(i) for i in range(4)]
    k8, v8 = (t.view(torch.uint8).permute(order).contiguous().permute(back).view(FP8) for t in pools[:2])
    got = fp8_attention(q, k8, v8, *pools[2:], return_lse=True, backend="hip")
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("hq", [8, 160, 320])
def test_rows_beyond_32_bits(hq):
    """Pools [page_size, pages, Hkv, D] of 6 GB, seen as [pages, Hkv, page_size,
    D]: 47.1 MB from one row of a page to the next, so that its last group of 16
    begins behind 4 GiB (112 * 47.1e6 = 5.3e9), and 47 rows are more than 2 GiB.
    The requests end 1 to 47 rows before the end of a step of 64 positions, with
    NaN behind them. With one, two and four waves per worker."""
    pages, hkv, d, page = 46000, 8, 128, 128
    lengths = [128, 113, 97, 81, 65, 17, 1, 250]
    k0, v0, sc, small, lens = make_cache(len(lengths), hkv, d, page, lengths, dtype=F16, seed=6, device="cuda")
    k8, v8 = (torch.empty(page, pages, hkv, d, dtype=torch.uint8, device="cuda").view(FP8).permute(1, 2, 0, 3)
              for _ in range(2))
    scales = torch.zeros(pages, hkv, page // 16, 2, device="cuda")
    tables = small.clone()
    for i, p in enumerate(small[small >= 0].tolist()):
        to = pages - 1 - 4001 * i
        for pool, have in ((k8, k0), (v8, v0)):
            pool.view(torch.uint8)[to] = have.view(torch.uint8)[p]
        scales[to] = sc[p]
        tables[small == p] = to
    q = _q(len(lengths), hq, 1, d)
    assert _hip.fp8_decode_check(q, k8, v8, scales, tables.shape[1]) == 0
    o, lse = fp8_attention(q, k8, v8, scales, tables, lens, return_lse=True, backend="hip")
    want = fp8_attention(q, k0, v0, sc, small, lens, return_lse=True, backend="hip")
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    _assert_close(o, q, *Cache(k0, v0, sc).held(F16), small, lens)


def test_store_and_read_beyond_32_bits():
    """The store and the read of such a pool."""
    pages, hkv, d, page = 46000, 8, 128, 128
    k8, v8 = (torch.empty(page, pages, hkv, d, dtype=torch.uint8, device="cuda").view(FP8).permute(1, 2, 0, 3)
              for _ in range(2))
    scales = torch.zeros(pages, hkv, page // 16, 2, device="cuda")
    tables = torch.tensor([[pages - 1, 5]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([150], dtype=torch.int32, device="cuda")
    t = torch.arange(150, device="cuda")
    slots = (tables[0].long()[t // page] * page + t % page)[None]
    k, v = _q(1, hkv, 150, d), _q(1, hkv, 150, d, seed=1)
    fp8_append(k8, v8, scales, k, v, slots, backend="hip")
    small = [torch.zeros(2, hkv, page, d, device="cuda").to(FP8) for _ in range(2)]
    ss = torch.zeros(2, hkv, page // 16, 2, device="cuda")
    fp8_append(*small, ss, k, v, t[None], backend="torch")
    got = fp8_read(k8, v8, scales, tables, lens, 150, dtype=F16, backend="hip")
    want = fp8_read(*small, ss, torch.arange(2, dtype=torch.int32, device="cuda")[None], lens, 150, dtype=F16, backend="torch")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
