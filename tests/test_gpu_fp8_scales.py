"""Scales of blocks that no row of a request is in, in attention and read over
8-bit pools: they may hold anything."""
import math

import pytest
import torch

from kotflash_amd.paged_fp8 import fp8_attention, fp8_read
from tests.fp8_oracle import BLOCK, Cache, assert_attention, make_cache

pytestmark = pytest.mark.gpu
F16, FP8 = torch.float16, torch.float8_e4m3fn


def _case(hq, sq, d, page, lengths):
    """Requests whose page 0 is nobody's."""
    k8, v8, scales, tables, lens = make_cache(len(lengths), 2, d, page, lengths, dtype=F16, seed=d + page, device="cuda",
                                              wild=False)
    k8, v8 = (torch.cat((t.view(torch.uint8)[:1], t.view(torch.uint8))).view(FP8) for t in (k8, v8))
    scales = torch.cat((scales[:1], scales))
    tables = torch.where(tables >= 0, tables + 1, tables)
    q = torch.randn(len(lengths), hq, sq, d, generator=torch.Generator().manual_seed(1)).half().cuda()
    return q, k8, v8, scales, tables, lens


def _unseen(case):
    """Blocks [pages, page / 16] without a visible row."""
    _, k8, _, scales, tables, lens = case
    pages, _, page, _ = k8.shape
    seen = torch.zeros(pages, page // BLOCK, dtype=torch.bool)
    for row, n in zip(tables.tolist(), lens.tolist()):
        for at in range(0, min(n, len(row) * page), BLOCK):
            if 0 <= row[at // page] < pages:
                seen[row[at // page], at % page // BLOCK] = True
    return ~seen.to(scales.device)


@pytest.mark.parametrize("value", [math.nan, math.inf, -1e38])
@pytest.mark.parametrize("hq,sq,causal", [(4, 1, False), (8, 4, True), (48, 1, False), (128, 1, False), (16, 16, True)])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 48), (128, 128)])
def test_blocks_without_rows(value, hq, sq, causal, d, page):
    case = _case(hq, sq, d, page, [0, 1, 16, 17, 40, 70, 129, 200])
    want = fp8_attention(*case, causal=causal, return_lse=True, backend="hip")
    scales = case[3].clone()
    scales.permute(0, 2, 1, 3)[_unseen(case)] = value
    got = fp8_attention(*case[:3], scales, *case[4:], causal=causal, return_lse=True, backend="hip")
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    held = [fp8_read(*case[1:3], s, *case[4:], 210, dtype=F16, backend="hip") for s in (case[3], scales)]
    assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(*held))


@pytest.mark.parametrize("hq", [4, 48, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_pages_outside_the_pool(hq, d):
    """Their positions are not seen, whatever page 0's scales hold."""
    case = _case(hq, 1, d, 32, [100, 64, 7, 200])
    q, k8, v8, scales, tables, lens = case
    tables[0, 1], tables[1, 0], tables[3, 6] = -1, 10 ** 6, -2 ** 31
    scales[0] = math.nan
    o, lse = fp8_attention(*case, return_lse=True, backend="hip")
    assert_attention(o, q, *Cache(k8, v8, scales).held(F16), tables, lens, lse=lse)
