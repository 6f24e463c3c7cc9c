"""How far the 8-bit cache's values are off, element by element, by the scale
of each element's own block."""
import pytest
import torch

from kotflash_amd.paged import PageTable
from kotflash_amd.paged_fp8 import PagedKVCacheFP8

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _cache(dtype, batch=2, hkv=3, d=32, page=32, max_len=200):
    table = PageTable(batch, max_len, num_pages=batch * -(-max_len // page), page_size=page, device="cpu")
    return PagedKVCacheFP8(table, hkv, d, dtype=dtype)


def _spread(*shape, dtype, seed, scale=1.0):
    """Values of very different sizes within a block: one in 64 is 2^12 times as
    large, one in 64 as small."""
    g = torch.Generator().manual_seed(seed)
    x, pick = torch.randn(*shape, generator=g) * scale, torch.randint(0, 64, shape, generator=g)
    return torch.where(pick == 0, x * 64, torch.where(pick == 1, x / 64, x)).to(dtype)


def _scales_of(cache, slots, which):
    """Each token's scale, [B, Hkv, n, 1]."""
    page = cache.table.page_size
    return cache.scales[slots // page, :, slots % page // 16, which].transpose(1, 2)[..., None].double()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("scale", [5.0, 0.01])
def test_one_rounding(dtype, scale):
    """A value is off by at most 2^-4 of itself, or half the smallest step of its
    block, 2^-10 of the scale. (Reading rounds nothing here: codes times scales of
    these sizes are values of every type.)"""
    cache = _cache(dtype)
    k, v = (_spread(2, 3, 90, 32, dtype=dtype, seed=i, scale=scale * 3.0 ** i) for i in range(2))
    slots = cache.table.reserve(90)
    cache.append(k, v, slots)
    for which, (got, x) in enumerate(zip(cache.read(90), (k, v))):
        s = _scales_of(cache, slots, which)
        err = (got.double() - x.double()).abs()
        assert bool((err <= torch.maximum(x.double().abs() / 16, s * 2.0 ** -10)).all())
        # Zero below half the smallest step, and the bound is reached there.
        small = x.double().abs() < s * 2.0 ** -10
        assert small.any() and not got[small].any()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rounding_of_grown_blocks(dtype):
    """Growth rounds codes below the normal ones again: half a step of each new
    scale more."""
    cache = _cache(dtype, batch=1, max_len=16)
    kept, scales = [], []
    for step, n in enumerate((5, 3, 1, 4)):
        x = _spread(1, 3, n, 32, dtype=dtype, seed=step, scale=4.0 ** step)
        slots = cache.table.reserve(n)
        cache.append(x, -x, slots)
        kept.append(x)
        scales.append([])
        for of_one in scales:
            of_one.append(_scales_of(cache, slots[:, :1], 0))
        at = 0
        for held, s in zip(kept, scales):
            got = cache.read(held.shape[2], start=at)
            tol = torch.maximum(held.double().abs() / 16, s[0] * 2.0 ** -10)
            for before, after in zip(s, s[1:]):
                tol = tol + torch.where(after > before, after * 2.0 ** -10, 0)
            for out, sign in zip(got, (1, -1)):
                assert bool(((sign * out.double() - held.double()).abs() <= tol).all())
            at += held.shape[2]
    assert len({float(s[0][0, 0, 0, 0]) for s in scales}) > 1  # it has grown
