"""The 8-bit cache from its definition: blocks one after the other, codes looked
up among all of e4m3's values, in 64 bits on the CPU."""
import math

import torch

from tests.paged_oracle import attention64

BLOCK = 16
# Values of the codes 0 to 126 (127 is NaN): 3 bits of mantissa, exponents from
# -6 on, subnormal below.
VALUES = torch.tensor([(m if e == 0 else 8 + m) * 2.0 ** (max(e, 1) - 10) for e in range(16) for m in range(8)][:127],
                      dtype=torch.float64)


def round_e4m3(x):
    """The nearest value, of two equally near the one whose code is even;
    magnitudes up to 448."""
    a = x.abs()
    hi = torch.searchsorted(VALUES, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    below, above = a - VALUES[lo], VALUES[hi] - a
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return torch.copysign(VALUES[code], x)


def scale_of(largest):
    s = 2.0 ** -126
    while largest > 448 * s:
        s *= 2
    return s


def top_of(dtype):
    return 2.0 ** (16 if dtype == torch.float16 else 128)


class Cache:
    """Pools as the values of their codes, in 64 bits."""

    def __init__(self, k_pages, v_pages, scales):
        self.pools = [t.detach().cpu().float().double() for t in (k_pages, v_pages)]
        self.scales = scales.detach().cpu().double()

    def append(self, new_k, new_v, slots):
        pages, heads, page, _ = self.pools[0].shape
        top = top_of(new_k.dtype)
        for b, row in enumerate(slots.tolist()):
            blocks = {}
            for t, slot in enumerate(row):
                if 0 <= slot < pages * page:
                    blocks.setdefault(slot // BLOCK, []).append((slot % BLOCK, t))
            for block, rows in blocks.items():
                at, where = block // (page // BLOCK), block % (page // BLOCK)
                for h in range(heads):
                    for i, new in enumerate((new_k, new_v)):
                        x = new[b, h, [t for _, t in rows]].detach().cpu().double()
                        fin = x[x.isfinite()].abs()
                        s = scale_of(float(fin.max()) if fin.numel() else 0.0)
                        mine = self.pools[i][at, h, where * BLOCK:(where + 1) * BLOCK]
                        old = float(self.scales[at, h, where, i])
                        if 0 not in [r for r, _ in rows] and old >= s:
                            s = old
                        elif 0 not in [r for r, _ in rows]:
                            mine[:] = torch.where(mine.isnan(), mine, round_e4m3(mine * (old / s)))
                        # The largest value that stands for one of the type.
                        y = (x / s).clamp(-448, 448)
                        y = torch.where(x.isfinite(), round_e4m3(y.nan_to_num(0)), math.nan)
                        while bool((y.abs() * s >= top).any()):
                            over = y.abs() * s >= top
                            down = VALUES[(torch.searchsorted(VALUES, y.abs().nan_to_num(0)) - 1).clamp(min=0)]
                            y = torch.where(over, torch.copysign(down, y), y)
                        mine[[r for r, _ in rows]] = y
                        self.scales[at, h, where, i] = s

    def assert_matches(self, k_pages, v_pages, scales, rows=None):
        """Same values everywhere, or in the given slots; same scales."""
        assert torch.equal(scales.cpu().double(), self.scales)
        for got, want in zip((k_pages, v_pages), self.pools):
            got = got.cpu().float().double()
            same = (got == want) | (got.isnan() & want.isnan())
            if rows is not None:
                page = got.shape[2]
                same = same[torch.div(rows, page, rounding_mode="floor"), :, rows % page]
            assert bool(same.all()), f"{int((~same).sum())} of {same.numel()} differ"

    def held(self, dtype):
        """The pools as they read back, in 64 bits: code times scale in the
        16-bit type (exact but below its smallest value)."""
        out = []
        for i, pool in enumerate(self.pools):
            s = self.scales[..., i].repeat_interleave(BLOCK, 2)[..., None]
            out.append((pool * s).to(dtype).double())
        return out

    def read(self, tables, lengths, width, starts, dtype):
        pages, heads, page, d = self.pools[0].shape
        k, v = self.held(dtype)
        out = [torch.zeros(len(lengths), heads, width, d, dtype=torch.float64) for _ in range(2)]
        for b, n in enumerate(lengths.tolist()):
            for t in range(width):
                at = max(starts[b], 0) + t
                if at < n and at < tables.shape[1] * page:
                    p = int(tables[b, at // page])
                    if 0 <= p < pages:
                        out[0][b, :, t], out[1][b, :, t] = k[p, :, at % page], v[p, :, at % page]
        return out


def make_cache(batch, hkv, d, page, lengths, *, dtype, seed, device="cpu", spare=3, wild=True):
    """Pools, scales, tables and lengths of requests that hold random rows,
    blocks of very different sizes if ``wild``; pages in no order; rows of nobody
    NaN, with scales that are theirs."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=g).tolist()
    columns = max(max(held), 1) + 1
    tables = torch.full((batch, columns), -1, dtype=torch.int32)
    codes = [torch.randint(0, 127, (pages, hkv, page, d), generator=g)
             + 128 * torch.randint(0, 2, (pages, hkv, page, d), generator=g) for _ in range(2)]
    spread = 6 if wild else 1
    exponent = torch.randint(-8 - spread, -8 + spread, (pages, hkv, page // BLOCK, 2), generator=g)
    scales = torch.exp2(exponent.float())
    mine = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for c in range(held[b]):
            p = order.pop()
            tables[b, c] = p
            mine[p, :min(page, n - c * page)] = True
    # Rows padded to 16 bytes, the padding NaN.
    codes = [torch.cat((torch.where(mine[:, None, :, None], c, 127), torch.full((pages, hkv, page, -d % 16), 127)), 3)
             for c in codes]
    pools = [c.to(torch.uint8).to(device).view(torch.float8_e4m3fn)[..., :d] for c in codes]
    lens = torch.tensor(lengths, dtype=torch.int32)
    return (*pools, *(t.to(device) for t in (scales, tables, lens)))


def assert_attention(got, q, k, v, tables, lengths, *, lse=None, **kw):
    """``paged_oracle``'s bound, and the rounding of an output below the type's
    smallest normal value, where blocks of tiny values lead: there a step is
    smallest_normal * eps, not eps of the value, and half of it is the error
    (fp16: 2^-14 2^-10 / 2 = 2^-25)."""
    o, ls, tol, ls_tol = attention64(q, k, v, tables, lengths, **kw)
    info = torch.finfo(got.dtype)
    tol = tol + info.smallest_normal * info.eps / 2
    err = (got.cpu().double() - o).abs()
    worst = int((err - tol).flatten().nan_to_num(math.inf).argmax())
    assert bool((err <= tol).all()), (
        f"{int((~(err <= tol)).sum())} of {err.numel()} outside; worst at {worst}: got "
        f"{float(got.flatten()[worst])} want {float(o.flatten()[worst])} +- {float(tol.flatten()[worst])}")
    if lse is not None:
        x = lse.cpu().double()
        assert torch.equal(x == -math.inf, ls == -math.inf)
        fin = ls > -math.inf
        assert bool(((x - ls).abs()[fin] <= ls_tol[fin]).all()), float((x - ls).abs()[fin].max())
