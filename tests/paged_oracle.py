"""The paged cache from its definition: the allocator page by page in Python
lists, attention position by position in 64 bits on the CPU, with the bound
that 16-bit kernels are held to."""
import math

import torch


class Pages:
    """``PageTable`` in lists: same order of pages on the stack."""

    def __init__(self, batch, columns, num_pages, page):
        self.tables = [[-1] * columns for _ in range(batch)]
        self.lengths = [0] * batch
        self.free = list(range(num_pages - 1, -1, -1))
        self.page, self.refused = page, 0

    def _pages(self, tokens):
        return -(-tokens // self.page)

    def reserve(self, counts, width):
        slots, asked, room, self.refused = [], 0, len(self.free), 0
        for b, c in enumerate(counts):
            row = [-1] * width
            held = self.lengths[b]
            fits = 0 <= c <= width and held + c <= len(self.tables[b]) * self.page
            need = self._pages(held + c) - self._pages(held) if fits else 0
            asked += need
            if not fits or (need and asked > room):
                self.refused += 1
            else:
                for i in range(need):
                    self.tables[b][self._pages(held) + i] = self.free.pop()
                for t in range(c):
                    at = held + t
                    row[t] = self.tables[b][at // self.page] * self.page + at % self.page
                self.lengths[b] = held + c
            slots.append(row)
        return slots

    def trim(self, lengths):
        back = []
        for b, n in enumerate(lengths):
            keep = min(max(n, 0), self.lengths[b])
            for col in range(self._pages(keep), self._pages(self.lengths[b])):
                back.append(self.tables[b][col])
                self.tables[b][col] = -1
            self.lengths[b] = keep
        self.free.extend(reversed(back))

    def assert_matches(self, table):
        assert table.lengths.tolist() == self.lengths
        assert table.num_free() == len(self.free)
        assert table.free_pages[:len(self.free)].tolist() == self.free
        assert table.tables.tolist() == self.tables
        assert int(table.refused) == self.refused
        assert table.counters[2:].tolist() == [0, 0]


def attention64(q, k_pages, v_pages, tables, lengths, *, causal=False, scale=None):
    """O and LSE in 64 bits, and how far a kernel may be off.

    For a row with weights w and A = sum w |v|, in units of the input type's
    half step u = eps / 2:
    - P is rounded to the type before the second product and the denominator
      sums the rounded P: |sum w (d_j - d) v_j| <= 2 u A;
    - a score is a sum of D products in fp32, a scale and a difference:
      ds <= (D + 4) 2^-24 |scale| max_j sum_d |q_d k_jd|, and exp2 is good to
      2^-21; both enter numerator and denominator: 2 (ds + 2^-21) A;
    - sums over n keys in fp32, in any order, numerator and denominator, and
      the merge of parts: 2 (n + 8) 2^-24 A;
    - the output is rounded once: u |O|.
    LSE: u + ds + 2^-21 + n 2^-24, and its own rounding 2^-23 |LSE|.
    """
    b, hq, sq, d = q.shape
    pages, hkv, page, _ = k_pages.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    q, k_pages, v_pages = (t.detach().cpu().double() for t in (q, k_pages, v_pages))
    tables, lengths = tables.cpu().long(), lengths.cpu().tolist()
    out = torch.zeros((b, hq, sq, d), dtype=torch.float64)
    lse = torch.full((b, hq, sq), -math.inf, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse_tol = torch.zeros_like(lse)
    for i in range(b):
        n = min(max(lengths[i], 0), tables.shape[1] * page)
        pos = torch.arange(n)
        ids = tables[i][pos // page]
        inside = (ids >= 0) & (ids < pages)
        pos, ids = pos[inside], ids[inside]
        for h in range(hkv):
            k, v = k_pages[ids, h, pos % page], v_pages[ids, h, pos % page]
            for r in range(sq):
                m = int((pos < n - (sq - 1 - r)).sum()) if causal else len(pos)
                if m == 0:
                    continue
                rows = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                x = q[i, rows, r]
                s = x @ k[:m].T * scale
                w = torch.softmax(s, -1)
                o = w @ v[:m]
                big = w @ v[:m].abs()
                ds = (d + 4) * 2.0 ** -24 * abs(scale) * (x.abs() @ k[:m].abs().T).amax(-1, keepdim=True)
                out[i, rows, r] = o
                tol[i, rows, r] = u * o.abs() + (2 * u + 2 * (ds + 2.0 ** -21) + 2 * (m + 8) * 2.0 ** -24) * big
                ls = torch.logsumexp(s, -1)
                lse[i, rows, r] = ls
                lse_tol[i, rows, r] = u + ds[:, 0] + 2.0 ** -21 + m * 2.0 ** -24 + 2.0 ** -23 * ls.abs()
    return out, lse, tol, lse_tol


def assert_attention(got, q, k_pages, v_pages, tables, lengths, *, lse=None, **kw):
    o, ls, tol, ls_tol = attention64(q, k_pages, v_pages, tables, lengths, **kw)
    err = (got.cpu().double() - o).abs()
    over = (err - tol).flatten()
    worst = int(over.nan_to_num(math.inf).argmax())
    assert bool((err <= tol).all()), (
        f"{int((~(err <= tol)).sum())} of {err.numel()} outside; worst at {worst}: got "
        f"{float(got.flatten()[worst])} want {float(o.flatten()[worst])} +- {float(tol.flatten()[worst])}")
    if lse is not None:
        x = lse.cpu().double()
        assert torch.equal(x == -math.inf, ls == -math.inf)
        fin = ls > -math.inf
        assert bool(((x - ls).abs()[fin] <= ls_tol[fin]).all()), float((x - ls).abs()[fin].max())


def make_case(batch, hq, hkv, sq, d, page, lengths, *, dtype, seed, device="cpu", spare=3,
              values=1.0, junk=float("nan")):
    """q, pools, tables, lengths: every request's pages in no order, the rows
    behind its last and the pages of nobody filled with ``junk``, and the table
    entries behind the last page with numbers that name no page."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=g).tolist()
    columns = max(held) + 1
    tables = torch.randint(-2 ** 31, 2 ** 31 - 1, (batch, columns), generator=g)
    tables = torch.where((tables >= 0) & (tables < pages), -1, tables).to(torch.int32)
    k = torch.full((pages, hkv, page, d), junk, dtype=dtype)
    v = k.clone()
    for b, n in enumerate(lengths):
        for c in range(held[b]):
            at = order.pop()
            tables[b, c] = at
            m = min(page, n - c * page)
            k[at, :, :m] = (torch.randn(hkv, m, d, generator=g) * values).to(dtype)
            v[at, :, :m] = torch.randn(hkv, m, d, generator=g).to(dtype)
    q = torch.randn(batch, hq, sq, d, generator=g).to(dtype)
    lens = torch.tensor(lengths, dtype=torch.int32)
    return tuple(t.to(device) for t in (q, k, v, tables, lens))
