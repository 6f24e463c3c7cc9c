"""Rotary positions and the 8-bit paged key-value cache, as timed cases.

A server holds its requests' keys and values in pages of a common pool,
``k_pages`` and ``v_pages`` [pages, Hkv, page, D] in e4m3 (4 significant bits,
largest value 448). A block is 16 positions of a page, one head; ``scales``
[pages, Hkv, page / 16, 2] holds its scale for K and for V, a power of two, and
a value is code * scale. A case is one of:

- rotary: queries and keys are turned by their positions, pair i of the first
  ``r`` dims by position * f_i; ``train`` takes the gradients too;
- write: new keys and values go to their slots (page * page size + offset).
  The block's scale is the least power of two s with |x| <= 448 s for the rows
  that come in; a block whose first row is not among them keeps its scale where
  that is larger, and where it grows the rows that are there are rounded to it;
- read: what the requests hold from a position on, in 16 bits, as a prompt's
  next chunk attends to it;
- attend: new tokens of every request (or a few drafts, causal among
  themselves) attend to all that it holds;
- step: one layer of a decoding step: fall back to the lengths before it, turn
  queries and keys, room in the page table, write, attend.

A second pass over the same state gives the same: the slots written are the
same, and a scale that has grown stays. ``own`` chooses between the plain form,
in elementary torch operations, and the package's own operators.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 16


def _case(op, b, top, *, page=16, n=1, counts="same", hq=0, hkv=0, d=0, dtype="bf16", spread="ragged",
          causal=False, empty=0, layout="bhsd", r=0, pairs="half", scaling="none", train=False, name=None):
    """``top``: tokens of the longest request, or the farthest position; ``n``:
    new tokens a request may bring; ``empty``: requests that hold nothing;
    ``r``: dims of a head that turn."""
    case = {"op": op, "b": b, "top": top, "page": page, "n": n, "counts": counts, "hq": hq, "hkv": hkv,
            "d": d, "dtype": dtype, "spread": spread, "causal": causal, "empty": empty, "layout": layout,
            "r": r, "pairs": pairs, "scaling": scaling, "train": train}
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # The new token of each of 64 requests, far into their conversations.
        _case("rotary", 64, 30000, hq=32, hkv=8, d=128, r=128, name="rotary_step"),
        # Prompts, on the transposed views that a model's projections give.
        _case("rotary", 8, 0, n=4096, hq=32, hkv=8, d=128, r=128, layout="bshd", name="rotary_prompts"),
        # A training step of a GQA model that turns half of each head, in
        # neighbouring pairs, with frequencies stretched for a longer context.
        _case("rotary", 2, 0, n=4096, hq=16, hkv=4, d=128, dtype="fp16", r=64, pairs="interleaved",
              scaling="ramp", layout="bshd", train=True, name="rotary_train"),
        # The new token of each of 64 requests, as a decoding step stores it.
        _case("write", 64, 4000, hkv=8, d=128, name="write_step"),
        # Sixteen prompts of their own lengths.
        _case("write", 16, 4096, n=4096, counts="ragged", hkv=8, d=128, dtype="fp16", layout="bshd",
              name="write_prompts"),
        # What a conversation holds, before its next prompt.
        _case("read", 1, 900, hkv=2, d=64, dtype="fp16", spread="even", name="read_900"),
        # The same for a batch with long prefixes.
        _case("read", 16, 8192, hkv=8, d=128, page=64, name="read_batch"),
        # Two short conversations of a small model.
        _case("attend", 2, 2000, hq=8, hkv=2, d=64, dtype="fp16", spread="even", name="attend_2k"),
        # A serving batch of a GQA model, requests of very different lengths.
        _case("attend", 64, 8192, hq=32, hkv=8, d=128, name="attend_batch"),
        # A model with a single key-value head and an odd head dim, requests
        # that have just come in and hold nothing yet among them.
        _case("attend", 48, 6001, hq=16, hkv=1, d=96, page=32, empty=3, name="attend_mqa"),
        # Verification of four draft tokens each.
        _case("attend", 8, 31000, n=4, hq=32, hkv=8, d=64, dtype="fp16", causal=True, name="attend_drafts"),
        # One layer of a decoding step of a batch.
        _case("step", 32, 4096, hq=32, hkv=8, d=128, r=128, name="step_batch"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above, no larger than the largest listed."""
    op = rng.choice(["rotary", "rotary", "write", "write", "read", "attend", "attend", "attend", "step"])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    dtype = rng.choice(["fp16", "bf16"])
    spread = rng.choice(["ragged", "ragged", "even"])
    layout = rng.choice(["bhsd", "bshd"])
    while True:
        b = _log(rng, 1, 256)
        hkv = rng.choice([1, 2, 4, 8, 16])
        hq = hkv * rng.choice([1, 2, 4, 7, 8, 16])
        d = rng.choice([32, 64, 64, 80, 96, 112, 128, 128])
        empty = rng.randint(0, b // 4)
        if hq > 64:
            continue
        turn = {"r": rng.choice([d, d, d // 2]), "pairs": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "base", "ramp"])}
        if op == "rotary":
            d = rng.choice([d, 40, 72, 192, 256])
            turn["r"] = rng.choice([d, d // 2])
            n = rng.choice([1, _log(rng, 2, 8192), _log(rng, 2, 8192)])
            case = _case(op, b, _log(rng, 1, 1_000_000), n=n, hq=hq, hkv=hkv, d=d, dtype=dtype, layout=layout,
                         train=rng.random() < 0.4, **turn)
            if b * n * (hq + hkv) * d <= (8e7 if case["train"] else 1.6e8):
                return case
            continue
        if op == "write":
            n = rng.choice([1, 1, _log(rng, 2, 4096)])
            case = _case(op, b, max(n, _log(rng, 16, 8192)), page=page, n=n, counts="ragged" if n > 1 else "same",
                         hkv=hkv, d=d, dtype=dtype, spread=spread, empty=empty, layout=layout)
        elif op == "read":
            case = _case(op, b, _log(rng, 16, 16384), page=page, hkv=hkv, d=d, dtype=dtype, spread=spread,
                         empty=empty)
        else:
            n = rng.choice([1, 1, 1, 2, 3, 4, 8])
            case = _case(op, b, _log(rng, 16, 131072), page=page, n=n, hq=hq, hkv=hkv, d=d, dtype=dtype,
                         spread=spread, empty=empty, causal=n > 1 and rng.random() < 0.8,
                         **(turn if op == "step" else {}))
        # The pools, and what the plain form gathers of them.
        if b * (case["top"] + case["n"]) * hkv * d <= (5.4e8 if op == "attend" else 1.3e8):
            return case


def _cdiv(a, b):
    return -(-a // b)


def _lengths(case, seed):
    """Tokens that the requests hold: evenly spread from a sixteenth of the
    longest up (or all as long as it), in the seed's order. Prompts that are
    written begin with nothing."""
    b, top = case["b"], case["top"]
    if case["op"] == "write" and case["n"] > 1:
        return [0] * b
    low = top if case["spread"] == "even" else top // 16
    lens = [top - (top - low) * i // b for i in range(b)]
    for i in range(case["empty"]):
        lens[b - 1 - i] = 0
    random.Random(seed).shuffle(lens)
    return lens


def _counts(case, seed):
    """New tokens of each request: n, or evenly spread over 0 to n."""
    b, n = case["b"], case["n"]
    counts = [n] * b if case["counts"] == "same" else [n - n * i // b for i in range(b)]
    random.Random(seed + 1).shuffle(counts)
    return counts


def _held(case, seed):
    """Tokens that the tables cover: with the new ones where they are written."""
    lens = _lengths(case, seed)
    if case["op"] not in ("write", "step"):
        return lens
    return [x + c for x, c in zip(lens, _counts(case, seed))]


def _sizes(case):
    """Pages in the pool and columns of the block tables: room for everything,
    an eighth to spare."""
    page = case["page"]
    full = sum(_cdiv(x, page) for x in _held(case, 0))
    return full * 9 // 8 + 1, _cdiv(max(case["top"], case["n"]) + case["n"], page)


def _device(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _paging(case, seed):
    """Every request's pages, in no order."""
    page, (pages, columns) = case["page"], _sizes(case)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()
    held = _device([_cdiv(x, page) for x in _held(case, seed)])
    tables = torch.full((case["b"], columns), -1, dtype=torch.int32, device="cuda")
    mine = torch.arange(columns, device="cuda")[None, :] < held[:, None]
    tables[mine] = order[:int(held.sum())]
    return tables


def _slots(case, seed, tables):
    """Slots of the new tokens behind the lengths, -1 behind each request's."""
    page = case["page"]
    t = torch.arange(case["n"], device="cuda")
    position = _device(_lengths(case, seed), torch.int64)[:, None] + t
    pages = torch.gather(tables.long(), 1, (position // page).clamp(max=tables.shape[1] - 1))
    given = t < _device(_counts(case, seed))[:, None]
    return torch.where(given, pages * page + position % page, -1)


def _frequencies(case):
    """Radians per position of every pair, in 64 bits."""
    r, factor = case["r"], 4.0
    base = 10000.0 * (factor ** (r / (r - 2)) if case["scaling"] == "base" else 1.0)
    f = torch.tensor([base ** (-2 * i / r) for i in range(r // 2)], dtype=torch.float64)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "ramp":
        # Those that turn less than once in 4096 positions are slowed down by
        # the factor, those over four times are left, a line between.
        w = ((4096 * f / (2 * math.pi) - 1) / 3).clamp(0, 1)
        f = f * w + f / factor * (1 - w)
    return f


def _inputs(case, seed):
    """Pools with their scales, queries, new keys and values, gradients. Blocks
    differ in size, as heads and tokens do."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, b, n, d, hq, hkv = (case[x] for x in ("dtype", "b", "n", "d", "hq", "hkv"))
    dt = DTYPES[dt]

    def new(heads):
        if case["layout"] == "bshd":
            return torch.randn((b, n, heads, d), device="cuda", dtype=dt, generator=g).transpose(1, 2)
        return torch.randn((b, heads, n, d), device="cuda", dtype=dt, generator=g)

    t = {}
    if case["op"] != "rotary":
        pages, page = _sizes(case)[0], case["page"]
        codes, scales = [], []
        for _ in range(2):
            x = torch.randn((pages, hkv, page // BLOCK, BLOCK * d), device="cuda", dtype=dt, generator=g)
            x *= torch.exp(torch.randn((pages, hkv, page // BLOCK, 1), device="cuda", generator=g)).to(dt)
            s = _scale_for(x.abs().amax(-1).float())
            scales.append(s)
            codes.append((x / s[..., None].to(dt)).float().to(torch.float8_e4m3fn).reshape(pages, hkv, page, d))
        t.update(k=codes[0], v=codes[1], scales=torch.stack(scales, -1))
    if case["op"] in ("rotary", "attend", "step"):
        t["q"] = new(hq)
    if case["op"] in ("rotary", "write", "step"):
        t["new_k"] = new(hkv)
    if case["op"] in ("write", "step"):
        t["new_v"] = new(hkv)
    if case["train"]:
        t["dq"], t["dk"] = new(hq), new(hkv)
    return t


def _starts(case, seed):
    """First positions of the requests' new tokens."""
    if case["op"] == "step":
        return _lengths(case, seed)
    rng = random.Random(seed + 2)
    return [rng.randint(0, case["top"]) for _ in range(case["b"])]


def prepare(case, seed):
    op, page = case["op"], case["page"]
    state = {"case": case, **_inputs(case, seed)}
    if case["r"]:
        state["frequencies"] = _frequencies(case).cuda()
        state["starts"] = _device(_starts(case, seed))
    if op != "rotary":
        tables = _paging(case, seed)
        state.update(tables=tables, lengths=_device(_held(case, seed)), slots=_slots(case, seed, tables))
    if op == "step":
        state["keep"] = _device(_lengths(case, seed))
    if case["train"]:
        state["q"].requires_grad_()
        state["new_k"].requires_grad_()
    if not own:
        return state
    if case["r"]:
        from kotflash_amd.rotary import Rotary

        state["rotary"] = Rotary(case["d"], rotary_dim=case["r"], interleaved=case["pairs"] == "interleaved",
                                 scaling=case["scaling"], factor=1.0 if case["scaling"] == "none" else 4.0,
                                 original_length=4096 if case["scaling"] == "ramp" else None, device="cuda")
    if op != "rotary":
        from kotflash_amd.paged import PageTable
        from kotflash_amd.paged_fp8 import PagedKVCacheFP8

        pages, columns = _sizes(case)
        table = PageTable(case["b"], columns * page, num_pages=pages, page_size=page, device="cuda")
        table.tables.copy_(state["tables"])
        table.lengths.copy_(state["lengths"])
        # Pages that belong to nobody.
        taken = torch.zeros(pages, dtype=torch.bool, device="cuda")
        taken[table.tables[table.tables >= 0].long()] = True
        left = (~taken).nonzero()[:, 0].to(torch.int32)
        table.free_pages[:len(left)] = left
        table.free_count.fill_(len(left))
        cache = PagedKVCacheFP8(table, case["hkv"], case["d"], dtype=DTYPES[case["dtype"]])
        cache.k_pages.copy_(state.pop("k"))
        cache.v_pages.copy_(state.pop("v"))
        cache.scales.copy_(state.pop("scales"))
        state.update(table=table, cache=cache)
    return state


# ---------------------------------------------------------------------------
# The plain form.

def _scale_for(largest):
    """The least power of two s >= 2^-126 with largest <= 448 s, in 32 bits."""
    mantissa, exponent = torch.frexp(largest)  # mantissa in [0.5, 1)
    exponent = torch.where(mantissa > 0.875, exponent + 1, exponent) - 9
    exponent = torch.where(largest > 0, exponent, -126).clamp(min=-126)
    return ((exponent + 127) << 23).view(torch.float32)  # 2^exponent, exactly


def _turned(x, angle, case, inverse):
    """The first r dims of x, pair by pair, by the angles; the rest as it is."""
    r = case["r"]
    c, s = angle.cos().float(), angle.sin().float()
    s = -s if inverse else s
    y = x.float().clone()
    if case["pairs"] == "half":
        one, two = y[..., :r // 2].clone(), y[..., r // 2:r].clone()
        y[..., :r // 2], y[..., r // 2:r] = one * c - two * s, one * s + two * c
    else:
        one, two = y[..., 0:r:2].clone(), y[..., 1:r:2].clone()
        y[..., 0:r:2], y[..., 1:r:2] = one * c - two * s, one * s + two * c
    return y.to(x.dtype)


def _angles(starts, n, frequencies):
    position = starts[:, None].double() + torch.arange(n, device="cuda")
    return (position[:, :, None] * frequencies)[:, None]


def _write(k, v, scales, new_k, new_v, slots, page):
    """Quantised rows to their slots; the blocks' scales, and their other rows
    where those have grown."""
    pages, h, _, d = k.shape
    given = slots >= 0
    at = slots[given]
    groups = page // BLOCK
    block = at // BLOCK  # over the pool: page * groups + group
    begun = torch.zeros(pages * groups, dtype=torch.bool, device="cuda")
    begun[block[at % BLOCK == 0]] = True
    touched = torch.zeros_like(begun)
    touched[block] = True
    for pool, new, which in ((k, new_k, 0), (v, new_v, 1)):
        x = new.transpose(1, 2)[given].float()  # [tokens, h, d]
        top = torch.zeros((pages * groups, h), device="cuda")
        top.scatter_reduce_(0, block[:, None].expand(-1, h), x.abs().amax(-1), "amax")
        old = scales[..., which].transpose(1, 2).reshape(pages * groups, h)
        need = _scale_for(top)
        scale = torch.where(touched[:, None], torch.where(begun[:, None], need, torch.maximum(old, need)), old)
        # [pages, groups, h, BLOCK, d] of the codes.
        codes = pool.view(torch.uint8).view(pages, h, groups, BLOCK, d).transpose(1, 2)
        grown = (touched & ~begun).nonzero()[:, 0]
        ratio = (old / scale)[grown][:, :, None, None]
        there = codes[grown // groups, grown % groups].view(torch.float8_e4m3fn).float()
        codes[grown // groups, grown % groups] = (there * ratio).to(torch.float8_e4m3fn).view(torch.uint8)
        fresh = (x / scale[block][:, :, None]).to(torch.float8_e4m3fn)
        codes[block // groups, block % groups, :, at % BLOCK] = fresh.view(torch.uint8)
        scales[..., which] = scale.view(pages, groups, h).transpose(1, 2)


def _values(pool, scales, pages, which):
    """What the pages [B, columns] hold, in 32 bits: [B, h, columns * page, d]."""
    b, columns = pages.shape
    _, h, page, d = pool.shape
    codes = pool.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()
    x = codes.view(b, columns, h, page // BLOCK, BLOCK, d) * scales[pages][..., which, None, None]
    return x.permute(0, 2, 1, 3, 4, 5).reshape(b, h, columns * page, d)


def _read(k, v, scales, tables, lengths, width, dtype):
    page = k.shape[2]
    pages = tables[:, :_cdiv(width, page)].clamp(min=0).long()
    there = torch.arange(width, device="cuda") < lengths[:, None]
    return [torch.where(there[:, None, :, None], _values(pool, scales, pages, which)[:, :, :width], 0.0).to(dtype)
            for which, pool in enumerate((k, v))]


def _attend(q, k, v, scales, tables, lengths, causal, longest):
    """softmax(q k^T / sqrt(d)) v in 32 bits over each request's positions; a
    row that sees nothing is zero."""
    b, hq, sq, d = q.shape
    hkv, page = k.shape[1], k.shape[2]
    columns = min(tables.shape[1], max(1, _cdiv(longest, page)))
    pages = tables[:, :columns].clamp(min=0).long()
    rows = q.reshape(b, hkv, (hq // hkv) * sq, d).float()
    s = torch.matmul(rows, _values(k, scales, pages, 0).transpose(-2, -1)) * (1.0 / math.sqrt(d))
    end = lengths[:, None].expand(b, sq)
    if causal:
        end = end - (sq - 1) + torch.arange(sq, device=q.device, dtype=torch.int32)[None, :]
    seen = torch.arange(columns * page, device=q.device, dtype=torch.int32)[None, None, :] < end[:, :, None]
    seen = seen.repeat(1, hq // hkv, 1)[:, None]
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, _values(v, scales, pages, 1)) / torch.where(total == 0, torch.ones_like(total), total)
    return o.reshape(b, hq, sq, d).to(q.dtype)


def _run_plain(state):
    case = state["case"]
    op, page, n = case["op"], case["page"], case["n"]
    if op == "rotary":
        angle = _angles(state["starts"], n, state["frequencies"])
        with torch.no_grad():
            out = {x: _turned(state[x], angle, case, False) for x in ("q", "new_k")}
            if case["train"]:
                out.update({x: _turned(state[x], angle, case, True) for x in ("dq", "dk")})
        return out
    k, v, scales, tables, lengths = (state[x] for x in ("k", "v", "scales", "tables", "lengths"))
    if op == "write":
        _write(k, v, scales, state["new_k"], state["new_v"], state["slots"], page)
        return {"k": k, "v": v, "scales": scales}
    if op == "read":
        return _read(k, v, scales, tables, lengths, case["top"], DTYPES[case["dtype"]])
    if op == "attend":
        return _attend(state["q"], k, v, scales, tables, lengths, case["causal"], case["top"])
    angle = _angles(state["starts"], n, state["frequencies"])
    q, new_k = (_turned(state[x], angle, case, False) for x in ("q", "new_k"))
    # Back to the lengths before the step, then room for its tokens: as many
    # pages as the tables have for them already.
    position = state["keep"][:, None] + torch.arange(n, device="cuda")
    slots = torch.gather(tables.long(), 1, position // page) * page + position % page
    _write(k, v, scales, new_k, state["new_v"], slots, page)
    o = _attend(q, k, v, scales, tables, state["keep"] + n, case["causal"], case["top"] + n)
    return {"o": o, "slots": slots, "k": k, "v": v, "scales": scales}


def run(state):
    if not own:
        return _run_plain(state)
    case = state["case"]
    if case["op"] == "rotary":
        q, k = state["rotary"](state["q"], state["new_k"], positions=state["starts"])
        if not case["train"]:
            return {"q": q, "new_k": k}
        dq, dk = torch.autograd.grad((q, k), (state["q"], state["new_k"]), (state["dq"], state["dk"]))
        return {"q": q.detach(), "new_k": k.detach(), "dq": dq, "dk": dk}
    cache = state["cache"]
    if case["op"] == "write":
        cache.append(state["new_k"], state["new_v"], state["slots"])
        return {"k": cache.k_pages, "v": cache.v_pages, "scales": cache.scales}
    if case["op"] == "read":
        return list(cache.read(case["top"]))
    if case["op"] == "attend":
        return cache.attend(state["q"], causal=case["causal"])
    table = state["table"]
    table.trim(state["keep"])
    q, k = state["rotary"](state["q"], state["new_k"], positions=table.lengths)
    slots = table.reserve(case["n"])
    o = cache.append_and_attend(q, k, state["new_v"], slots, causal=case["causal"])
    return {"o": o, "slots": slots, "k": cache.k_pages, "v": cache.v_pages, "scales": cache.scales}


def work(case):
    """Each input read once, each output written once."""
    b, n, hq, hkv, d = (case[x] for x in ("b", "n", "hq", "hkv", "d"))
    turned = b * n * (hq + hkv)
    if case["op"] == "rotary":
        return {"bytes": 4 * turned * d * (2 if case["train"] else 1),
                "flops": 3 * turned * case["r"] * (2 if case["train"] else 1)}
    lens, counts = _lengths(case, 0), _counts(case, 0)
    token = 2 * hkv * d  # K and V in 8 bits; scales of 8 bytes per block and head

    def blocks(x):
        return 8 * hkv * _cdiv(x, BLOCK)

    written = sum(3 * c * token + blocks(c) for c in counts)
    if case["op"] == "write":
        return {"bytes": written + 8 * b * n, "flops": 0}
    if case["op"] == "read":
        return {"bytes": sum(x * token + blocks(x) for x in lens) + b * case["top"] * 2 * token, "flops": 0}
    total = 0
    if case["op"] == "step":
        lens = [x + n for x in lens]
        total = written + 4 * turned * d + 8 * b * n
    total += sum(x * token + blocks(x) for x in lens) + 2 * b * hq * n * d * 2
    return {"bytes": total, "flops": 4 * d * hq * n * sum(lens)}


# ---------------------------------------------------------------------------
# From the definition, in 64 bits.

def _exact_turn(case, x, starts, inverse=False):
    """Pair by pair, as the product with a complex number of length 1."""
    r, n = case["r"], case["n"]
    place = torch.tensor(starts, dtype=torch.float64)[:, None] + torch.arange(n, dtype=torch.float64)
    angle = (place[:, :, None] * _frequencies(case)).cuda()
    unit = torch.polar(torch.ones_like(angle), -angle if inverse else angle)[:, None]
    out = x.detach().double().clone()
    i = torch.arange(r // 2, device="cuda")
    one, two = (i, i + r // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(out[..., one], out[..., two]) * unit
    out[..., one], out[..., two] = z.real, z.imag
    return out


def _power(exponent):
    """2^exponent in 64 bits, exactly."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _exact_round(x):
    """To 4 significant bits, half to even, no finer than 2^-9."""
    exponent = (torch.frexp(x)[1] - 1).clamp(min=-6)
    step = _power(exponent - 3)
    return torch.round(x / step) * step


def _exact_scale(top):
    """The least power of two from 2^-126 up that is no less than top / 448."""
    mantissa, exponent = torch.frexp((top / 448).clamp(min=2.0 ** -126))
    return _power(torch.where(mantissa == 0.5, exponent - 1, exponent))


def _exact_write(case, k, v, scales, new_k, new_v, slots):
    """Block by block; codes as the values that they are, in 64 bits."""
    page = case["page"]
    pools = [k.double(), v.double()]
    scales = scales.double()
    for i, row in enumerate(slots.tolist()):
        t = 0
        while t < len(row) and row[t] >= 0:
            end = t
            while end < len(row) and row[end] >= 0 and row[end] // BLOCK == row[t] // BLOCK:
                end += 1
            p, first = row[t] // page, row[t] % page
            group, at = first // BLOCK, first % BLOCK
            rows = slice(group * BLOCK, (group + 1) * BLOCK)
            for which, (pool, new) in enumerate(zip(pools, (new_k, new_v))):
                x = new[i, :, t:end].double()
                top = x.abs().amax((1, 2))
                s = _exact_scale(top)
                if at:
                    old = scales[p, :, group, which].clone()
                    s = torch.maximum(s, old)
                    there = pool[p, :, rows] * (old / s)[:, None, None]
                    pool[p, :, rows] = _exact_round(there)
                pool[p, :, first:first + end - t] = _exact_round(x / s[:, None, None])
                scales[p, :, group, which] = s
            t = end
    return pools[0], pools[1], scales


def _exact_held(pool, scales, which, pages, h, n):
    """The first n rows that the pages hold for one head, in 64 bits."""
    x = pool[pages, h].double()
    x = x.view(x.shape[0], -1, BLOCK, x.shape[-1]) * scales[pages, h][:, :, which, None, None].double()
    return x.reshape(-1, x.shape[-1])[:n]


def _exact_attend(case, q, k, v, scales, tables, lengths):
    b, hq, sq, d = q.shape
    hkv, page = k.shape[1], k.shape[2]
    out = torch.zeros((b, hq, sq, d), dtype=torch.float64, device="cuda")
    if k.dtype == torch.float8_e4m3fn:
        k, v = k.view(torch.uint8), v.view(torch.uint8)
    for i, n in enumerate(lengths):
        if n == 0:
            continue
        mine = tables[i, :_cdiv(n, page)].long()
        for h in range(hkv):
            kd, vd = (_exact_held(x[mine].view(torch.float8_e4m3fn) if x.dtype == torch.uint8 else x[mine],
                                  scales[mine], which, slice(None), h, n) for which, x in enumerate((k, v)))
            for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                for r in range(sq):
                    m = n - (sq - 1 - r) if case["causal"] else n
                    if m > 0:
                        w = torch.softmax((kd[:m] * q[i, j, r].double()).sum(-1) / math.sqrt(d), 0)
                        out[i, j, r] = (w[:, None] * vd[:m]).sum(0)
    return out


def exact(case, seed):
    op = case["op"]
    if op in ("attend", "step") and case["b"] * case["hq"] * case["n"] > 6000:
        return None
    if op == "write" and sum(_cdiv(c, BLOCK) + 1 for c in _counts(case, seed)) > 10000:
        return None
    t = _inputs(case, seed)
    if op == "rotary":
        starts = _starts(case, seed)
        out = {x: _exact_turn(case, t[x], starts) for x in ("q", "new_k")}
        if case["train"]:
            out.update({x: _exact_turn(case, t[x], starts, inverse=True) for x in ("dq", "dk")})
        return out
    tables, held = _paging(case, seed), _held(case, seed)
    k, v, scales = t["k"], t["v"], t["scales"]
    if op == "attend":
        return _exact_attend(case, t["q"], k, v, scales, tables, held)
    if op == "read":
        out = [torch.zeros((case["b"], case["hkv"], case["top"], case["d"]), dtype=torch.float64, device="cuda")
               for _ in range(2)]
        for i, n in enumerate(held):
            if n == 0:
                continue
            mine = tables[i, :_cdiv(n, case["page"])].long()
            for h in range(case["hkv"]):
                for which, pool in enumerate((k, v)):
                    codes = pool.view(torch.uint8)[mine].view(torch.float8_e4m3fn)
                    out[which][i, h, :n] = _exact_held(codes, scales[mine], which, slice(None), h, n)
        return out
    slots = _slots(case, seed, tables)
    q, new_k = t.get("q"), t["new_k"]
    if op == "step":
        # What one operator hands to the next is in the 16-bit type.
        q, new_k = (_exact_turn(case, x, _starts(case, seed)).to(x.dtype) for x in (q, new_k))
    k, v, scales = _exact_write(case, k, v, scales, new_k, t["new_v"], slots)
    if op == "write":
        return {"k": k, "v": v, "scales": scales}
    o = _exact_attend(case, q, k, v, scales, tables, held)
    return {"o": o, "slots": slots, "k": k, "v": v, "scales": scales}
