"""Refusals of the 8-bit cache's and the rotary's C entry points: they come
before any GPU work, with a message. No kernel is launched here."""
import ctypes

import pytest

from kotflash_amd import _hip

P = 0x10000


def _arr(*vals):
    return ctypes.cast((ctypes.c_int64 * len(vals))(*vals), _hip._I64P)


def _expect(rc, match):
    assert rc != 0 and match in _hip.lib().kf_last_error().decode(), _hip.lib().kf_last_error()


POOLS = dict(k=P, v=P, scales=P, H=2, D=64, pages=8, page=16, ks=_arr(2048, 1024, 64), vs=_arr(2048, 1024, 64), ss=_arr(4, 2))

POOL_REFUSALS = [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(scales=None), "null"), (dict(ks=None), "strides"),
    (dict(ss=None), "strides"), (dict(H=0), "positive"), (dict(D=0), "positive"), (dict(pages=0), "positive"),
    (dict(page=-16), "positive"), (dict(D=76), "multiple of 8 up to 128"), (dict(D=136), "multiple of 8 up to 128"),
    (dict(page=24), "page_size must be a multiple of 16"), (dict(pages=2 ** 31), "too large"),
    (dict(pages=2 ** 30, page=64), "too large"), (dict(k=P + 8), "aligned"), (dict(scales=P + 4), "aligned"),
    (dict(vs=_arr(2048, 1024, 72)), "multiples of 16"), (dict(ss=_arr(4, 1)), "pair"),
]


@pytest.mark.parametrize("kw,match", POOL_REFUSALS + [
    (dict(slots=None), "slots"), (dict(B=0), "positive"), (dict(n=0), "positive"), (dict(nk=None), "new_k is null"),
    (dict(nk=P + 2), "new_k must be 16-byte"), (dict(ns=_arr(128, 64, 3)), "strides"), (dict(dtype=2), "dtype"),
    (dict(B=2 ** 26), "grid"), (dict(n=2 ** 30), "grid"),
])
def test_append(kw, match):
    a = {**POOLS, **dict(nk=P, slots=P, B=1, n=3, ns=_arr(384, 192, 64), dtype=0), **kw}
    _expect(_hip.lib().kf_fp8_append(a["k"], a["v"], a["scales"], a["nk"], P, a["slots"], a["B"], a["H"], a["n"], a["D"],
                                     a["pages"], a["page"], a["n"], a["ks"], a["vs"], a["ss"], a["ns"], a["ns"],
                                     a["dtype"], None), match)


@pytest.mark.parametrize("kw,match", POOL_REFUSALS + [
    (dict(tables=None), "tables"), (dict(lengths=None), "lengths"), (dict(B=0), "positive"), (dict(width=0), "positive"),
    (dict(columns=0), "positive"), (dict(stride=-1), "table stride"), (dict(start=-1), "start"), (dict(out=None), "k_out is null"),
    (dict(out=P + 8), "k_out must be 16-byte"), (dict(os=_arr(384, 192, 60)), "strides"), (dict(dtype=3), "dtype"),
    (dict(columns=2 ** 27), "32-bit positions"), (dict(width=2 ** 28), "width"), (dict(start=2 ** 30), "start"),
    (dict(B=2 ** 23, width=100), "grid"),
])
def test_read(kw, match):
    a = {**POOLS, **dict(out=P, tables=P, lengths=P, start=0, B=1, width=3, columns=4, stride=4, os=_arr(384, 192, 64), dtype=0), **kw}
    _expect(_hip.lib().kf_fp8_read(a["k"], a["v"], a["scales"], a["out"], P, a["tables"], a["lengths"], None, a["start"],
                                   a["B"], a["H"], a["width"], a["D"], a["pages"], a["page"], a["columns"], a["stride"],
                                   a["ks"], a["vs"], a["ss"], a["os"], a["os"], a["dtype"], None), match)


DECODE = dict(q=P, tables=P, lengths=P, B=2, Hq=4, Hkv=2, Sq=1, columns=4, stride=4, qs=_arr(256, 64, 64), os=_arr(256, 64, 64),
              scale=0.1, dtype=0, ws=P, ws_bytes=1 << 40)


@pytest.mark.parametrize("kw,match", [
    (dict(scales=None), "scales"), (dict(scales=P + 4), "scales"), (dict(ks=None), "strides"), (dict(ss=None), "strides"),
    (dict(B=0), "positive"), (dict(Hq=3), "divisible"), (dict(D=76), "multiple of 8"), (dict(D=136), "multiple of 8"), (dict(D=72), "overlap"),
    (dict(dtype=7), "dtype"), (dict(q=None), "q is null"), (dict(k=P + 8), "k_pages must be 16-byte"),
    (dict(ks=_arr(2048, 1024, 72)), "multiples of 16"), (dict(vs=_arr(4096, 1024, 64)), "same strides"),
    (dict(ks=_arr(2048, 1024, 48), vs=_arr(2048, 1024, 48)), "overlap"),
    (dict(ks=_arr(2048, 1024, 2 ** 27), vs=_arr(2048, 1024, 2 ** 27)), "2 GiB"), (dict(ss=_arr(3, 2)), "pair"),
    (dict(ss=_arr(2 ** 28, 2)), "4 GiB"), (dict(ss=_arr(4, 2 ** 30)), "4 GiB"), (dict(ss=_arr(-4, 2)), "4 GiB"),
    (dict(tables=None), "tables"), (dict(scale=float("nan")), "finite"), (dict(pages=0), "num_pages"),
    (dict(page=24), "multiple of 16"), (dict(stride=-1), "table stride"), (dict(columns=2 ** 27), "32-bit positions"),
    (dict(ws_bytes=16), "workspace"), (dict(ws=None), "workspace"), (dict(ws=P + 4), "16-byte aligned"),
])
def test_decode(kw, match):
    a = {**POOLS, **DECODE, **kw}
    _expect(_hip.lib().kf_fp8_decode(a["q"], a["k"], a["v"], a["scales"], P, None, a["tables"], a["lengths"], a["B"],
                                     a["Hq"], a["Hkv"], a["Sq"], a["D"], a["pages"], a["page"], a["columns"], a["stride"],
                                     a["qs"], a["ks"], a["vs"], a["ss"], a["os"], a["scale"], 0, a["dtype"], a["ws"],
                                     a["ws_bytes"], None), match)


@pytest.mark.parametrize("kw,match", [({}, None), (dict(D=76), "multiple of 8"), (dict(D=56), None), (dict(D=72), "overlap"), (dict(B=0), "positive"), (dict(ss=None), "strides"),
                                      (dict(pages=2 ** 28), "4 GiB"), (dict(Sq=2 ** 24, Hkv=1), "grid")])
def test_decode_check(kw, match):
    a = {**POOLS, **DECODE, **kw}
    rc = _hip.lib().kf_fp8_decode_check(a["B"], a["Hq"], a["Hkv"], a["Sq"], a["D"], a["pages"], a["page"], a["columns"],
                                        a["qs"], a["ks"], a["vs"], a["ss"])
    if match is None:
        assert rc == 0, _hip.lib().kf_last_error()
    else:
        _expect(rc, match)


def test_workspace_size():
    size = _hip.lib().kf_fp8_decode_workspace_bytes
    assert size(0, 4, 2, 1, 64) == 0 and size(2, 3, 2, 1, 64) == 0 and size(2, 4, 2, 1, 136) == 0
    for b, hq, hkv, sq, d in ((1, 1, 1, 1, 16), (64, 32, 8, 1, 128), (8, 64, 1, 3, 64)):
        rows = min(64, hq // hkv * sq)
        assert size(b, hq, hkv, sq, d) >= (256 + b * hkv) * rows * (d + 1) * 4


@pytest.mark.parametrize("kw,match", [
    (dict(q=None), "null"), (dict(turns=None), "null"), (dict(k=None), "null"), (dict(qs=None), "strides"),
    (dict(ks=None), "strides"), (dict(ps=None, positions=P), "strides"), (dict(B=0), "positive"), (dict(S=0), "positive"),
    (dict(Hk=-1), "positive"), (dict(R=0), "even"), (dict(R=7), "even"), (dict(R=66), "even"), (dict(dtype=5), "dtype"),
    (dict(amplitude=float("inf")), "amplitude"), (dict(amplitude=float("nan")), "amplitude"),
    (dict(D=2 ** 17, R=64), "too large"), (dict(B=2 ** 16, S=2 ** 15), "too large"), (dict(Hq=2 ** 21), "too large"),
])
def test_rotary(kw, match):
    a = dict(q=P, k=P, turns=P, positions=None, B=1, Hq=2, Hk=1, S=3, D=64, R=64, qs=_arr(384, 192, 64, 1),
             ks=_arr(192, 192, 64, 1), ps=_arr(0, 0), amplitude=1.0, dtype=0)
    a.update(kw)
    _expect(_hip.lib().kf_rotary(a["q"], a["k"], P, P, a["turns"], a["positions"], 0, 0, 1, a["B"], a["Hq"], a["Hk"], a["S"],
                                 a["D"], a["R"], a["qs"], a["ks"], a["qs"], a["ks"], a["ps"], a["amplitude"], 0, 0,
                                 a["dtype"], None), match)
