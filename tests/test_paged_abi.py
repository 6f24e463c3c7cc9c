"""Refusals of the paged cache's C entry points: they come before any GPU
work, with a message. No kernel is launched here."""
import ctypes

import pytest

from kotflash_amd import _hip

P = 0x10000


def _arr(*vals):
    return ctypes.cast((ctypes.c_int64 * len(vals))(*vals), _hip._I64P)


def _expect(rc, match):
    assert rc != 0 and match in _hip.lib().kf_last_error().decode()


def _reserve(**kw):
    a = dict(tables=P, lengths=P, free=P, counters=P, counts=None, count=1, slots=P, width=1, B=2, columns=4,
             stride=4, page=16, pages=8)
    a.update(kw)
    return _hip.lib().kf_page_reserve(a["tables"], a["lengths"], a["free"], a["counters"], a["counts"], a["count"],
                                      a["slots"], a["width"], a["B"], a["columns"], a["stride"], a["page"],
                                      a["pages"], None)


@pytest.mark.parametrize("kw,match", [
    (dict(tables=None), "null"), (dict(lengths=None), "null"), (dict(free=None), "null"),
    (dict(counters=None), "null"), (dict(slots=None), "slots"), (dict(width=0), "width"),
    (dict(width=2 ** 30), "width"), (dict(count=2), "do not fit"), (dict(count=-1), "do not fit"),
    (dict(B=0), "positive"), (dict(columns=0), "positive"), (dict(page=-16), "positive"), (dict(pages=0), "positive"),
    (dict(stride=3), "overlap"), (dict(page=2 ** 28), "32-bit"), (dict(B=2 ** 30), "32-bit"),
    (dict(pages=2 ** 30), "32-bit"),
])
def test_reserve(kw, match):
    _expect(_reserve(**kw), match)


@pytest.mark.parametrize("kw,match", [
    (dict(tables=None), "null"), (dict(length=-1), "negative"), (dict(B=0), "positive"), (dict(stride=1), "overlap"),
])
def test_trim(kw, match):
    a = dict(tables=P, length=0, B=2, columns=4, stride=4)
    a.update(kw)
    _expect(_hip.lib().kf_page_trim(a["tables"], P, P, P, None, a["length"], a["B"], a["columns"], a["stride"], 16, 8,
                                    None), match)


@pytest.mark.parametrize("kw,match", [
    (dict(k=None), "null"), (dict(slots=None), "null"), (dict(ks=None), "strides"), (dict(ns=None), "strides"),
    (dict(B=0), "positive"), (dict(D=0), "positive"), (dict(pages=0), "positive"), (dict(dtype=2), "dtype"),
    (dict(H=2 ** 31), "too large"), (dict(S=2 ** 20, H=2 ** 10, D=2), "too large"), (dict(B=2 ** 31), "grid"),
])
def test_append(kw, match):
    a = dict(k=P, slots=P, B=1, H=2, S=3, D=64, pages=4, ks=_arr(2048, 1024, 64), ns=_arr(384, 192, 64, 1), dtype=0)
    a.update(kw)
    _expect(_hip.lib().kf_paged_append(a["k"], P, P, P, a["slots"], a["B"], a["H"], a["S"], a["D"], a["pages"], 16,
                                       a["S"], a["ks"], a["ks"], a["ns"], a["ns"], a["dtype"], None), match)


@pytest.mark.parametrize("kw,match", [
    (dict(B=0), "positive"), (dict(Hq=3), "divisible"), (dict(D=76), "multiple of 8"), (dict(D=136), "multiple of 8"),
    (dict(dtype=7), "dtype"), (dict(q=None), "q is null"), (dict(k=P + 8), "k_pages must be 16-byte"),
    (dict(qs=_arr(512, 256, 63)), "strides"), (dict(ks=None), "strides"), (dict(tables=None), "tables"),
    (dict(lengths=None), "lengths"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
    (dict(pages=0), "num_pages"), (dict(columns=0), "columns"), (dict(page=24), "multiple of 16"),
    (dict(page=0), "multiple of 16"), (dict(stride=-1), "table stride"), (dict(columns=2 ** 27), "32-bit positions"),
    (dict(B=2 ** 20, columns=2 ** 20), "step numbers"), (dict(ws_bytes=16), "workspace"), (dict(ws=None), "workspace"),
    (dict(ws=P + 4), "16-byte aligned"), (dict(ks=_arr(2 ** 31, 1024, 64)), "page more than 4"),
    (dict(ks=_arr(2 ** 30, 1024, 2 ** 27)), "16 rows of a page"), (dict(qs=_arr(512, 2 ** 31, 64)), "2 GiB"),
    (dict(os=_arr(512, 2 ** 31, 64)), "2 GiB"),
])
def test_decode(kw, match):
    a = dict(q=P, k=P, tables=P, lengths=P, B=2, Hq=4, Hkv=2, Sq=1, D=64, pages=8, page=16, columns=4, stride=4,
             qs=_arr(256, 64, 64), ks=_arr(2048, 1024, 64), os=_arr(256, 64, 64), scale=0.1, dtype=0, ws=P,
             ws_bytes=1 << 40)
    a.update(kw)
    _expect(_hip.lib().kf_paged_decode(a["q"], a["k"], P, P, None, a["tables"], a["lengths"], a["B"], a["Hq"],
                                       a["Hkv"], a["Sq"], a["D"], a["pages"], a["page"], a["columns"], a["stride"],
                                       a["qs"], a["ks"], _arr(2048, 1024, 64), a["os"], a["scale"], 0, a["dtype"],
                                       a["ws"], a["ws_bytes"], None), match)


def test_workspace_size():
    size = _hip.lib().kf_paged_decode_workspace_bytes
    assert size(0, 4, 2, 1, 64) == 0 and size(2, 3, 2, 1, 64) == 0 and size(2, 4, 2, 1, 136) == 0
    # At least a partial of every row for each of the workers and row groups.
    for b, hq, hkv, sq, d in ((1, 1, 1, 1, 8), (64, 32, 8, 1, 128), (8, 64, 1, 3, 64)):
        rows = min(64, hq // hkv * sq)
        assert size(b, hq, hkv, sq, d) >= (256 + b * hkv) * rows * (d + 1) * 4


@pytest.mark.parametrize("kw,match", [
    (dict(nk=None), "new_k is null"), (dict(nk=P + 2), "new_k must be 16-byte"), (dict(ns=_arr(64, 64, 3)), "strides"),
    (dict(slots=None), "slots"), (dict(n=0), "1 to 16"), (dict(n=17), "1 to 16"), (dict(pages=2 ** 27), "2^31 slots"),
    (dict(page=8), "multiple of 16"), (dict(B=0), "positive"),
])
def test_append_decode(kw, match):
    a = dict(nk=P, ns=_arr(128, 64, 64), slots=P, n=1, B=2, pages=8, page=16)
    a.update(kw)
    s = _arr(2048, 1024, 64)
    _expect(_hip.lib().kf_paged_append_decode(P, P, P, a["nk"], P, a["slots"], P, None, P, P, a["B"], 4, 2, 1, a["n"],
                                              64, a["pages"], a["page"], 4, 4, 1, s, s, s, a["ns"], a["ns"], s, 0.1,
                                              0, 0, P, 1 << 40, None), match)


@pytest.mark.parametrize("kw,match", [
    (dict(B=17, n=16), "256 new tokens in all"), (dict(B=257), "256 new tokens in all"),
    (dict(Hq=2 ** 26, Hkv=2 ** 26), "grid"),
])
def test_append_decode_sizes(kw, match):
    a = dict(n=1, B=2, Hq=4, Hkv=2)
    a.update(kw)
    s = _arr(2048, 1024, 64)
    _expect(_hip.lib().kf_paged_append_decode(P, P, P, P, P, P, P, None, P, P, a["B"], a["Hq"], a["Hkv"], 1, a["n"],
                                              64, 8, 16, 4, 4, 1, s, s, s, s, s, s, 0.1, 0, 0, P, 1 << 40, None), match)


@pytest.mark.parametrize("kw,match", [
    ({}, None), (dict(B=0), "positive"), (dict(D=76), "multiple of 8"), (dict(page=24), "multiple of 16"),
    (dict(pages=0), "num_pages"), (dict(columns=0), "columns"), (dict(columns=2 ** 27), "32-bit positions"),
    (dict(B=16, columns=2 ** 25), None), (dict(B=64, columns=2 ** 25), "step numbers"), (dict(qs=None), "strides"),
    (dict(B=63, columns=2 ** 25), None), (dict(Sq=2 ** 20, Hkv=1), None), (dict(Sq=2 ** 24, Hkv=1), "grid"),
    (dict(ks=_arr(2 ** 31, 1024, 64)), "page more than 4"), (dict(qs=_arr(512, 2 ** 31, 64)), "2 GiB"),
    (dict(B=1, Hq=1, Hkv=1, Sq=2 ** 24, D=128, qs=_arr(64, 64, 64)), "2 GiB"),
])
def test_decode_check(kw, match):
    """The host's own answer, before any tensor is made."""
    a = dict(B=2, Hq=4, Hkv=2, Sq=1, D=64, pages=8, page=16, columns=4, qs=_arr(256, 64, 64), ks=_arr(2048, 1024, 64))
    a.update(kw)
    rc = _hip.lib().kf_paged_decode_check(a["B"], a["Hq"], a["Hkv"], a["Sq"], a["D"], a["pages"], a["page"],
                                          a["columns"], a["qs"], a["ks"], _arr(2048, 1024, 64))
    if match is None:
        assert rc == 0, _hip.lib().kf_last_error()
    else:
        _expect(rc, match)
