"""The 8-bit paged cache's entry points on a machine without a GPU: what they refuse, and the
oracle's own arithmetic."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import kv8_oracle as ko

P = 0x1000  # a fake non-null, aligned address; never dereferenced


def pool(pkg, codes=P, scales=P, layers=2, n_pages=10, heads=8, d=64):
    return pkg.kv8_pool(codes, scales, layers, n_pages, heads, d)


def refs(pkg, p):
    return C.byref(p)


def append_args(pkg, **kw):
    a = dict(pool=pool(pkg), layer=0, T=4, qkv=P, dtype=pkg.BF16, stride=80 * 64, n_q=64, n_seqs=2, row_start=P, kv_len=P,
             pages=P, width=5, max_new=2)
    a.update(kw)
    return a


def append(pkg, **kw):
    a = append_args(pkg, **kw)
    return pkg.load().gptoss_kv8_append(None, C.byref(a["pool"]) if a["pool"] else None, a["layer"], a["T"], a["qkv"], a["dtype"],
                                        a["stride"], a["n_q"], a["n_seqs"], a["row_start"], a["kv_len"], a["pages"],
                                        a["width"], a["max_new"], 0)


def attend(pkg, **kw):
    a = append_args(pkg, scale=0.125, window=0, first=0, sinks=None, out=P, out_dtype=pkg.BF16, out_stride=64 * 64, ws=P,
                    ws_bytes=1 << 40)
    a.update(kw)
    return pkg.load().gptoss_kv8_attention(None, C.byref(a["pool"]) if a["pool"] else None, a["layer"], a["T"], a["qkv"],
                                           a["dtype"], a["stride"], a["n_q"], a["n_seqs"], a["row_start"], a["kv_len"],
                                           a["pages"], a["width"], a["max_new"], a["scale"], a["window"], a["first"],
                                           a["sinks"], a["out"], a["out_dtype"], a["out_stride"], a["ws"], a["ws_bytes"], 0)


def test_rows_calls_refuse_bad_arguments(pkg):
    B, U = pkg.ERR_BAD_ARG, pkg.ERR_UNSUPPORTED
    for call in (append, attend):
        for bad in (dict(pool=None), dict(pool=pool(pkg, codes=None)), dict(pool=pool(pkg, codes=P + 8)),
                    dict(pool=pool(pkg, scales=P + 4)), dict(pool=pool(pkg, layers=0)), dict(pool=pool(pkg, n_pages=0)),
                    dict(pool=pool(pkg, heads=0)), dict(layer=2), dict(layer=-1), dict(T=-1), dict(qkv=None),
                    dict(qkv=P + 1), dict(dtype=7), dict(stride=80 * 64 - 1), dict(n_seqs=0), dict(row_start=None),
                    dict(kv_len=None), dict(pages=None), dict(width=0), dict(max_new=0)):
            assert call(pkg, **bad) == B, (call.__name__, bad)
        for odd in (dict(pool=pool(pkg, d=96)), dict(T=(1 << 30) + 1), dict(width=1 << 25)):
            assert call(pkg, **odd) == U, (call.__name__, odd)
        assert call(pkg, T=0, qkv=None, row_start=None) == pkg.OK
    for bad in (dict(window=-1), dict(first=-1), dict(out=None), dict(out=P + 1), dict(out_dtype=3), dict(out_stride=64 * 64 - 1),
                dict(n_q=0), dict(ws=None), dict(ws=P + 8), dict(ws_bytes=0)):
        assert attend(pkg, **bad) == B, bad
    assert attend(pkg, n_q=12) == U  # query heads are not a multiple of the key/value heads
    ws = pkg.load().gptoss_kv8_attention_workspace
    assert ws(C.byref(pool(pkg)), 0, 64, 2, 1) == 0 and ws(C.byref(pool(pkg, d=32)), 4, 64, 2, 1) == 0


def test_page_calls_refuse_bad_arguments(pkg):
    lib, B, U, OK = pkg.load(), pkg.ERR_BAD_ARG, pkg.ERR_UNSUPPORTED, pkg.OK
    p = C.byref(pool(pkg))
    ws = pkg.kv8_pages_workspace(10, 4)
    assert ws > 0 and pkg.kv8_pages_workspace(0, 4) == 0
    assert lib.gptoss_kv8_release(None, -1, P, 4, P, P, 5, 10, P, 0, 0, 0) == B
    assert lib.gptoss_kv8_release(None, 1, P, 4, P, P, 5, 10, P, -1, 0, 0) == B
    assert lib.gptoss_kv8_release(None, 1, None, 4, P, P, 5, 10, P, 0, 0, 0) == B
    assert lib.gptoss_kv8_release(None, 1, P, 4, P, None, 5, 10, P, 0, 0, 0) == B
    assert lib.gptoss_kv8_release(None, 0, None, 4, None, P, 5, 10, P, 0, 0, 0) == OK
    assert lib.gptoss_kv8_reserve(None, 5, P, P, 4, P, P, 5, 10, P, P, P, ws, 0) == B  # more requests than sequences
    assert lib.gptoss_kv8_reserve(None, 2, P, P, 4, P, P, 5, 10, P, P, P, ws - 1, 0) == B
    assert lib.gptoss_kv8_reserve(None, 2, P, P, 4, P, P, 5, 10, P, P, None, ws, 0) == B
    assert lib.gptoss_kv8_reserve(None, 2, P, None, 4, P, P, 5, 10, P, P, P, ws, 0) == B
    assert lib.gptoss_kv8_reserve(None, 0, None, None, 4, P, P, 5, 10, P, None, None, 0, 0) == OK
    assert lib.gptoss_kv8_fork(None, p, 5, P, P, 4, P, P, 5, P, P, P, ws, 0) == B
    assert lib.gptoss_kv8_fork(None, p, 2, P, None, 4, P, P, 5, P, P, P, ws, 0) == B
    assert lib.gptoss_kv8_fork(None, p, 2, P, P, 4, P, P, 5, P, P, P, 0, 0) == B
    assert lib.gptoss_kv8_fork(None, C.byref(pool(pkg, d=32)), 2, P, P, 4, P, P, 5, P, P, P, ws, 0) == U
    assert lib.gptoss_kv8_compact(None, p, 4, P, 5, P, None, P, P, ws, 0) == B
    assert lib.gptoss_kv8_compact(None, p, 4, P, 5, P, P, P, P, ws - 1, 0) == B
    assert lib.gptoss_kv8_compact(None, p, 0, P, 5, P, P, P, P, ws, 0) == B
    assert lib.gptoss_kv8_copy_pages(None, p, -1, P, P, 0) == B
    assert lib.gptoss_kv8_copy_pages(None, p, 1, P, None, 0) == B
    assert lib.gptoss_kv8_copy_pages(None, p, 0, None, None, 0) == OK
    with pytest.raises(pkg.GptossError):
        pkg.kv8_fork(pool(pkg), 1, P, P, 4, P, P, 5, 9, P, P, P, ws)  # the table is of another pool


@pytest.mark.parametrize("top", [1e-45, 2.0 ** -126, 1e-38, 0.5, 126.999, 127.0, 127.0001, 128.0, 254.0, 3e38, ko.F32_MAX])
def test_oracle_scale_is_the_smallest_power_of_two(top):
    s = ko.scale_for(top)
    assert np.float32(s) == s and np.log2(s) == np.rint(np.log2(s)) and s >= 2.0 ** -126
    assert top <= 127 * s and (s == 2.0 ** -126 or top > 127 * (s / 2))


def test_oracle_growth_stays_within_one_step_of_the_final_scale():
    """The promise that goes with powers of two: however often a page's scale grew, a stored value
    is off by at most half a step of its own rounding plus less than one step of the final scale."""
    r = np.random.default_rng(3)
    codes, scales = np.zeros((1, 1, 2, 64, 64), np.int8), np.zeros((1, 1, 2), np.float32)
    rows = (r.standard_normal((64, 3 * 64)) * 1.13 ** np.arange(64)[:, None]).astype(np.float32)
    for i in range(64):
        codes, scales = ko.append(codes, scales, rows[i:i + 1], 1, [0, 1], [i + 1], np.zeros((1, 1), np.int32), 1)
    for kind in range(2):
        got = codes[0, 0, kind].astype(np.float64) * scales[0, 0, kind]
        assert np.max(np.abs(got - rows[:, 64 * (1 + kind):64 * (2 + kind)])) < 1.0 * scales[0, 0, kind]
