"""The 8-bit paged cache on the GPU against tests/kv8_oracle.py: appending and the page calls to the
bit, attention within bounds worked out beside the oracle."""
from __future__ import annotations

import numpy as np
import pytest

import kv8_oracle as ko
from conftest import assert_bit_equal
from gpu_util import Dev, widen

pytestmark = pytest.mark.gpu
PAGE = 64


class Step:
    """A cache with junk wherever nothing may look, and one step's rows."""

    def __init__(self, pkg, seed, lens, new, n_q, heads, D, dtype, *, layers=1, layer=0, pad=0, offset=0, width=None,
                 missing=(), spare=3, lead=0, trail=0, scales=(-7, -3)):
        r = np.random.default_rng(seed)
        self.pkg, self.n_q, self.heads, self.D, self.dtype, self.layer = pkg, n_q, heads, D, dtype, layer
        n = len(lens)
        self.T = lead + sum(new) + trail
        self.row_start = (lead + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
        self.kv_len = np.asarray(lens, np.int32)
        self.width = width or max(1, max(-(-x // PAGE) for x in lens))
        held = [min(-(-x // PAGE), self.width) for x in lens]
        n_pages = sum(held) + spare
        order = r.permutation(n_pages).astype(np.int32)
        self.pages = np.full((n, self.width), -1, np.int32)
        at = 0
        for s, h in enumerate(held):
            self.pages[s, :h] = order[at:at + h]
            at += h
        self.codes = np.clip(np.rint(r.standard_normal((layers, n_pages, heads, 2, PAGE, D)) * 32), -127, 127).astype(np.int8)
        self.scales = (2.0 ** r.integers(*scales, (layers, n_pages, heads, 2))).astype(np.float32)
        self.scales[:, order[at:]] = np.nan  # pages that no sequence has
        for l in range(layers):
            if l != layer:
                self.scales[l] = np.nan
        for s, j, value in missing:
            self.scales[:, self.pages[s, j]] = np.nan
            self.pages[s, j] = value
        self.row = (n_q + 2 * heads) * D
        self.stride, self.offset = self.row + pad, offset
        self.x = widen(pkg, (r.standard_normal((self.T, self.row)) * np.exp(0.5 * r.standard_normal(self.row))).astype(np.float32), dtype)
        self.max_new = max(max(new), 1)
        self.r = r

    def put(self):
        """Uploads everything; codes and scales between guards."""
        d = self.dev = Dev(self.pkg)
        flat = np.full(self.offset + self.T * self.stride, np.nan, np.float32)
        flat[self.offset:].reshape(self.T, self.stride)[:, :self.row] = self.x
        buf = d.put(flat, self.dtype)
        self.qkv = buf.ptr + self.offset * (4 if self.dtype == self.pkg.F32 else 2)
        self.d_codes, self.d_scales = d.put_inout(self.codes), d.put_inout(self.scales)
        self.d_rows, self.d_len, self.d_pages = d.put(self.row_start), d.put(self.kv_len), d.put(self.pages)
        layers, n_pages = self.codes.shape[:2]
        self.pool = self.pkg.kv8_pool(self.d_codes, self.d_scales, layers, n_pages, self.heads, self.D)
        return self

    def append(self, **kw):
        self.pkg.kv8_append(self.pool, self.layer, self.T, self.qkv, self.dtype, self.stride, self.n_q, len(self.kv_len),
                            self.d_rows, self.d_len, self.d_pages, self.width, kw.pop("max_new", self.max_new), **kw)

    def attend(self, out, out_dtype, scale, window=0, first=0, sinks=None, ws=None, out_stride=None, **kw):
        max_new = kw.pop("max_new", self.max_new)
        n = self.pkg.kv8_attention_workspace(self.pool, self.T, self.n_q, len(self.kv_len), max_new)
        if ws is None:
            ws = self.dev.out((n,), np.uint8)  # canaries around it, 0x55 in it
        self.pkg.kv8_attention(self.pool, self.layer, self.T, self.qkv, self.dtype, self.stride, self.n_q, len(self.kv_len),
                               self.d_rows, self.d_len, self.d_pages, self.width, max_new, scale, window, first, sinks, out,
                               out_dtype, out_stride or self.n_q * self.D, ws, n, **kw)
        return ws

    def check_append(self, max_new=None):
        want_c, want_s = self.codes.copy(), self.scales.copy()
        want_c[self.layer], want_s[self.layer] = ko.append(self.codes[self.layer], self.scales[self.layer], self.x, self.n_q,
                                                           self.row_start, self.kv_len, self.pages, max_new or self.max_new)
        assert_bit_equal(self.d_scales.get(), want_s, "scales")
        assert np.array_equal(self.d_codes.get(), want_c)

    def check_attend(self, out_dtype=None, window=0, first=0, sinks=None, max_new=None, pad_out=0, scale=None, **kw):
        pkg = self.pkg
        out_dtype = self.dtype if out_dtype is None else out_dtype
        scale = 1 / np.sqrt(self.D) if scale is None else scale
        stride = self.n_q * self.D + pad_out
        out = self.dev.out((self.T, stride), out_dtype)
        d_sinks = self.dev.put(sinks) if sinks is not None else None
        ws = self.attend(out, out_dtype, scale, window, first, d_sinks, out_stride=stride, max_new=max_new or self.max_new, **kw)
        raw = out.get(as_f32=False)
        got = out.get()[:, :self.n_q * self.D].reshape(self.T, self.n_q, self.D)
        if hasattr(ws, "get"):
            ws.get()
        ref, *bounds = ko.attend(self.codes[self.layer], self.scales[self.layer], self.x, self.n_q, self.row_start,
                                 self.kv_len, self.pages, max_new or self.max_new, float(np.float32(scale)), window, first, sinks)
        skipped = np.isnan(ref).any((1, 2))
        untouched = np.frombuffer(b"\x55" * 4, raw.dtype)[0]
        assert (raw[skipped] == untouched).all(), "a row that belongs to no sequence was written"
        assert (raw[:, self.n_q * self.D:] == untouched).all(), "written past the row"
        tol = ko.tolerance(ref, *bounds, self.dtype == pkg.F32, out_dtype == pkg.F32)
        err = np.abs(got - ref)[~skipped]
        assert np.isfinite(got[~skipped]).all()
        over = err > tol[~skipped]
        assert not over.any(), f"{int(over.sum())} of {over.size} elements off; worst {np.max(err / tol[~skipped]):.3g} of the bound"


# ---- append -----------------------------------------------------------------------------

SHAPES = [(64, 8, 64), (40, 8, 64), (8, 8, 64), (3, 1, 64), (16, 1, 128), (12, 3, 128)]


@pytest.mark.parametrize("dtype_name", ["bf16", "f32"])
@pytest.mark.parametrize("lens,new", [
    ([1], [1]), ([64], [1]), ([65], [1]), ([63, 64, 65, 200], [1, 1, 1, 1]), ([70, 5], [6, 5]), ([64], [64]), ([130], [130]),
    ([200, 77, 3, 64, 129], [137, 0, 3, 64, 1]), ([300], [9]), ([128, 128], [8, 8]),
])
def test_append(gpu, dtype_name, lens, new):
    pkg = gpu
    n_q, heads, D = SHAPES[(sum(lens) + len(dtype_name)) % len(SHAPES)]
    st = Step(pkg, 11 + sum(lens), lens, new, n_q, heads, D, pkg.BF16 if dtype_name == "bf16" else pkg.F32).put()
    st.append()
    st.check_append()


@pytest.mark.parametrize("n_q,heads,D", SHAPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (3, 0), (0, 1), (1, 3)])
def test_append_strides_and_alignment(gpu, n_q, heads, D, pad, offset):
    pkg = gpu
    for dtype in (pkg.BF16, pkg.F32):
        for new in ([1, 3], [20, 70]):
            st = Step(pkg, 5, [66, 75], new, n_q, heads, D, dtype, pad=pad, offset=offset, layers=3, layer=1, lead=2, trail=3).put()
            before = pkg.load().gptoss_generic_launch_count()
            st.append()
            aligned = (pad * (2 if dtype == pkg.BF16 else 4)) % 16 == 0 and offset == 0
            assert (pkg.load().gptoss_generic_launch_count() == before) == aligned
            st.check_append()


def test_append_token_by_token_grows_the_scale(gpu):
    pkg = gpu
    st = Step(pkg, 9, [70, 129], [70, 129], 4, 2, 64, pkg.F32)
    st.x *= (1.07 ** np.arange(st.T))[:, None].astype(np.float32)
    st.x[30:40] = 0
    st.put()
    codes, scales = st.codes[0], st.scales[0]
    for i in range(129):
        new = [1 if i < n else 0 for n in (70, 129)]
        rows = np.concatenate([st.x[i:i + 1], st.x[70 + i:71 + i]])[[k for k in (0, 1) if new[k]]]
        lens = np.array([min(i + 1, 70), i + 1], np.int32)
        start = np.array([0, new[0], new[0] + new[1]], np.int32)
        keep = [st.dev.put(a) for a in (rows, start, lens)]
        pkg.kv8_append(st.pool, 0, rows.shape[0], keep[0], pkg.F32, st.row, 4, 2, keep[1], keep[2], st.d_pages, st.width, 1)
        codes, scales = ko.append(codes, scales, rows, 4, start, lens, st.pages, 1)
    assert_bit_equal(st.d_scales.get()[0], scales)
    assert np.array_equal(st.d_codes.get()[0], codes)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 64, 3]])
def test_append_special_values(gpu, new):
    pkg = gpu
    for dtype in (pkg.F32, pkg.BF16):
        st = Step(pkg, 21, [40, 64, 70], new, 2, 2, 64, dtype)
        k = st.x[:, 128:]
        k[0, :64] = 0
        k[-1, 64:128] = 0
        k[0, 130:140] = np.nan
        k[1, 200] = np.inf
        k[2, 3] = -np.inf
        k[0, 192:] = np.nan
        k[1, 64:128] *= np.float32(1e-38)
        st.x = widen(pkg, st.x, dtype)
        st.put()
        st.append()
        st.check_append()


def test_append_rows_without_a_place(gpu):
    """Positions before the start, past the table, on pages that are not there; more rows than
    max_new; row_start out of range; an empty batch of rows."""
    pkg = gpu
    st = Step(pkg, 31, [200, 300, 20, 90], [100, 150, 40, 30], 4, 2, 64, pkg.F32, width=3,
              missing=[(0, 2, -1), (1, 1, 10 ** 9), (3, 1, -7)]).put()
    st.append()
    st.check_append()
    st = Step(pkg, 32, [200, 300], [100, 150], 4, 2, 64, pkg.BF16).put()
    st.append(max_new=37)
    st.check_append(max_new=37)
    st = Step(pkg, 33, [200, 300], [10, 15], 4, 2, 64, pkg.BF16)
    st.row_start[:] = [-3, 10, 1000]
    st.put()
    st.append(max_new=25)
    st.check_append(max_new=25)
    st = Step(pkg, 34, [200, 300], [10, 15], 4, 2, 64, pkg.BF16)
    st.row_start[:] = [9, 5, 5]
    st.put()
    st.append()
    st.check_append()


# ---- attention ----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype_name", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,heads,D", SHAPES)
@pytest.mark.parametrize("window,first,sink", [(0, 0, False), (0, 0, True), (128, 4, True), (1, 0, False), (70, 65, False)])
def test_attend_tokens(gpu, dtype_name, n_q, heads, D, window, first, sink):
    """A decode step: lengths around page borders, a sequence that sits out."""
    pkg = gpu
    lens, new = [1, 63, 64, 65, 200, 129, 517], [1, 1, 1, 1, 0, 1, 1]
    st = Step(pkg, 41 + n_q, lens, new, n_q, heads, D, pkg.BF16 if dtype_name == "bf16" else pkg.F32, lead=1, trail=2).put()
    sinks = (st.r.standard_normal(n_q) * 2).astype(np.float32) if sink else None
    st.check_attend(window=window, first=first, sinks=sinks)


@pytest.mark.parametrize("dtype_name", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,heads,D", SHAPES)
@pytest.mark.parametrize("lens,new,window,first", [
    ([200, 5, 64], [5, 5, 3], 0, 0), ([321, 140, 64, 190], [17, 100, 64, 0], 0, 0), ([321, 140, 64, 190], [17, 100, 64, 9], 50, 3),
    ([150], [150], 0, 0), ([400], [33], 64, 130),
])
def test_attend_several_rows(gpu, dtype_name, n_q, heads, D, lens, new, window, first):
    pkg = gpu
    st = Step(pkg, 51 + n_q, lens, new, n_q, heads, D, pkg.BF16 if dtype_name == "bf16" else pkg.F32, layers=2, layer=1, trail=1).put()
    sinks = (st.r.standard_normal(n_q)).astype(np.float32)
    st.check_attend(window=window, first=first, sinks=sinks if window == 0 else None)


@pytest.mark.parametrize("dtype_name", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,heads,D", [(64, 8, 64), (40, 8, 64), (32, 8, 128)])
@pytest.mark.parametrize("window,first", [(0, 0), (200, 70)])
def test_attend_prompts_that_fill_the_gpu(gpu, dtype_name, n_q, heads, D, window, first):
    """Enough rows for a block per SM and more, a short prompt and a few single tokens among them; values of very
    different pages, a page that is not there."""
    pkg = gpu
    lens, new = [1500, 1, 700, 130, 90], [1500, 1, 650, 120, 0]
    st = Step(pkg, 65 + n_q, lens, new, n_q, heads, D, pkg.BF16 if dtype_name == "bf16" else pkg.F32, scales=(-16, 2),
              missing=[(0, 3, -1), (2, 0, 99999)], trail=3).put()
    st.check_attend(window=window, first=first, sinks=st.r.standard_normal(n_q).astype(np.float32))


@pytest.mark.parametrize("in_name,out_name", [("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("pad,offset,pad_out", [(0, 0, 0), (3, 0, 1), (8, 1, 8), (1, 3, 5)])
def test_attend_strides_and_types(gpu, in_name, out_name, pad, offset, pad_out):
    pkg = gpu
    types = {"bf16": pkg.BF16, "f32": pkg.F32}
    for new in ([1, 1], [7, 2], [70, 30]):
        st = Step(pkg, 61, [130, 75], new, 6, 2, 64, types[in_name], pad=pad, offset=offset).put()
        st.check_attend(types[out_name], pad_out=pad_out)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [30, 64, 20, 100]])
def test_attend_missing_pages_and_masks(gpu, new):
    """Pages that are not there are not seen; a row that sees nothing gives 0, with and without a sink
    logit; kv_len below the rows and beyond the table; more rows than max_new."""
    pkg = gpu
    st = Step(pkg, 71, [300, 200, 10, 500], new, 4, 2, 64, pkg.F32, width=5,
              missing=[(0, 0, -1), (0, 2, 1 << 30), (1, 3, -5), (1, 2, -1), (3, 4, -1), (3, 3, -1)]).put()
    sinks = np.array([0.5, -np.inf, 3.0, -40.0], np.float32)
    st.check_attend()
    st.check_attend(sinks=sinks)
    st.check_attend(window=10)
    st.check_attend(window=10, first=70, sinks=sinks)
    st.check_attend(max_new=max(1, max(new) // 3))


def test_attend_bad_row_starts(gpu):
    pkg = gpu
    for starts in ([-3, 10, 1000], [9, 5, 5], [4, 4, 25], [30, 40, 50]):
        st = Step(pkg, 73, [200, 300], [10, 15], 4, 2, 64, pkg.BF16)
        st.row_start[:] = starts
        st.put()
        st.check_attend(max_new=25)


@pytest.mark.parametrize("new", [1, 90])
def test_attend_extreme_values(gpu, new):
    """Scores far apart (one token takes everything), equal scores, values of very different pages, a zero
    page, a scale of 0, a large negative sink, huge and tiny query rows."""
    pkg = gpu
    for dtype in (pkg.F32, pkg.BF16):
        st = Step(pkg, 81, [640, 333], [new, new], 8, 2, 64, dtype, scales=(-24, 4))
        st.x[:, :64] *= 40
        st.x[:, 64:128] = 0
        st.x[:, 128:192] *= np.float32(1e-18)
        st.x[:, 192:256] *= np.float32(2e4)
        st.x = widen(pkg, st.x, dtype)
        st.scales[0, st.pages[0, 3], :, 1] = 0
        st.scales[0, st.pages[0, 4], :, 0] = 0
        st.scales[0, st.pages[0, 5], :, 1] = 2.0 ** -100
        st.scales[0, st.pages[1, 1], :, 1] = 2.0 ** 60
        st.codes[0, st.pages[1, 0]] = 0
        st.put()
        st.check_attend(scale=0.125)
        st.check_attend(scale=0.125, sinks=np.full(8, -1e30, np.float32))
        st.check_attend(scale=0.0)
        st.check_attend(scale=-0.25)


@pytest.mark.parametrize("dtype_name", ["bf16", "f32"])
def test_attend_long_context_few_rows(gpu, dtype_name):
    """One long sequence beside short ones: its cache is split over the whole GPU and joined."""
    pkg = gpu
    st = Step(pkg, 91, [9000, 40, 1, 700], [1, 3, 1, 2], 16, 2, 64, pkg.BF16 if dtype_name == "bf16" else pkg.F32).put()
    st.check_attend(sinks=np.zeros(16, np.float32))
    st.check_attend(window=5000, first=100)


@pytest.mark.parametrize("dtype_name", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,heads,D,lens,new", [(16, 2, 64, [5000, 300, 3], [20, 12, 1]), (16, 1, 128, [4099], [5]),
                                                  (64, 8, 64, [3000], [33]), (12, 3, 128, [2500, 130], [40, 100])])
def test_attend_long_context_some_rows(gpu, dtype_name, n_q, heads, D, lens, new):
    """More rows than the token kernel takes, too few for a block per SM: the context is shared out and joined; with
    parts that see nothing, a page that is not there, a row with a NaN."""
    pkg = gpu
    st = Step(pkg, 97, lens, new, n_q, heads, D, pkg.BF16 if dtype_name == "bf16" else pkg.F32, missing=[(0, 1, -1), (0, 17, -1)]).put()
    st.check_attend(sinks=st.r.standard_normal(n_q).astype(np.float32))
    st.check_attend(window=1000, first=70)
    st.check_attend(window=64, first=0)


def test_attend_masked_query_does_not_leak(gpu):
    """NaN and infinities in one row's query show in that row alone."""
    pkg = gpu
    for new in (2, 80):
        st = Step(pkg, 95, [200, 200], [new, new], 4, 2, 64, pkg.BF16)
        st.x[1, 5], st.x[new, 64] = np.nan, np.inf
        st.put()
        out = st.dev.out((st.T, 256), pkg.BF16)
        st.attend(out, pkg.BF16, 0.125)
        got = out.get().reshape(st.T, 4, 64)
        ref, *bounds = ko.attend(st.codes[0], st.scales[0], np.nan_to_num(st.x, nan=0, posinf=0), 4, st.row_start, st.kv_len,
                                 st.pages, st.max_new, 0.125, 0, 0, None)
        ok = np.ones((st.T, 4), bool)
        ok[1, 0] = ok[new, 1] = False
        assert (np.abs(got - ref) <= ko.tolerance(ref, *bounds, False, False))[ok].all()
        assert np.isnan(got[1, 0]).all()


@pytest.mark.parametrize("dtype_name", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,heads,D", [(80, 1, 64), (130, 1, 128), (33, 1, 64), (400, 2, 64)])
def test_attend_wide_groups(gpu, dtype_name, n_q, heads, D):
    """Many query heads to one key/value head: a single token is then many rows."""
    pkg = gpu
    st = Step(pkg, 121 + n_q, [300, 64, 2000, 7], [1, 1, 1, 2], n_q, heads, D, pkg.BF16 if dtype_name == "bf16" else pkg.F32, trail=1).put()
    st.check_attend(sinks=st.r.standard_normal(n_q).astype(np.float32))
    st.check_attend(window=100, first=5)


@pytest.mark.parametrize("n,most_new,n_q,heads", [(3000, 1, 2, 1), (1100, 3, 2, 1), (130, 10, 8, 1)])
def test_many_sequences(gpu, n, most_new, n_q, heads):
    """More sequences than a block has threads or a warp lanes: lengths from 0 to three pages and one long one, in a wide
    table; row counts from 0 on (10 rows of 8 heads: the tile kernel's, 8 and fewer the token kernels')."""
    pkg = gpu
    r = np.random.default_rng(n)
    lens = r.integers(0, 190, n)
    lens[n // 2] = 1200
    new = np.minimum(r.integers(0, most_new + 1, n), lens)
    st = Step(pkg, n, [int(x) for x in lens], [int(x) for x in new], n_q, heads, 64, pkg.BF16, width=20).put()
    st.append()
    st.check_append()
    st.codes[0], st.scales[0] = ko.append(st.codes[0], st.scales[0], st.x, n_q, st.row_start, st.kv_len, st.pages, st.max_new)
    st.check_attend()
    st.check_attend(window=40, first=3)


@pytest.mark.parametrize("new", [1, 200])
def test_offsets_past_32_bits(gpu, new):
    """A pool of 4.6 GB, pages at both ends of it, the second of two layers."""
    pkg = gpu
    n_pages, heads, D, n_q, length = 35001, 8, 64, 16, 200
    page_bytes = heads * 2 * PAGE * D
    d = Dev(pkg)
    codes, scales = pkg.DeviceBuffer(2 * n_pages * page_bytes), pkg.DeviceBuffer.filled(2 * n_pages * heads * 8, 0xff)
    pool = pkg.kv8_pool(codes, scales, 2, n_pages, heads, D)
    used = np.array([35000, 3, 17500, 34999], np.int32)
    r = np.random.default_rng(5)
    x = widen(pkg, r.standard_normal((length, (n_q + 2 * heads) * D)).astype(np.float32), pkg.BF16)
    small = np.arange(4, dtype=np.int32)[None]
    want_c, want_s = ko.append(np.zeros((4, heads, 2, PAGE, D), np.int8), np.full((4, heads, 2), np.nan, np.float32), x, n_q,
                               [0, length], [length], small, length)
    row = x.shape[1]
    args = (1, length, d.put(x, pkg.BF16), pkg.BF16, row, n_q, 1, d.put(np.array([0, length], np.int32)),
            d.put(np.array([length], np.int32)), d.put(used[None]), 4)
    pkg.kv8_append(pool, *args, length)
    pkg.kv8_copy_pages(pool, 1, d.put(used[:1]), d.put(np.array([34000], np.int32)))
    for i, page in list(enumerate(used)) + [(0, 34000)]:
        at = (n_pages + int(page))
        got = codes.numpy(np.int8, (heads, 2, PAGE, D), at * page_bytes)
        full = min(length - i * PAGE, PAGE)
        assert np.array_equal(got[:, :, :full], want_c[i][:, :, :full])
        assert_bit_equal(scales.numpy(np.float32, (heads, 2), at * heads * 8), want_s[i])
    rows = x[length - new:]
    n = pkg.kv8_attention_workspace(pool, new, n_q, 1, new)
    out = d.out((new, n_q * D), pkg.BF16)
    pkg.kv8_attention(pool, 1, new, d.put(rows, pkg.BF16), pkg.BF16, row, n_q, 1, d.put(np.array([0, new], np.int32)), *args[8:],
                      new, 0.125, 0, 0, None, out, pkg.BF16, n_q * D, d.out((n,), np.uint8), n)
    ref, *bounds = ko.attend(want_c, want_s, rows, n_q, [0, new], [length], small, new, 0.125, 0, 0, None)
    assert (np.abs(out.get().reshape(new, n_q, D) - ref) <= ko.tolerance(ref, *bounds, False, False)).all()
    codes.free()


def test_two_streams_at_once(gpu):
    """Calls that overlap in time, each with its own workspace and output."""
    pkg = gpu
    sts = [Step(pkg, 111 + i, [4000, 900, 70], new, 16, 2, 64, pkg.BF16).put() for i, new in enumerate(([1, 1, 1], [1, 90, 30]))]
    streams = [pkg.Stream() for _ in sts]
    outs = [[st.dev.out((st.T, 16 * 64), pkg.BF16) for _ in range(6)] for st in sts]
    wss = [st.attend(o[0], pkg.BF16, 0.125) for st, o in zip(sts, outs)]
    pkg.synchronize()
    for k in range(1, 6):
        for st, o, ws, stream in zip(sts, outs, wss, streams):
            st.attend(o[k], pkg.BF16, 0.125, ws=ws, stream=stream.h)
    pkg.synchronize()
    for o in outs:
        for k in range(1, 6):
            assert np.array_equal(o[0].get(as_f32=False), o[k].get(as_f32=False))
    for stream in streams:
        stream.close()


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 2, 1], [70, 1, 200]])
def test_attend_repeats_to_the_bit_and_replays(gpu, new):
    """Twice the same bits; on a stream of its own; captured and replayed with other lengths and rows;
    with programmatic launch."""
    pkg = gpu
    st = Step(pkg, 101, [3000, 65, 400], new, 16, 2, 64, pkg.BF16).put()
    outs = [st.dev.out((st.T, 16 * 64), pkg.BF16) for _ in range(4)]
    st.attend(outs[0], pkg.BF16, 0.125)
    ws = st.attend(outs[1], pkg.BF16, 0.125, flags=pkg.PDL)
    first = outs[0].get(as_f32=False)
    assert np.array_equal(first, outs[1].get(as_f32=False))
    stream = pkg.Stream()
    g = pkg.Graph(stream.h)
    with g:
        st.append(stream=stream.h)
        st.attend(outs[2], pkg.BF16, 0.125, ws=ws, stream=stream.h)
    g.launch()
    stream.synchronize()
    lens = np.array([2900, 70, 401], np.int32)
    pkg.check(pkg.load().gptoss_upload(st.d_len.ptr, lens.ctypes.data, lens.nbytes, None))
    pkg.synchronize()
    for _ in range(2):
        g.launch()
    stream.synchronize()
    got = outs[2].get().reshape(st.T, 16, 64)
    c, s = ko.append(st.codes[0], st.scales[0], st.x, 16, st.row_start, st.kv_len, st.pages, st.max_new)
    c, s = ko.append(c, s, st.x, 16, st.row_start, lens, st.pages, st.max_new)
    c, s = ko.append(c, s, st.x, 16, st.row_start, lens, st.pages, st.max_new)
    ref, *bounds = ko.attend(c, s, st.x, 16, st.row_start, lens, st.pages, st.max_new, 0.125, 0, 0, None)
    assert (np.abs(got - ref) <= ko.tolerance(ref, *bounds, False, False)).all()
    g.close()
    stream.close()


# ---- pages --------------------------------------------------------------------------------


class Table:
    def __init__(self, pkg, seed, lens, width, n_pages, heads=2, D=64, layers=2, share=True):
        r = self.r = np.random.default_rng(seed)
        self.pkg = pkg
        self.kv_len = np.asarray(lens, np.int32)
        self.pages = np.full((len(lens), width), -1, np.int32)
        order = list(r.permutation(n_pages))
        for s, x in enumerate(lens):
            n = -(-x // PAGE)
            self.pages[s, :n] = [order.pop() for _ in range(n)]
            if share and s and x >= PAGE and lens[s - 1] >= PAGE:  # a common first page
                order.append(self.pages[s, 0])
                self.pages[s, 0] = self.pages[s - 1, 0]
        self.refs = np.bincount(self.pages[self.pages >= 0], minlength=n_pages).astype(np.int32)
        self.codes = r.integers(-127, 128, (layers, n_pages, heads, 2, PAGE, D)).astype(np.int8)
        self.scales = r.standard_normal((layers, n_pages, heads, 2)).astype(np.float32)
        self.put()

    def put(self):
        d = self.dev = Dev(self.pkg)
        self.model = ko.Tables(self.kv_len, self.pages, self.refs)
        self.d_len, self.d_pages, self.d_refs = (d.put_inout(a) for a in (self.kv_len, self.pages, self.refs))
        self.d_codes, self.d_scales = d.put_inout(self.codes), d.put_inout(self.scales)
        L, n, h, _, _, D = self.codes.shape
        self.pool = self.pkg.kv8_pool(self.d_codes, self.d_scales, L, n, h, D)
        nbytes = self.pkg.kv8_pages_workspace(n, len(self.kv_len))
        self.ws = (d.out((nbytes,), np.uint8), nbytes)
        self.table = (len(self.kv_len), self.d_len, self.d_pages, self.pages.shape[1], n, self.d_refs)

    def ints(self, x):
        return self.dev.put(np.asarray(x, np.int32))

    def release(self, seqs, window=0, first=0):
        self.pkg.kv8_release(len(seqs), self.ints(seqs), *self.table, window, first)
        self.model.release(seqs, window, first)

    def reserve(self, seqs, new_len):
        served = self.dev.out((len(seqs),), np.int32)
        self.pkg.kv8_reserve(len(seqs), self.ints(seqs), self.ints(new_len), *self.table, served, *self.ws)
        assert served.get().tolist() == self.model.reserve(seqs, new_len)

    def fork(self, parents, children):
        served = self.dev.out((len(parents),), np.int32)
        self.pkg.kv8_fork(self.pool, len(parents), self.ints(parents), self.ints(children), *self.table, served, *self.ws)
        want, copies = self.model.fork(parents, children)
        assert served.get().tolist() == want
        self.moved(copies)

    def compact(self):
        remap, n_live = self.dev.out((len(self.refs),), np.int32), self.dev.out((1,), np.int32)
        self.pkg.kv8_compact(self.pool, *self.table, remap, n_live, *self.ws)
        want, n, moves = self.model.compact()
        assert np.array_equal(remap.get(), want) and n_live.get()[0] == n
        self.moved(moves)

    def moved(self, pairs):
        for a, b in pairs:
            self.codes[:, b], self.scales[:, b] = self.codes[:, a], self.scales[:, a]

    def check(self):
        assert np.array_equal(self.d_pages.get(), self.model.pages)
        assert np.array_equal(self.d_refs.get(), self.model.refs)
        assert np.array_equal(self.d_len.get(), self.model.kv_len)
        assert np.array_equal(self.d_codes.get(), self.codes)
        assert_bit_equal(self.d_scales.get(), self.scales)
        self.ws[0].get()


@pytest.mark.parametrize("heads,D", [(2, 64), (8, 64), (1, 128), (3, 128)])
def test_pages_a_life(gpu, heads, D):
    """The calls one after the other, as an engine makes them."""
    t = Table(gpu, 7 + heads, [130, 64, 200, 0, 1, 63, 0, 257, 128, 0], 6, 40, heads, D)
    t.release([1, 5])
    t.check()
    t.fork([2, 0, 2, 8], [3, 6, 9, 1])
    t.check()
    t.reserve([0, 2, 3, 4, 7, 8], [193, 200, 260, 64, 384, 128])
    t.check()
    t.compact()
    t.check()
    t.release([7], 70, 5)
    t.check()
    t.release(list(range(10)))
    t.check()
    assert (t.model.refs == 0).all()
    t.compact()
    t.check()


def test_pages_awkward_lists(gpu):
    """The same index twice, indexes outside the table, children that are parents or not empty, lengths
    that the table does not hold, too few free pages, empty lists."""
    t = Table(gpu, 3, [130, 64, 200, 0, 1, 0, 0, 0], 4, 13)
    t.release([])
    t.reserve([], [])
    t.fork([], [])
    t.release([4, 4, -1, 99, 4])
    t.check()
    t.fork([0, 0, 2, 0, 99, 0, 1], [3, 3, 4, 0, 5, -4, 5])
    t.check()
    t.reserve([0, 0, 5, 77, 6, 2], [256, 256, 257, 10, 65, 200])
    t.check()
    t.reserve([7, 6, 3, 0], [256, 100, 192, 0])  # more than there is: later, smaller ones may still be served
    t.check()
    t.compact()
    t.check()
    t.fork([0, 2, 0, 0], [7, 7, 4, 6])
    t.check()


@pytest.mark.parametrize("n_pages", [1, 2, 31, 1024, 8192, 8193, 20000])
def test_pages_pool_sizes(gpu, n_pages):
    r = np.random.default_rng(n_pages)
    n = min(300, max(1, n_pages // 40))
    t = Table(gpu, n_pages, [int(x) for x in r.integers(0, 64 * max(1, min(30, n_pages // n - 1)), n)], 64, n_pages, 1, 64, 1, share=False)
    t.check()
    t.release(sorted(set(r.integers(0, n, n // 3).tolist())))
    t.compact()
    t.check()
    grow = sorted(set(r.integers(0, n, n // 2).tolist()))
    t.reserve(grow, [int(t.model.kv_len[s]) + int(x) for s, x in zip(grow, r.integers(0, 1500, len(grow)))])
    t.check()
    t.compact()
    t.check()


@pytest.mark.parametrize("window,first", [(1, 0), (64, 0), (65, 64), (128, 4), (100, 65), (1000, 0), (1 << 30, 1)])
def test_release_behind_a_window_keeps_what_is_seen(gpu, window, first):
    """What is let go of is what no later row sees: attention gives the same before and after."""
    pkg = gpu
    t = Table(pkg, 5, [0, 64, 65, 300, 383, 256], 6, 40)
    t.release([0, 1, 2, 3, 4, 5], window, first)
    t.check()
    for s in range(6):
        for p in range(int(t.model.kv_len[s]), int(t.model.kv_len[s]) + 3):
            seen = {x // PAGE for x in range(int(t.kv_len[s])) if x > p - window or x < first}
            assert all(t.model.pages[s, j] == t.pages[s, j] for j in seen)


def test_copy_pages(gpu):
    t = Table(gpu, 13, [200], 4, 12, heads=3, layers=3)
    src, dst = [3, 5, -1, 4, 12, 1], [7, 8, 2, 99, 6, 1]
    gpu.kv8_copy_pages(t.pool, len(src), t.ints(src), t.ints(dst))
    t.moved([(3, 7), (5, 8)])
    t.check()


# ---- together -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype_name", ["bf16", "f32"])
def test_an_engine_with_the_cache(gpu, dtype_name):
    """Rotation, append and attention over a windowed and a full layer, with sequences that start,
    fork, end, and are compacted in between: every step against the oracle."""
    pkg = gpu
    dtype = pkg.BF16 if dtype_name == "bf16" else pkg.F32
    n_q, heads, D, width, n_pages, layers = 16, 2, 64, 6, 26, 2
    r = np.random.default_rng(17)
    t = Table(pkg, 1, [0] * 6, width, n_pages, heads, D, layers)
    cos, sin = pkg.build_rope_tables(512, D)
    d = t.dev
    d_cos, d_sin = d.put(cos), d.put(sin)
    sinks = [r.standard_normal(n_q).astype(np.float32) for _ in range(layers)]
    d_sinks = [d.put(s) for s in sinks]

    def step(rows_of):
        """rows_of: new rows per sequence."""
        seqs = [s for s in range(6) if rows_of[s]]
        after = t.model.kv_len + np.asarray(rows_of, np.int32)
        t.reserve(seqs, [int(after[s]) for s in seqs])
        t.check()
        T, start = sum(rows_of), np.concatenate([[0], np.cumsum(rows_of)]).astype(np.int32)
        pos = np.concatenate([np.arange(t.model.kv_len[s], after[s]) for s in range(6)]).astype(np.int32)
        t.model.kv_len = after
        pkg.check(pkg.load().gptoss_upload(t.d_len.ptr, after.ctypes.data, after.nbytes, None))
        row, d_start, d_pos = (n_q + 2 * heads) * D, d.put(start), d.put(pos)
        for layer, window in enumerate((128, 0)):
            x = r.standard_normal((T, row)).astype(np.float32)
            qkv = d.out((T, row), dtype)
            pkg.qkv_bias_rope(T, d.put(x, dtype), dtype, row, None, d_pos, 0, d_cos, d_sin, 512, n_q, heads, D, qkv, dtype, row)
            rotated = qkv.get()
            batch = (6, d_start, t.d_len, t.d_pages, width, max(rows_of))
            pkg.kv8_append(t.pool, layer, T, qkv, dtype, row, n_q, *batch)
            t.codes[layer], t.scales[layer] = ko.append(t.codes[layer], t.scales[layer], rotated, n_q, start, after, t.model.pages, T)
            nbytes = pkg.kv8_attention_workspace(t.pool, T, n_q, 6, max(rows_of))
            out = d.out((T, n_q * D), dtype)
            pkg.kv8_attention(t.pool, layer, T, qkv, dtype, row, n_q, *batch, 0.125, window, 4 if window else 0, d_sinks[layer], out,
                              dtype, n_q * D, d.out((nbytes,), np.uint8), nbytes)
            ref, *bounds = ko.attend(t.codes[layer], t.scales[layer], rotated, n_q, start, after, t.model.pages, T, 0.125, window,
                                     4 if window else 0, sinks[layer])
            tol = ko.tolerance(ref, *bounds, dtype == pkg.F32, dtype == pkg.F32)
            assert (np.abs(out.get().reshape(T, n_q, D) - ref) <= tol).all()
        t.check()

    step([70, 130, 0, 9, 0, 0])
    step([1, 1, 0, 1, 0, 0])
    t.fork([1, 1, 0], [2, 4, 5])
    step([1, 1, 1, 1, 1, 1])
    t.release([0, 3])
    t.compact()
    step([64, 1, 1, 0, 3, 1])
    step([1, 1, 1, 200, 1, 1])
    assert pkg.load().gptoss_wait_giveups() == 0
