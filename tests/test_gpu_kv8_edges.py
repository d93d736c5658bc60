"""The 8-bit paged cache where its definition is easy to lose: values of very different size, sink
logits and queries that are not numbers, scales at the ends of fp32, tables with holes.  Every form of
the attention (rows per sequence, type, how the work is shared out) takes the same cases."""
from __future__ import annotations

import numpy as np
import pytest

import kv8_oracle as ko
from gpu_util import widen
from test_gpu_kv8 import PAGE, Step, Table

pytestmark = pytest.mark.gpu

# name: lengths, new rows, query heads, key/value heads, head_dim, types
FORMS = {
    "tokens": ([333, 64, 700], [1, 1, 1], 8, 2, 64, ("bf16", "f32")),
    "tokens of wide heads": ([333, 700], [1, 1], 16, 2, 128, ("bf16", "f32")),
    "pieces of a long one": ([9000, 130], [1, 1], 8, 1, 64, ("bf16", "f32")),
    "16 rows": ([333, 700], [4, 2], 8, 2, 64, ("bf16", "f32")),
    "some rows": ([333, 640, 90], [13, 7, 1], 8, 2, 64, ("bf16", "f32")),
    "two tiles": ([300, 333], [300, 90], 8, 2, 64, ("bf16", "f32")),
    "two tiles of wide heads": ([300, 333], [300, 90], 8, 2, 128, ("bf16", "f32")),
    "columns shared out": ([3000, 200], [40, 30], 16, 2, 64, ("bf16", "f32")),
    "four tiles": ([700, 500, 5], [700, 430, 1], 64, 8, 64, ("bf16",)),
}
every_form = pytest.mark.parametrize("form,dtype_name", [(f, t) for f, v in FORMS.items() for t in v[5]])


def step_of(pkg, form, dtype_name, seed, **kw):
    lens, new, n_q, heads, D, _ = FORMS[form]
    return Step(pkg, seed, lens, new, n_q, heads, D, pkg.BF16 if dtype_name == "bf16" else pkg.F32, trail=2, **kw)


def run(st, out_dtype, scale=0.125, window=0, first=0, sinks=None):
    pkg = st.pkg
    out = st.dev.out((st.T, st.n_q * st.D), out_dtype)
    ws = st.attend(out, out_dtype, scale, window, first, st.dev.put(sinks) if sinks is not None else None)
    got = out.get().reshape(st.T, st.n_q, st.D)
    ws.get()
    assert pkg.load().gptoss_wait_giveups() == 0
    return got


def want(st, scale=0.125, window=0, first=0, sinks=None):
    """The definition in 64 bits, and per (row, head) what errors scale with: sum p |v|, the largest
    scale * sum |q k|, the tokens seen; and what fp16 weights may lose.  A row's weights are fp16 numbers of which
    the largest is at least 2^7, so that each is rounded by at most 2^-25, or 2^-32 of the largest, and by
    no more than itself."""
    codes, scales = st.codes[st.layer].astype(np.float64), st.scales[st.layer].astype(np.float64)
    T, n_q, D, G = st.T, st.n_q, st.D, st.n_q // st.heads
    x = st.x.reshape(T, -1, D)[:, :n_q].astype(np.float64)
    out, weight, grain = np.full((T, n_q, D), np.nan), np.zeros((T, n_q, D)), np.zeros((T, n_q, D))
    reach, seen = np.zeros((T, n_q, 1)), np.zeros((T, n_q, 1))
    for s, r0, q, pos in ko.spans(st.row_start, st.kv_len, T, st.max_new):
        t = np.array([i for i in range(max(pos + q, 0)) if ko.page_of(st.pages, s, i, codes.shape[0]) >= 0], np.int64)
        if not q:
            continue
        pg, slot, p = st.pages[s, t // PAGE] if len(t) else t, t % PAGE, pos + np.arange(q)[:, None]
        ok = t[None] <= p
        if window > 0:
            ok &= (t[None] > p - window) | (t[None] < first)
        any_ = ok.any(1, keepdims=True)
        for h in range(n_q):
            g, r = h // G, slice(r0, r0 + q)
            k, v = (codes[pg, g, i, slot] * scales[pg, g, i][:, None] for i in (0, 1))
            z = np.where(ok, scale * (x[r, h] @ k.T), -np.inf)
            sink = -np.inf if sinks is None else float(sinks[h])
            top = np.maximum(z.max(1, initial=-np.inf, keepdims=True), sink)
            top = np.where(np.isfinite(top), top, 0.0)
            w = np.exp(z - top)
            w = w / np.where(any_, w.sum(1, keepdims=True) + np.exp(sink - top), 1.0)
            out[r, h], weight[r, h] = w @ v, w @ np.abs(v)
            grain[r, h] = np.minimum(w, w.max(1, initial=0, keepdims=True) * 2.0 ** -32) @ np.abs(v)
            reach[r, h] = np.where(ok, np.abs(x[r, h]) @ np.abs(k.T), 0).max(1, initial=0, keepdims=True) * abs(scale)
            seen[r, h] = ok.sum(1, keepdims=True)
    return out, weight, reach, seen, grain


def check(st, got, ref, weight, reach, seen, grain, out_dtype, rows=None):
    """ko.tolerance's shares, element by element, with `grain` for its term of the largest value."""
    pkg = st.pkg
    tol = ko.tolerance(ref, weight, reach, seen, np.zeros_like(seen), st.dtype == pkg.F32, out_dtype == pkg.F32) + grain
    there = ~np.isnan(ref).any((1, 2))
    if rows is not None:
        there &= rows
    err, tol = np.abs(got.astype(np.float64) - ref)[there], tol[there]
    assert np.isfinite(got[there]).all(), "not finite"
    assert (err <= tol).all(), f"{int((err > tol).sum())} of {err.size} off; worst {np.max(err / tol):.3g} of the bound"


# ---- values of very different size ---------------------------------------------------------


@every_form
def test_values_of_pages_far_apart(gpu, form, dtype_name):
    """Value scales from 2^-60 to 2^60, pages of zeros among them, scores that differ by some tens: a small
    page counts where the large ones weigh nothing, or are not seen."""
    st = step_of(gpu, form, dtype_name, 201)
    st.x[:, :st.n_q * st.D] *= 4
    st.x = widen(gpu, st.x, st.dtype)
    st.scales[..., 1] = 2.0 ** st.r.integers(-60, 61, st.scales.shape[:-1])
    st.scales[0, st.pages[0, 1], 0, 1] = 0
    st.put()
    sinks = st.r.standard_normal(st.n_q).astype(np.float32)
    for kw in (dict(), dict(window=100, first=3, sinks=sinks), dict(window=64, scale=-0.125)):
        check(st, run(st, gpu.F32, **kw), *want(st, **kw), gpu.F32)


@every_form
@pytest.mark.parametrize("window", [0, 70])
def test_an_infinite_value_shows_only_where_it_is_seen(gpu, form, dtype_name, window):
    """One value as append stores an infinity (64 x 2^122, all others of its page 0), among ordinary ones:
    rows before it, and rows whose window has passed it, do not know of it."""
    st = step_of(gpu, form, dtype_name, 211)
    for s in range(len(st.kv_len)):
        n = int(st.kv_len[s])
        t = max(n - 40 if n - 40 < n - st.max_new // 2 else n - st.max_new // 2, 0) if window == 0 else max(n - 85, 0)
        page = st.pages[s, t // PAGE]
        st.scales[0, page, :, 1], st.codes[0, page, :, 1] = 2.0 ** 122, 0
        st.codes[0, page, :, 1, t % PAGE, 3] = 64
    st.put()
    ref = want(st, window=window)
    check(st, run(st, gpu.F32, window=window), *ref, gpu.F32)
    out = run(st, gpu.BF16, window=window)
    sane = (np.abs(ref[0]) < 1e30).all((1, 2)) & ~np.isnan(ref[0]).any((1, 2))
    if st.max_new > 60 or window:
        assert sane.any()
    check(st, out, *ref, gpu.BF16, sane)


@every_form
def test_a_huge_value_that_weighs_nothing(gpu, form, dtype_name):
    """Every row sees a token whose value is 2^60 times the others' and whose weight is some 2^-70 or less."""
    st = step_of(gpu, form, dtype_name, 221)
    n = st.n_q * st.D
    st.x[:, :n] = np.abs(st.x[:, :n])
    st.x = widen(gpu, st.x, st.dtype)
    for s in range(len(st.kv_len)):
        page = st.pages[s, 0]
        st.codes[0, page, :, 0, 0], st.scales[0, page, :, 0] = -127, 2.0 ** -3
        st.codes[0, page, :, 0, 1:] //= 4
        st.scales[0, page, :, 1] = 2.0 ** 57
        st.codes[0, page, :, 1, 1:] = 0
    st.put()
    check(st, run(st, gpu.F32), *want(st), gpu.F32)


# ---- what is not a number -----------------------------------------------------------------


@every_form
def test_a_sink_that_is_not_a_number_shows(gpu, form, dtype_name):
    """In its own head, in every row that sees something; a row that sees nothing stays 0."""
    st = step_of(gpu, form, dtype_name, 231)
    st.pages[0, :] = -1
    st.put()
    sinks = st.r.standard_normal(st.n_q).astype(np.float32)
    sinks[0], sinks[-1] = np.inf, np.nan
    got = run(st, gpu.F32, sinks=sinks)
    one = slice(st.row_start[0], st.row_start[1])
    rest = slice(st.row_start[1], st.row_start[-1])
    assert (got[one] == 0).all()
    assert np.isnan(got[rest, -1]).all() and (got[rest, 0] == 0).all()
    with np.errstate(invalid="ignore"):
        ref = want(st, sinks=np.where(np.isfinite(sinks), sinks, 0).astype(np.float32))
    for h in (slice(1, st.n_q - 1),):
        check(st, got[:, h], *(a[:, h] for a in ref), gpu.F32)


@every_form
def test_queries_that_are_not_numbers_show_in_their_own_rows(gpu, form, dtype_name):
    """NaN and infinities in single query heads give NaN there and show nowhere else, also where the row's
    context is cut and joined; a row that sees nothing gives 0 all the same."""
    st = step_of(gpu, form, dtype_name, 241)
    clean = st.x.copy()
    last, D = int(st.row_start[-1]) - 1, st.D
    bad = {(0, 0): np.nan, (last, 1): np.inf, (last // 2, st.n_q - 1): -np.inf}
    for (r, h), value in bad.items():
        st.x[r, h * D + 5] = value
        clean[r, h * D + 5] = 0
    st.put()
    got = run(st, gpu.F32)
    st.x = clean
    ref = want(st)
    for r, h in bad:
        assert np.isnan(got[r, h]).all(), (r, h)
        got[r, h] = ref[0][r, h]
    check(st, got, *ref, gpu.F32)
    st = step_of(gpu, form, dtype_name, 242)
    st.pages[:] = -1
    st.x[:, 7] = np.nan
    st.put()
    got = run(st, gpu.F32, sinks=np.zeros(st.n_q, np.float32))
    assert (got[:st.row_start[-1]] == 0).all()


@every_form
def test_an_infinite_key_that_is_not_seen(gpu, form, dtype_name):
    """A page whose key scale is 2^122 for the sake of a token behind the rows (guessed and given up): the
    others' codes in it are 0, and large queries times them are still 0."""
    st = step_of(gpu, form, dtype_name, 251)
    n = st.n_q * st.D
    st.x[:, :n] *= np.float32(2.0 ** 24)
    st.x = widen(gpu, st.x, st.dtype)
    st.kv_len[:] = np.where(st.kv_len % PAGE == 0, st.kv_len - 1, st.kv_len)
    for s in range(len(st.kv_len)):
        last = int(st.kv_len[s])
        page = st.pages[s, last // PAGE]
        st.pages[s, :last // PAGE] = -1
        st.scales[0, page, :, 0], st.codes[0, page, :, 0] = 2.0 ** 122, 0
        st.codes[0, page, :, 0, last % PAGE:, 2] = 64
    st.put()
    check(st, run(st, gpu.F32), *want(st), gpu.F32)


# ---- arguments ---------------------------------------------------------------------------------


def test_very_many_query_heads(gpu):
    """More query heads than a grid's second dimension, all on one key/value head."""
    pkg = gpu
    n_q, D, length = 262144, 64, 100
    st = Step(pkg, 261, [length], [1], n_q, 1, D, pkg.BF16).put()
    got = run(st, pkg.BF16)[0]
    k, v = (st.codes[0, st.pages[0, np.arange(length) // PAGE], 0, i, np.arange(length) % PAGE].astype(np.float64)
            * st.scales[0, st.pages[0, np.arange(length) // PAGE], 0, i][:, None] for i in (0, 1))
    x = st.x[0, :n_q * D].reshape(n_q, D).astype(np.float64)
    z = 0.125 * x @ k.T
    w = np.exp(z - z.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    reach = 0.125 * (np.abs(x) @ np.abs(k.T)).max(1, keepdims=True)
    tol = ko.tolerance(w @ v, w @ np.abs(v), reach, float(length), np.abs(v).max(), False, False)
    assert (np.abs(got - w @ v) <= tol).all()


def test_workspace_of_calls_that_are_refused(gpu):
    pkg = gpu
    pool = pkg.kv8_pool(0x1000, 0x1000, 1, 10, 8, 64)
    ws = pkg.kv8_attention_workspace
    assert ws(pool, 1 << 30, 64, 2, 1) > 0
    assert ws(pool, (1 << 30) + 1, 64, 2, 1) == 0 and ws(pool, 4, 64, (1 << 28) + 1, 1) == 0 and ws(pool, 4, 12, 2, 1) == 0


# ---- tables with holes ----------------------------------------------------------------------------


def test_reserve_refuses_a_sequence_whose_begun_page_is_gone(gpu):
    """Its next token has no place, and a free page in place of the lost one would show what another
    sequence left there.  Nobody else is held up; who asks for no token is served."""
    t = Table(gpu, 41, [70, 130, 64, 10, 64], 6, 20, share=False)
    t.pages[0, 1], t.pages[1, 2], t.pages[3, 0] = -1, -5, 20
    t.refs = np.bincount(t.pages[(t.pages >= 0) & (t.pages < 20)], minlength=20).astype(np.int32)
    t.put()
    free = np.flatnonzero(t.refs == 0)
    served = t.dev.out((5,), np.int32)
    gpu.kv8_reserve(5, t.ints([0, 3, 2, 1, 4]), t.ints([71, 200, 64, 130, 129]), *t.table, served, *t.ws)
    assert served.get().tolist() == [0, 0, 1, 1, 1]
    pages, refs = t.pages.copy(), t.refs.copy()
    pages[4, 1:3], refs[free[:2]] = free[:2], 1
    assert np.array_equal(t.d_pages.get(), pages) and np.array_equal(t.d_refs.get(), refs)


def test_entries_outside_the_pool_are_no_pages(gpu):
    """A table entry of n_pages or more means that there is no page, as a negative one does: reserve fills
    it, and a sequence that has only such entries can become a child."""
    t = Table(gpu, 43, [70, 0, 0, 64], 5, 20, share=False)
    t.pages[1] = [20, -7, 1 << 30, 99, -1]
    t.pages[3, 1:3] = [21, -3]
    t.put()
    free = np.flatnonzero(t.refs == 0)
    served = t.dev.out((1,), np.int32)
    gpu.kv8_reserve(1, t.ints([3]), t.ints([192]), *t.table, served, *t.ws)
    assert served.get().tolist() == [1]
    assert t.d_pages.get()[3].tolist() == [t.pages[3, 0], free[0], free[1], -1, -1]
    served = t.dev.out((1,), np.int32)
    gpu.kv8_fork(t.pool, 1, t.ints([0]), t.ints([1]), *t.table, served, *t.ws)
    assert served.get().tolist() == [1]
    pages, refs = t.d_pages.get(), t.d_refs.get()
    assert pages[1, 0] == t.pages[0, 0] and pages[1, 1] == free[2] and refs[pages[1, 0]] == 2 and refs[free[2]] == 1
    assert t.d_len.get()[1] == 70
    assert all(not 0 <= p < 20 for p in pages[1, 2:])


# ---- the four-tile form, where the others are tested at smaller sizes -------------------------------


FILL = ([700, 430, 5, 64], [700, 430, 1, 0])  # rows for a block of four tiles on most SMs


@pytest.mark.parametrize("out_name,pad,offset,pad_out", [("f32", 3, 1, 5), ("bf16", 8, 0, 8), ("f32", 4, 4, 4)])
def test_four_tiles_strides_and_types(gpu, out_name, pad, offset, pad_out):
    pkg = gpu
    st = Step(pkg, 301 + pad, *FILL, 64, 8, 64, pkg.BF16, pad=pad, offset=offset, layers=2, layer=1, lead=2, trail=3).put()
    st.check_attend(pkg.F32 if out_name == "f32" else pkg.BF16, pad_out=pad_out, sinks=st.r.standard_normal(64).astype(np.float32))


def test_four_tiles_extreme_values(gpu):
    """Scores far apart, equal scores, huge and tiny rows, pages of zeros and of scale 0, a negative and a zero scale; more
    rows than max_new; windows that leave nothing where pages are missing."""
    pkg = gpu
    st = Step(pkg, 311, *FILL, 64, 8, 64, pkg.BF16, scales=(-24, 4), missing=[(0, 2, -1), (0, 3, 1 << 30), (1, 1, -9)])
    st.x[:, :64] *= 40
    st.x[:, 64:128] = 0
    st.x[:, 128:192] *= np.float32(1e-18)
    st.x[:, 192:256] *= np.float32(2e4)
    st.x = widen(pkg, st.x, pkg.BF16)
    st.scales[0, st.pages[0, 5], :, 1] = 0
    st.scales[0, st.pages[0, 4], :, 0] = 0
    st.scales[0, st.pages[0, 6], :, 1] = 2.0 ** -100
    st.codes[0, st.pages[1, 0]] = 0
    st.put()
    st.check_attend(scale=-0.25)
    st.check_attend(scale=0.0, sinks=np.full(64, -1e30, np.float32))
    st.check_attend(window=30, max_new=640)
    assert pkg.load().gptoss_wait_giveups() == 0


# ---- release and attention together --------------------------------------------------------------


@pytest.mark.parametrize("window,first", [(1, 0), (64, 0), (65, 64), (128, 4), (100, 70), (1000, 0)])
@pytest.mark.parametrize("new", [1, 9])
def test_what_is_released_is_not_missed(gpu, window, first, new):
    """Pages let go of behind a window belong to others from then on (junk, scales that are NaN): the rows that come
    next give what the definition gives with the whole cache."""
    pkg = gpu
    lens = [1, 64, 65, 300, 383, 256]
    st = Step(pkg, 321 + window, [n + new for n in lens], [new] * 6, 8, 2, 64, pkg.BF16).put()
    ref = want(st, window=window, first=first)
    refs = np.bincount(st.pages[st.pages >= 0], minlength=st.codes.shape[1]).astype(np.int32)
    d_len, d_refs, d_pages = (st.dev.put_inout(a) for a in (np.asarray(lens, np.int32), refs, st.pages))
    pkg.kv8_release(6, st.dev.put(np.arange(6, dtype=np.int32)), 6, d_len, d_pages, st.width, len(refs), d_refs, window, first)
    left = d_refs.get()
    assert (left <= refs).all() and (left < refs).any() == (window < 1000)
    st.scales[:, (refs > 0) & (left == 0)] = np.nan
    st.d_scales, st.d_pages = st.dev.put_inout(st.scales), d_pages
    st.pool = pkg.kv8_pool(st.d_codes, st.d_scales, 1, st.codes.shape[1], st.heads, st.D)
    check(st, run(st, pkg.F32, window=window, first=first), *ref, pkg.F32)


# ---- long sums ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("n,new,kv,n_q,heads", [(1, 5000, 5000, 4, 1), (296, 1, 9600, 16, 4), (150, 3, 9600, 16, 4), (1, 30, 40000, 4, 1)])
def test_fp32_rows_over_long_contexts(gpu, n, new, kv, n_q, heads):
    """The matrix units cut off, on average half a unit (2^-24) per addition, and sums that grow evenly lose half of what
    their last additions would: over 64 additions 64 / 2 * 2^-24 = 2^-19 of the whole, to which everything else that
    rounds to nearest adds little.  One chain of additions over all tokens loses 10 to 100 times that.  Values of one
    sign, so that nothing cancels."""
    pkg = gpu
    st = Step(pkg, 401 + new, [kv], [n * new], n_q, heads, 64, pkg.F32)
    st.row_start, st.kv_len = np.arange(0, n * new + 1, new, dtype=np.int32), np.full(n, kv, np.int32)
    st.pages, st.max_new = np.tile(st.pages, (n, 1)), new  # all read one sequence's pages
    st.x[:, :n_q * 64] *= 0.25
    st.codes[0, :, :, 1] = np.abs(st.codes[0, :, :, 1])
    st.put()
    got = run(st, pkg.F32).astype(np.float64)
    rows = np.unique(np.linspace(0, st.T - 1, 24).astype(int))  # the definition at some of the rows
    k, v = ((st.codes[0, st.pages[0], :, i].astype(np.float64) * st.scales[0, st.pages[0], :, i][..., None, None])
            .transpose(1, 0, 2, 3).reshape(heads, -1, 64) for i in (0, 1))
    ref = np.zeros((len(rows), n_q, 64))
    for i, r in enumerate(rows):
        pos = kv - new + r % new
        q = st.x[r, :n_q * 64].reshape(n_q, 64).astype(np.float64)
        for h in range(n_q):
            z = 0.125 * (k[h * heads // n_q, :pos + 1] @ q[h])
            w = np.exp(z - z.max())
            ref[i, h] = w @ v[h * heads // n_q, :pos + 1] / w.sum()
    assert np.linalg.norm(got[rows] - ref) <= 2.0 ** -19 * np.linalg.norm(ref)
