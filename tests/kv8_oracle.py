"""What the 8-bit paged cache's entry points are defined to do, in numpy: appending in exact
arithmetic, attention in 64 bits, and the page calls as the sequential programs their results are
those of."""
from __future__ import annotations

import math

import numpy as np

PAGE = 64
F32_MAX = float(np.finfo(np.float32).max)


def scale_for(top: float) -> float:
    """The smallest power of two s >= 2^-126 with top <= 127 s; 0 for 0."""
    if top == 0:
        return 0.0
    s = 2.0 ** max(-126, math.frexp(top)[1] - 8)
    while top > 127 * s:
        s *= 2
    return s


def spans(row_start, kv_len, T, max_new):
    """Per sequence: first row, processed rows, position of the first row."""
    for s in range(len(kv_len)):
        r0, r1 = (min(max(int(r), 0), T) for r in row_start[s:s + 2])
        n = max(r1 - r0, 0)
        yield s, r0, min(n, max_new), max(int(kv_len[s]), 0) - n


def page_of(pages, s, pos, n_pages):
    if pos < 0 or pos // PAGE >= pages.shape[1]:
        return -1
    p = int(pages[s, pos // PAGE])
    return p if 0 <= p < n_pages else -1


def append(codes, scales, rows, n_q, row_start, kv_len, pages, max_new):
    """codes [pages][heads][2][64][D], scales [pages][heads][2], rows [T][(n_q + 2 heads) D] fp32:
    new codes and scales."""
    codes, scales = codes.copy(), scales.copy()
    n_pages, heads, _, _, D = codes.shape
    x = rows.reshape(rows.shape[0], -1, D)[:, n_q:].astype(np.float64).reshape(rows.shape[0], 2, heads, D)
    x = np.clip(np.where(np.isnan(x), 0.0, x), -F32_MAX, F32_MAX)
    for s, r0, q, pos in spans(row_start, kv_len, rows.shape[0], max_new):
        groups = {}
        for i in range(q):
            if page_of(pages, s, pos + i, n_pages) >= 0:
                groups.setdefault((pos + i) // PAGE, []).append(i)
        for p, idx in groups.items():
            page, slot = int(pages[s, p]), (pos + idx[0]) % PAGE
            for h in range(heads):
                for kind in range(2):
                    new = x[r0 + idx[0]:r0 + idx[-1] + 1, kind, h]
                    scale, old = scale_for(float(np.abs(new).max())), float(scales[page, h, kind])
                    if slot > 0 and old >= scale:
                        scale = old
                    elif slot > 0 and old > 0:
                        c = codes[page, h, kind, :slot].astype(np.float64)
                        codes[page, h, kind, :slot] = np.rint(c * (old / scale)).astype(np.int8)
                    codes[page, h, kind, slot:slot + len(idx)] = (np.rint(new / scale) if scale else new * 0).astype(np.int8)
                    scales[page, h, kind] = scale
    return codes, scales


def attend(codes, scales, rows, n_q, row_start, kv_len, pages, max_new, scale, window, n_first, sinks):
    """out [T][n_q][D] in fp64 (NaN where no row is processed); and per (row, head) what errors scale
    with: sum p |v| per element, the largest scale * sum |q k|, the tokens seen, the largest |v|."""
    n_pages, heads, _, _, D = codes.shape
    T, G = rows.shape[0], n_q // codes.shape[1]
    x = rows.reshape(T, -1, D)[:, :n_q].astype(np.float64)
    out, weight = np.full((T, n_q, D), np.nan), np.zeros((T, n_q, D))
    reach, seen, vmax = np.zeros((T, n_q, 1)), np.zeros((T, n_q, 1)), np.zeros((T, n_q, 1))
    for s, r0, q, pos in spans(row_start, kv_len, T, max_new):
        if not q:
            continue
        t = np.array([i for i in range(max(pos + q, 0)) if page_of(pages, s, i, n_pages) >= 0], np.int64)
        pg, slot = pages[s, t // PAGE] if len(t) else t, t % PAGE
        for h in range(n_q):
            g = h // G
            k = codes[pg, g, 0, slot].astype(np.float64) * scales[pg, g, 0].astype(np.float64)[:, None]
            v = codes[pg, g, 1, slot].astype(np.float64) * scales[pg, g, 1].astype(np.float64)[:, None]
            p = pos + np.arange(q)[:, None]
            ok = t[None] <= p
            if window > 0:
                ok &= (t[None] > p - window) | (t[None] < n_first)
            r = slice(r0, r0 + q)
            z = np.where(ok, scale * (x[r, h] @ k.T), -np.inf)
            top = z.max(1, initial=-np.inf, keepdims=True)
            if sinks is not None:
                top = np.maximum(top, sinks[h])
            top = np.where(np.isfinite(top), top, 0.0)
            w = np.exp(z - top)
            total = w.sum(1, keepdims=True)
            if sinks is not None:
                total = total + np.exp(float(sinks[h]) - top)
            any_ = ok.any(1, keepdims=True)
            total = np.where(any_, total, 1.0)
            out[r, h], weight[r, h] = w @ v / total, w @ np.abs(v) / total
            reach[r, h] = np.where(ok, np.abs(x[r, h]) @ np.abs(k.T), 0).max(1, initial=0, keepdims=True) * abs(scale)
            seen[r, h] = ok.sum(1, keepdims=True)
            vmax[r, h] = np.where(ok, np.abs(v).max(1), 0).max(1, initial=0, keepdims=True) if len(t) else 0
    return out, weight, reach, seen, vmax


def tolerance(ref, weight, reach, seen, vmax, in_f32, out_f32):
    """Absolute error allowed per element of `attend`'s first output.

    A score z is off by at most reach * 2^-18: the query is carried to 2^-22 (fp32 rows) or exactly
    (bf16 rows), each of at most 16 tensor-core steps may truncate the running sum by 2^-23 of it, and
    three fp32 roundings of 2^-24 follow.  That moves exp(z), and with it numerator and denominator, by
    the same fraction.  The weights are rounded to 2^-22 (fp32 rows: two fp16 parts) or to 2^-11
    (bf16 rows: one), their exponential is good to 2^-21, sums over the tokens truncate 2^-23 per 16
    tokens, merging parts and dividing costs some 2^-21 more.  A weight below fp16's normal range is
    off by 2^-33 of the largest weight.  Last, the output's own rounding."""
    share = 2 * reach * 2.0 ** -18 + 2.0 ** -19 + (seen / 16) * 2.0 ** -22 + (2.0 ** -22 if in_f32 else 2.0 ** -11)
    return weight * share + seen * vmax * 2.0 ** -33 + np.abs(ref) * (2.0 ** -23 if out_f32 else 2.0 ** -8) + 1e-30


# ---- pages ------------------------------------------------------------------------------


class Tables:
    def __init__(self, kv_len, pages, refs):
        self.kv_len, self.pages, self.refs = kv_len.copy(), pages.copy(), refs.copy()

    def has(self, s):
        return 0 <= s < len(self.kv_len)

    def is_page(self, p):
        return 0 <= p < len(self.refs)

    def free(self):
        return [int(p) for p in np.flatnonzero(self.refs == 0)]

    def release(self, seqs, window=0, n_first=0):
        for s in seqs:
            if not self.has(s):
                continue
            for j in range(self.pages.shape[1]):
                last = j * PAGE + PAGE - 1
                if window > 0 and (last > int(self.kv_len[s]) - window or j * PAGE < n_first):
                    continue
                if self.is_page(self.pages[s, j]):
                    self.refs[self.pages[s, j]] -= 1
                self.pages[s, j] = -1
            if window <= 0:
                self.kv_len[s] = 0

    def reserve(self, seqs, new_len):
        free, asked, served, before = self.free(), 0, [], set()
        give = []
        for s, want in zip(seqs, new_len):
            if not self.has(s) or s in before or want > self.pages.shape[1] * PAGE:
                before.add(s)
                served.append(0)
                continue
            before.add(s)
            cols = [j for j in range(-(-max(int(self.kv_len[s]), 0) // PAGE), -(-want // PAGE)) if self.pages[s, j] < 0]
            ok = asked + len(cols) <= len(free) or not cols
            if ok:
                give += [(s, j, free[asked + n]) for n, j in enumerate(cols)]
            asked += len(cols)
            served.append(int(ok))
        for s, j, p in give:
            self.pages[s, j], self.refs[p] = p, 1
        return served

    def fork(self, parents, children):
        """Returns served and the (src, dst) pages copied."""
        free, copies, served = self.free(), [], []
        asked = 0
        for i, (p, c) in enumerate(zip(parents, children)):
            ok = (self.has(p) and self.has(c) and c not in children[:i] and p not in children
                  and self.kv_len[c] == 0 and (self.pages[c] < 0).all() and 0 <= self.kv_len[p] <= self.pages.shape[1] * PAGE)
            served.append(int(ok))
            if not ok:
                continue
            full, part = divmod(int(self.kv_len[p]), PAGE)
            if part and self.is_page(self.pages[p, full]):
                asked += 1
                if asked > len(free):
                    served[-1] = 0
                    continue
                copies.append((int(self.pages[p, full]), free[asked - 1]))
        new = iter(copies)
        for i, (p, c) in enumerate(zip(parents, children)):
            if not served[i]:
                continue
            full, part = divmod(int(self.kv_len[p]), PAGE)
            for j in range(full):
                if self.is_page(self.pages[p, j]):
                    self.pages[c, j] = self.pages[p, j]
                    self.refs[self.pages[p, j]] += 1
            if part and self.is_page(self.pages[p, full]):
                self.pages[c, full] = next(new)[1]
                self.refs[self.pages[c, full]] = 1
            self.kv_len[c] = self.kv_len[p]
        return served, copies

    def compact(self):
        """Returns remap, the live pages, and the (src, dst) pages moved."""
        live = self.refs != 0
        n = int(live.sum())
        idx = np.arange(len(self.refs))
        dst, src = idx[~live & (idx < n)], idx[live & (idx >= n)]
        remap = np.where(live, idx, -1).astype(np.int32)
        remap[src] = dst
        self.refs[dst] = self.refs[src]
        self.refs[src] = 0
        ok = (self.pages >= 0) & (self.pages < len(self.refs))
        self.pages = np.where(ok, remap[np.where(ok, self.pages, 0)], self.pages).astype(np.int32)
        return remap, n, list(zip(src.tolist(), dst.tolist()))
