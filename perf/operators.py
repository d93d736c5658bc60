"""The 8-bit paged key/value cache as operators to be timed: appending rows, attention over the
cache, and the pages' bookkeeping.

A cache page holds 64 tokens.  For each page, key/value head and kind (0 key, 1 value) it has
64 x head_dim int8 codes and ONE fp32 scale, a power of two; a value is code * scale.  A pool is

    codes  [n_layers][n_pages][n_kv_heads][2][64][head_dim]  int8
    scales [n_layers][n_pages][n_kv_heads][2]                fp32

and a sequence's tokens are found through its row of a page table, shared by all layers
(-1: no page).  A step's rows come as rows of the rotated qkv tensor, sequence after sequence:
rows row_start[s] .. row_start[s+1] are the newest tokens of sequence s, whose length WITH them
is kv_len[s].

`own` false computes the operators from elementary torch operations; true makes the calls of
this repository's library.
"""
import importlib
import math
import random

import torch

own = False
PAGE = 64

# ---- the cases -------------------------------------------------------------------------

# The attention heads of the model family this library serves: 64 query and 8 key/value heads of
# 64 elements; a window of 128 in every other layer, one learned sink logit per query head.
HEADS = dict(hq=64, hkv=8, d=64)


def _append(name, n, new, kv, dtype, ragged, shape=1, **heads):
    return {"name": name, "op": "append", "n": n, "new": new, "kv": kv, "dtype": dtype, "ragged": ragged,
            "shape": shape, **(heads or HEADS)}


def _attend(name, n, new, kv, dtype, ragged, window=0, first=0, sinks=False, shape=1, **heads):
    return {"name": name, "op": "attend", "n": n, "new": new, "kv": kv, "dtype": dtype, "ragged": ragged,
            "window": window, "first": first, "sinks": sinks, "shape": shape, **(heads or HEADS)}


def _pages(name, n, kv, layers, spare, shape=1, **heads):
    return {"name": name, "op": "pages", "n": n, "kv": kv, "layers": layers, "spare": spare, "shape": shape,
            **(heads or HEADS)}


def listed():
    return [
        # one request decoding: the smallest call there is, fp32 activations
        _append("append_one_f32", 1, 1, 77, "f32", False),
        # a decode step of a full batch
        _append("append_batch", 192, 1, 120, "bf16", True),
        # prompts of very different lengths arriving together
        _append("append_prompts", 12, 2500, 2500, "bf16", True),
        # one request decoding with a short context, a windowed layer
        _attend("attend_one", 1, 1, 777, "bf16", False, window=128, first=4, sinks=True),
        # a decode step of a full batch on a windowed layer: contexts long, what is read short
        _attend("attend_window_batch", 128, 1, 8000, "bf16", True, window=128, first=4, sinks=True),
        # the same on a full layer: the cache is streamed
        _attend("attend_batch", 64, 1, 16000, "bf16", True, sinks=True),
        # one request with a very long context, wider heads
        _attend("attend_long", 1, 1, 131072, "bf16", False, hq=32, hkv=8, d=128),
        # a step that checks a few guessed tokens per request, fp32 mode
        _attend("attend_verify_f32", 24, 5, 4099, "f32", True, sinks=True),
        # chunks of prompts that continue what is in the cache; five query heads per key head
        _attend("attend_chunks", 5, 600, 9000, "bf16", True, first=16, window=4096, hq=40, hkv=8, d=64),
        # a whole prompt against itself
        _attend("attend_prompt", 1, 8192, 8192, "bf16", False, sinks=True),
        # a small server's table, one layer's pool
        _pages("pages_small", 13, 300, 1, 0.3),
        # a beam or sampling step of a big batch: sequences end, others fork, all grow, the pool
        # is compacted; several layers share the table
        _pages("pages_batch", 200, 1500, 8, 0.5),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads = rng.choice([HEADS, HEADS, dict(hq=32, hkv=8, d=128), dict(hq=40, hkv=8, d=64), dict(hq=8, hkv=8, d=64),
                        dict(hq=16, hkv=1, d=128), dict(hq=12, hkv=4, d=64)])
    dtype, shape = rng.choice(["bf16", "bf16", "f32"]), rng.randrange(1 << 20)
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "pages"])
    if op == "append":
        new = rng.choice([1, 1, _spread(rng, 2, 2500)])
        n = _spread(rng, 1, 192 if new == 1 else max(1, min(64, 28000 // new)))
        c = _append("", n, new, new + rng.randrange(0, 150), dtype, n > 1 and rng.random() < 0.7, shape, **heads)
    elif op == "attend":
        window = rng.choice([0, 0, 128, _spread(rng, 1, 5000)])
        first = rng.choice([0, 4, rng.randrange(0, 200)])
        kind = rng.choice(["token", "token", "verify", "chunk", "prompt"])
        if kind == "prompt":  # whole prompts
            new = kv = _spread(rng, 17, 6000)
            n = max(1, min(8, 6000 * 6000 // (new * new)))
        elif kind == "chunk":
            new, kv = _spread(rng, 20, 1000), _spread(rng, 1100, 20000)
            n = max(1, min(8, 20_000_000 // (new * kv)))
        else:
            new = 1 if kind == "token" else rng.randrange(2, 9)
            kv = _spread(rng, 9, 100000)
            n = _spread(rng, 1, max(1, min(192, 500000 // (kv * new))))
        c = _attend("", n, new, kv, dtype, n > 1 and rng.random() < 0.7, window, first, rng.random() < 0.5, shape, **heads)
    else:
        c = _pages("", _spread(rng, 5, 160), _spread(rng, 40, 1200), rng.randrange(1, 6), rng.uniform(0.1, 0.8), shape, **heads)
    del c["name"]
    return c


def _lengths(case):
    """(kv_len, new rows) of each sequence; fixed by the case, not by the seed."""
    r = random.Random(case["shape"])
    kv, new = [], []
    for _ in range(case["n"]):
        q = r.randint((case["new"] + 1) // 2, case["new"]) if case["ragged"] else case["new"]
        k = r.randint(min(q, case["kv"]), case["kv"]) if case["ragged"] else case["kv"]
        if case["ragged"] and case["new"] == case["kv"]:  # whole prompts
            k = q = r.randint(1, case["kv"])
        kv.append(max(k, q))
        new.append(q)
    if case["ragged"] and case["n"] >= 4 and case["new"] > 1:
        new[1] = 0  # a sequence that sits this step out
    return kv, new


def _visible(case, kv, new):
    """(distinct tokens seen by any of the new rows, pairs of row and token seen)."""
    if not new:
        return 0, 0
    first_pos, w, f = kv - new, case["window"], case["first"]
    if w <= 0:
        return kv, sum(range(first_pos + 1, kv + 1))
    lo = max(0, first_pos - w + 1)
    pairs = sum(p + 1 - max(0, p - w + 1) + min(f, max(0, p - w + 1)) for p in range(first_pos, kv))
    return kv - lo + min(f, lo), pairs


def _elt(case):
    return 2 if case["dtype"] == "bf16" else 4


def _pages_plan(case):
    """A pages case's sequences: lengths, who is let go, who forks into whom, who grows to what."""
    r = random.Random(case["shape"])
    n = case["n"]
    lens = [r.randint(max(1, case["kv"] // 4), case["kv"]) for _ in range(n)]
    order = list(range(n))
    r.shuffle(order)
    n_gone, n_empty = max(1, n // 5), max(1, n // 5)
    gone, empty, stay = order[:n_gone], order[n_gone:n_gone + n_empty], order[n_gone + n_empty:]
    for s in empty:
        lens[s] = 0
    children = (gone + empty)[: max(1, (n_gone + n_empty) * 3 // 4)]
    parents = [r.choice(stay) for _ in children]
    grow = [lens[s] + r.randint(0, 100) for s in stay]
    return lens, gone, parents, children, stay, grow


def _pages_counts(case):
    lens, gone, parents, children, stay, grow = _pages_plan(case)
    table = -(-max(lens + grow) // PAGE)
    held = sum(-(-x // PAGE) for x in lens)
    n_pages = int((held + len(children) + sum(-(-g // PAGE) - -(-lens[s] // PAGE) for s, g in zip(stay, grow)))
                  * (1 + case["spare"])) + 2
    return table, held, n_pages


def work(case):
    elt, hkv, d = _elt(case) if "dtype" in case else 0, case["hkv"], case["d"]
    if case["op"] == "append":
        kv, new = _lengths(case)
        rows = sum(new) * 2 * hkv * d
        touched = sum(-(-k // PAGE) - (k - q) // PAGE for k, q in zip(kv, new) if q)
        # rows in, codes out, a scale in and out per touched page; then the pool's values come back as bf16
        pool = _append_pages(case)[1] * hkv * 2 * PAGE * d
        return {"bytes": rows * (elt + 1) + touched * hkv * 2 * 8 + pool * 3, "flops": rows * 4}
    if case["op"] == "attend":
        kv, new = _lengths(case)
        seen = [_visible(case, k, q) for k, q in zip(kv, new)]
        tokens, pairs = sum(t for t, _ in seen), sum(p for _, p in seen)
        return {"bytes": tokens * hkv * 2 * d + sum(-(-t // PAGE) for t, _ in seen) * hkv * 8
                + sum(new) * case["hq"] * d * elt * 2, "flops": pairs * case["hq"] * 4 * d}
    lens, gone, parents, children, stay, grow = _pages_plan(case)
    table, held, n_pages = _pages_counts(case)
    page = case["layers"] * hkv * 2 * (PAGE * d + 4)
    copies = sum(lens[p] % PAGE != 0 for p in parents)
    after = held - sum(-(-lens[s] // PAGE) for s in gone) + copies + sum(
        -(-g // PAGE) - -(-lens[s] // PAGE) for s, g in zip(stay, grow))
    moves = after * (1 - after / n_pages)  # live pages lie anywhere; the pages asked for take the lowest free ones
    return {"bytes": (copies + moves) * page * 2 + case["n"] * table * 8 + n_pages * 12, "flops": 0}


# ---- inputs ----------------------------------------------------------------------------

def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _two_to(e):
    """2^e as fp32, exact (exp2 and pow are not on every device)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _random_pool(g, layers, n_pages, hkv, d):
    codes = torch.empty(layers, n_pages, hkv, 2, PAGE, d, dtype=torch.int8, device="cuda")
    for i in range(layers):  # bell-shaped codes that use the whole range, as a page with its own scale has them
        codes[i] = (torch.randn(n_pages, hkv, 2, PAGE, d, generator=g, device="cuda") * 32).round_().clamp_(-127, 127)
    scales = _two_to(torch.randint(-7, -3, (layers, n_pages, hkv, 2), generator=g, device="cuda"))
    return codes, scales


def _append_pages(case):
    """Table width and pool size of an append case: only pages that new rows touch are in the pool."""
    kv, new = _lengths(case)
    touched = sum(-(-k // PAGE) - (k - q) // PAGE for k, q in zip(kv, new) if q)
    return -(-max(kv) // PAGE), touched + touched // 8 + 1


def _table(g, spans, width, n_pages):
    """A page table [n][width] whose entries lo..hi of each row are distinct random pages, the others -1."""
    table = torch.full((len(spans), width), -1, dtype=torch.int32)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(g.initial_seed())).to(torch.int32)
    at = 0
    for s, (lo, hi) in enumerate(spans):
        table[s, lo:hi] = order[at:at + hi - lo]
        at += hi - lo
    return table.cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hkv, d = case["hkv"], case["d"]
    st = {"case": case, "op": case["op"]}
    if case["op"] == "pages":
        lens, gone, parents, children, stay, grow = _pages_plan(case)
        width, held, n_pages = _pages_counts(case)
        st["codes"], st["scales"] = _random_pool(g, case["layers"], n_pages, hkv, d)
        st["pages"] = _table(g, [(0, -(-x // PAGE)) for x in lens], width, n_pages)
        st["kv_len"] = _ints(lens)
        st["refs"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        st["refs"][st["pages"][st["pages"] >= 0].long()] = 1
        for k, v in dict(gone=gone, parents=parents, children=children, stay=stay, grow=grow).items():
            st[k] = _ints(v)
        st["served"] = torch.zeros(2, max(len(stay), len(children)), dtype=torch.int32, device="cuda")
        st["remap"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        st["n_live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        kv, new = _lengths(case)
        T, width = sum(new), (case["hq"] + 2 * hkv) * d
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        st["qkv"] = torch.randn(T, width, generator=g, device="cuda").to(dtype)
        head = torch.exp(torch.randn(width // d, generator=g, device="cuda") * 0.5)  # heads differ in size
        st["qkv"] *= head.repeat_interleave(d).to(dtype)
        st["kv_len"], st["new"] = _ints(kv), _ints(new)
        st["row_start"] = _ints([sum(new[:s]) for s in range(len(new) + 1)])
        st["T"], st["max_new"] = T, max(new)
        if case["op"] == "append":
            table, n_pages = _append_pages(case)
            spans = [((k - q) // PAGE, -(-k // PAGE)) if q else (0, 0) for k, q in zip(kv, new)]
        else:
            table, n_pages = -(-max(kv) // PAGE), sum(-(-k // PAGE) for k in kv) + 3
            spans = [(0, -(-k // PAGE)) for k in kv]
            st["out"] = torch.zeros(T, case["hq"] * d, dtype=dtype, device="cuda")
            st["sinks"] = torch.randn(case["hq"], generator=g, device="cuda") if case["sinks"] else None
        st["codes"], st["scales"] = _random_pool(g, 1, n_pages, hkv, d)
        st["pages"] = _table(g, spans, table, n_pages)
    if own:
        _prepare_own(st)
    return st


def _prepare_own(st):
    lib = st["lib"] = importlib.import_module("optimize_inference_gpt-oss_b200")
    layers, n_pages, hkv, _, _, d = st["codes"].shape
    st["pool"] = lib.kv8_pool(st["codes"].data_ptr(), st["scales"].data_ptr(), layers, n_pages, hkv, d)
    nbytes = 0
    if st["op"] == "attend":
        nbytes = lib.kv8_attention_workspace(st["pool"], st["T"], st["case"]["hq"], st["case"]["n"], st["max_new"])
    elif st["op"] == "pages":
        nbytes = lib.kv8_pages_workspace(n_pages, st["pages"].shape[0])
    st["workspace"] = torch.zeros(max(nbytes, 16), dtype=torch.uint8, device="cuda")


# ---- one pass --------------------------------------------------------------------------

def run(st):
    return {"append": _run_append, "attend": _run_attend, "pages": _run_pages}[st["op"]](st)


def _run_append(st):
    c = st["case"]
    if own:
        lib = st["lib"]
        lib.kv8_append(st["pool"], 0, st["T"], st["qkv"].data_ptr(), _dtype(lib, c), st["qkv"].stride(0), c["hq"], c["n"],
                       st["row_start"].data_ptr(), st["kv_len"].data_ptr(), st["pages"].data_ptr(), st["pages"].shape[1],
                       st["max_new"], stream=torch.cuda.current_stream().cuda_stream)
    else:
        _plain_append(st)
    # the cache as the values it stands for (a code times a power of two is exact in bf16)
    return st["codes"][0].bfloat16() * st["scales"][0].bfloat16()[..., None, None]


def _run_attend(st):
    c = st["case"]
    if not own:
        return _plain_attend(st)
    lib = st["lib"]
    lib.kv8_attention(st["pool"], 0, st["T"], st["qkv"].data_ptr(), _dtype(lib, c), st["qkv"].stride(0), c["hq"], c["n"],
                      st["row_start"].data_ptr(), st["kv_len"].data_ptr(), st["pages"].data_ptr(), st["pages"].shape[1],
                      st["max_new"], 1.0 / math.sqrt(c["d"]), c["window"], c["first"],
                      st["sinks"].data_ptr() if st["sinks"] is not None else None, st["out"].data_ptr(), _dtype(lib, c),
                      st["out"].stride(0), st["workspace"].data_ptr(), st["workspace"].numel(),
                      stream=torch.cuda.current_stream().cuda_stream)
    return st["out"]


def _run_pages(st):
    # the tables are copied so that every pass starts from the same ones; the pool is changed in
    # place: what a pass writes, it writes again with the same values
    pages, refs, kv_len = st["pages"].clone(), st["refs"].clone(), st["kv_len"].clone()
    if not own:
        return _plain_pages(st, pages, refs, kv_len)
    lib, stream = st["lib"], torch.cuda.current_stream().cuda_stream
    n_seqs, width, n_pages = pages.shape[0], pages.shape[1], refs.shape[0]
    table = (n_seqs, kv_len.data_ptr(), pages.data_ptr(), width, n_pages, refs.data_ptr())
    ws = (st["workspace"].data_ptr(), st["workspace"].numel())
    n_fork, n_grow = st["children"].numel(), st["stay"].numel()
    lib.kv8_release(st["gone"].numel(), st["gone"].data_ptr(), *table, stream=stream)
    lib.kv8_fork(st["pool"], n_fork, st["parents"].data_ptr(), st["children"].data_ptr(), *table,
                 st["served"][0].data_ptr(), *ws, stream=stream)
    lib.kv8_reserve(n_grow, st["stay"].data_ptr(), st["grow"].data_ptr(), *table, st["served"][1].data_ptr(), *ws, stream=stream)
    lib.kv8_compact(st["pool"], *table, st["remap"].data_ptr(), st["n_live"].data_ptr(), *ws, stream=stream)
    return _pages_out(st, pages, refs, kv_len, st["served"][0, :n_fork], st["served"][1, :n_grow], st["remap"], st["n_live"])


def _pages_out(st, pages, refs, kv_len, forked, grown, remap, n_live):
    # pages are moved as bytes: codes and scales are whole numbers here
    return {"pages": pages, "refs": refs, "kv_len": kv_len, "forked": forked, "grown": grown, "remap": remap,
            "n_live": n_live, "codes": st["codes"], "scales": st["scales"].view(torch.int32)}


def _dtype(lib, case):
    return lib.BF16 if case["dtype"] == "bf16" else lib.F32


# ---- the operators in plain form ---------------------------------------------------------

def _rows_of(st):
    """Sequence and position of every row."""
    t = torch.arange(st["T"], device="cuda")
    start = st["row_start"].long()
    seq = torch.searchsorted(start[1:], t, right=True)
    return seq, st["kv_len"].long()[seq] - start[seq + 1] + t


def _power_of_two(need):
    """The smallest power of two s, at least 2^-126, with need <= 127 s; 0 for need = 0."""
    f, x = torch.frexp(need)
    e = torch.where(f <= 127 / 128, x - 7, x - 6).clamp_(min=-126)
    return torch.where(need > 0, _two_to(e), torch.zeros_like(need))


def _plain_append(st):
    codes, scales = st["codes"][0], st["scales"][0]
    n_pages, hkv, _, _, d = codes.shape
    rows = st["qkv"][:, -2 * hkv * d:].float().view(-1, 2, hkv, d).transpose(1, 2)
    seq, pos = _rows_of(st)
    page, slot = st["pages"][seq, pos // PAGE].long(), pos % PAGE
    need = torch.zeros_like(scales).index_reduce_(0, page, rows.abs().amax(-1), "amax")
    first = torch.full((n_pages,), PAGE, device="cuda").index_reduce_(0, page, slot, "amin")
    old = torch.where((first > 0)[:, None, None], scales, 0.0)
    new = torch.maximum(old, _power_of_two(need))
    # codes that were there already are brought to the page's new scale
    keep = torch.where(new > 0, old / new, 1.0)[..., None, None]
    earlier = (torch.arange(PAGE, device="cuda") < first[:, None])[:, None, None, :, None]
    codes.copy_(torch.where(earlier, (codes.float() * keep).round(), codes.float()))
    inverse = torch.where(new > 0, 1.0 / new, 0.0)
    codes[page, :, :, slot] = (rows * inverse[page][..., None]).round().to(torch.int8)
    scales.copy_(new)


def _plain_attend(st):
    c = st["case"]
    hq, hkv, d, n, M = c["hq"], c["hkv"], c["d"], c["n"], st["max_new"]
    G, L = hq // hkv, st["pages"].shape[1] * PAGE
    at = st["pages"].clamp(min=0).long()
    kv = (st["codes"][0][at].float() * st["scales"][0][at][..., None, None]).permute(3, 0, 2, 1, 4, 5)
    K, V = kv.reshape(2, n, hkv, L, d)
    seq, pos = _rows_of(st)
    i = torch.arange(st["T"], device="cuda") - st["row_start"].long()[seq]
    q = torch.zeros(n, M, hkv, G, d, device="cuda")
    q[seq, i] = st["qkv"][:, : hq * d].float().view(-1, hkv, G, d)
    S = (q.permute(0, 2, 3, 1, 4).reshape(n, hkv, G * M, d) @ K.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(n, hkv, G, M, L)
    p = (st["kv_len"] - st["new"])[:, None] + torch.arange(M, device="cuda")  # position of row i of each sequence
    t = torch.arange(L, device="cuda")
    sees = (t <= p[..., None]) & (st["pages"] >= 0).repeat_interleave(PAGE, 1)[:, None]
    if c["window"] > 0:
        sees &= (t > p[..., None] - c["window"]) | (t < c["first"])
    S.masked_fill_(~sees[:, None, None], -math.inf)
    m = S.amax(-1, keepdim=True)
    if st["sinks"] is not None:
        sink = st["sinks"].view(hkv, G, 1, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    P = S.sub_(m).exp_()
    l = P.sum(-1, keepdim=True)
    if st["sinks"] is not None:
        l = l + (sink - m).exp()
    O = (P.view(n, hkv, G * M, L) @ V).view(n, hkv, G, M, d) / torch.where(l > 0, l, 1.0)
    return O.permute(0, 3, 1, 2, 4)[seq, i].reshape(-1, hq * d).to(st["out"].dtype)


def _lowest_free(refs):
    """A function from k (1-based) to the k-th lowest page that nobody holds."""
    count = torch.cumsum(refs == 0, 0)
    return lambda k: torch.searchsorted(count, k)


def _plain_pages(st, pages, refs, kv_len):
    one, j = torch.ones((), dtype=torch.int32, device="cuda"), torch.arange(pages.shape[1], device="cuda")
    # release: every page of the sequences has one holder fewer
    gone = st["gone"].long()
    held = pages[gone]
    refs.index_put_((held.clamp(min=0).flatten().long(),), -(held >= 0).int().flatten(), accumulate=True)
    pages[gone], kv_len[gone] = -1, 0
    # fork: full pages are shared, a last page that is not full is copied into a free one
    par, kid = st["parents"].long(), st["children"].long()
    length = kv_len[par]
    full = (length // PAGE)[:, None]
    shared = torch.where(j < full, pages[par], -1)
    part = length % PAGE > 0
    src = pages[par].gather(1, full.long().clamp(max=pages.shape[1] - 1))[:, 0].long()
    dst = torch.where(part, _lowest_free(refs)(torch.cumsum(part, 0)), src)
    refs.index_put_((shared.clamp(min=0).flatten().long(),), (shared >= 0).int().flatten(), accumulate=True)
    refs[dst[part]] = one
    pages[kid] = torch.where((j == full) & part[:, None], dst[:, None].int(), shared)
    kv_len[kid] = length
    st["codes"][:, dst[part]] = st["codes"][:, src[part]]
    st["scales"][:, dst[part]] = st["scales"][:, src[part]]
    # reserve: pages for the tokens to come
    stay = st["stay"].long()
    fresh = (j >= ((kv_len[stay] + PAGE - 1) // PAGE)[:, None]) & (j < ((st["grow"] + PAGE - 1) // PAGE)[:, None]) & (pages[stay] < 0)
    k = torch.cumsum(fresh.flatten(), 0).view_as(fresh)
    page = _lowest_free(refs)(k)
    refs[page[fresh]] = one
    pages[stay] = torch.where(fresh, page.int(), pages[stay])
    # compact: the live pages furthest back move into the holes in front of them
    live, index = refs > 0, torch.arange(refs.shape[0], device="cuda")
    n_live = live.sum()
    to = torch.nonzero(~live & (index < n_live))[:, 0]
    fro = torch.nonzero(live & (index >= n_live))[:, 0]
    remap = torch.where(live, index, -1).int()
    remap[fro] = to.int()
    st["codes"][:, to] = st["codes"][:, fro]
    st["scales"][:, to] = st["scales"][:, fro]
    refs[to], refs[fro] = refs[fro], 0
    pages = torch.where(pages >= 0, remap[pages.clamp(min=0).long()], -1)
    return _pages_out(st, pages, refs, kv_len, torch.ones_like(st["parents"]), torch.ones_like(st["stay"]), remap, n_live.int()[None])


# ---- the definitions in 64 bits ------------------------------------------------------------

def exact(case, seed):
    """What run() returns, sequence by sequence from the definitions, in fp64."""
    if case["op"] == "pages":
        return None  # nothing is computed: pages move
    global own
    was, own = own, False
    st = prepare(case, seed)
    own = was
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    kv, new = _lengths(case)
    x = st["qkv"].double().view(st["T"], hq + 2 * hkv, d)
    table = st["pages"].tolist()
    codes, scales = st["codes"][0].double(), st["scales"][0].double()
    start = 0
    if case["op"] == "append":
        for s, (length, q) in enumerate(zip(kv, new)):
            for p in range((length - q) // PAGE, -(-length // PAGE) if q else 0):
                a, b = max(length - q, p * PAGE), min(length, (p + 1) * PAGE)  # positions of its new rows
                r = x[start + a - (length - q): start + b - (length - q), hq:]
                r = r.reshape(b - a, 2, hkv, d).permute(2, 1, 0, 3)  # head, kind, row, element
                page, slot = table[s][p], a % PAGE
                top = r.abs().amax((2, 3))
                want = torch.tensor([[2.0 ** math.ceil(math.log2(u / 127)) if u else 0.0 for u in w] for w in top.tolist()],
                                    dtype=torch.float64, device="cuda")
                now = torch.maximum(want, scales[page]) if slot else want
                if slot:
                    codes[page, :, :, :slot] = torch.round(codes[page, :, :, :slot] * (scales[page] / now)[..., None, None])
                codes[page, :, :, slot: slot + b - a] = torch.round(r / now.clamp(min=1e-300)[..., None, None])
                scales[page] = now
            start += q
        return codes * scales[..., None, None]
    if sum(_visible(case, k, q)[1] for k, q in zip(kv, new)) * hq * d > 4e12:
        return None
    out = torch.zeros(st["T"], hq, d, dtype=torch.float64, device="cuda")
    for s, (length, q) in enumerate(zip(kv, new)):
        page = torch.tensor(table[s][: -(-length // PAGE)], device="cuda")
        for h in range(hq if q else 0):
            g = h // (hq // hkv)
            k, v = ((codes[page, g, i] * scales[page, g, i][:, None, None]).reshape(-1, d)[:length] for i in (0, 1))
            z = x[start: start + q, h] @ k.T / d ** 0.5
            at, seen = torch.arange(length - q, length, device="cuda")[:, None], torch.arange(length, device="cuda")[None]
            ok = seen <= at
            if case["window"] > 0:
                ok = ok & ((at - seen < case["window"]) | (seen < case["first"]))
            z = torch.where(ok, z, -math.inf)
            if case["sinks"]:
                z = torch.cat([z, st["sinks"][h].double().expand(q, 1)], 1)
            out[start: start + q, h] = torch.softmax(z, 1)[:, :length] @ v
        start += q
    return out.reshape(st["T"], hq * d)
