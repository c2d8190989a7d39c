"""The serving operators' workloads: a paged key-value cache, the attention that
reads it one token a sequence, the prompt's attention over a sliding window, and
the bookkeeping of the cache's pages.

Each case is one pass of one operator on operands that are resident on the GPU.
With `own` false, run() computes it in elementary torch operations in 32 bits;
with `own` true it makes the calls of sile_amd a serving program makes.

Layouts: pages [num_pages, kv_heads, page, d]; page tables int32 [rows, width],
-1 where a row holds no page; q, o [batch, q_heads, d] for one token and
[batch, heads, length, d] for a prompt.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
SIZE = {"f16": 2, "bf16": 2, "fp8": 1}
WORKSPACE = 64 << 20


def listed():
    return [
        # the smallest call: one short conversation, a small model's heads
        {"name": "decode_f16_1x300", "op": "decode", "dtype": "f16", "cache": "f16", "batch": 1,
         "kv_heads": 2, "group": 4, "d": 64, "page": 16, "longest": 300, "ragged": False,
         "window": 0, "sinks": 0},
        # a server's ordinary step: 32 conversations of all lengths up to 8192
        {"name": "decode_bf16_32x8192_ragged", "op": "decode", "dtype": "bf16", "cache": "bf16",
         "batch": 32, "kv_heads": 8, "group": 4, "d": 128, "page": 16, "longest": 8192,
         "ragged": True, "window": 0, "sinks": 0},
        # one long document: the only parallelism is over the cache's length
        {"name": "decode_f16_1x131071", "op": "decode", "dtype": "f16", "cache": "f16", "batch": 1,
         "kv_heads": 8, "group": 4, "d": 128, "page": 64, "longest": 131071, "ragged": False,
         "window": 0, "sinks": 0},
        # an 8-bit cache under many query heads
        {"name": "decode_fp8_64x4000", "op": "decode", "dtype": "bf16", "cache": "fp8", "batch": 64,
         "kv_heads": 8, "group": 8, "d": 128, "page": 32, "longest": 4000, "ragged": True,
         "window": 0, "sinks": 0},
        # long conversations under a model that sees 1000 tokens back and the first four
        {"name": "decode_bf16_100x20000_w1000", "op": "decode", "dtype": "bf16", "cache": "bf16",
         "batch": 100, "kv_heads": 4, "group": 5, "d": 80, "page": 16, "longest": 20000,
         "ragged": True, "window": 1000, "sinks": 4},
        # a long prompt's attention over its last 1024 tokens and the first four
        {"name": "window_bf16_8192_w1024", "op": "window", "dtype": "bf16", "batch": 1,
         "kv_heads": 8, "group": 4, "d": 128, "q_len": 8192, "start": 0, "window": 1024,
         "sinks": 4},
        # a prompt taken in pieces: 512 new tokens behind 7680 cached ones
        {"name": "window_f16_chunk512_w4096", "op": "window", "dtype": "f16", "batch": 2,
         "kv_heads": 4, "group": 4, "d": 128, "q_len": 512, "start": 7680, "window": 4096,
         "sinks": 4},
        # short prompts, narrow heads of a width no tile has, a window of a hundred
        {"name": "window_f16_777_d72", "op": "window", "dtype": "f16", "batch": 2, "kv_heads": 2,
         "group": 3, "d": 72, "q_len": 777, "start": 0, "window": 100, "sinks": 1},
        # one token of each of 64 conversations into the cache, out of the fused projection
        {"name": "append_bf16_64", "op": "append", "dtype": "bf16", "cache": "bf16", "rows": 64,
         "each": 1, "kv_heads": 8, "group": 4, "d": 128, "page": 16},
        # two prompts of 8191 tokens into an 8-bit cache
        {"name": "append_fp8_2x8191", "op": "append", "dtype": "bf16", "cache": "fp8", "rows": 2,
         "each": 8191, "kv_heads": 8, "group": 4, "d": 128, "page": 32},
        # a step of beam search: finished rows dropped, beams forked, a page made
        # writable for each (the forks' last pages copied)
        {"name": "pages_step_256", "op": "pages_step", "rows": 256, "width": 128, "page": 16,
         "kv_heads": 8, "d": 128, "forks": 4},
        # a pool of 4500 pages, a third of them free here and there, closed up
        {"name": "pages_compact_4500", "op": "pages_compact", "rows": 64, "width": 96, "page": 16,
         "kv_heads": 8, "d": 128, "free": 0.34},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "window", "window", "append", "pages_step",
                     "pages_compact", "pages_copy"])
    kv_heads, d = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if op == "decode":
        dtype = rng.choice(["f16", "bf16"])
        batch = _log(rng, 1, 256)
        most = (1 << 27) // (batch * kv_heads * d)   # keys a row: the longest listed cache
        longest = _log(rng, 1, max(2, min(131072, most)))
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        return {"op": op, "dtype": dtype, "cache": rng.choice([dtype, dtype, "fp8"]),
                "batch": batch, "kv_heads": kv_heads, "group": rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 24]),
                "d": d, "page": page, "longest": longest, "ragged": rng.random() < 0.6,
                "window": window, "sinks": rng.choice([0, 1, 4, 40]) if window else 0}
    if op == "window":
        d = rng.choice([d, 72, 40])
        heads = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 3, 4])
        q_len = _log(rng, 1, 8192)
        start = rng.choice([0, 0, _log(rng, 1, 8192)])
        start = min(start, max(0, (1 << 31) // (heads * group * q_len) - q_len))
        return {"op": op, "dtype": rng.choice(["f16", "bf16"]), "batch": rng.choice([1, 1, 2]),
                "kv_heads": heads, "group": group, "d": d, "q_len": q_len, "start": start,
                "window": _log(rng, 16, 8192), "sinks": rng.choice([0, 1, 4, 4, 100])}
    if op == "append":
        dtype, rows = rng.choice(["f16", "bf16"]), _log(rng, 1, 256)
        return {"op": op, "dtype": dtype, "cache": rng.choice([dtype, "fp8"]), "rows": rows,
                "each": _log(rng, 1, max(2, (1 << 24) // (rows * kv_heads * d))),
                "kv_heads": kv_heads, "group": rng.choice([1, 4]), "d": d, "page": page}
    if op == "pages_step":
        return {"op": op, "rows": _log(rng, 4, 512), "width": _log(rng, 2, 256), "page": page,
                "kv_heads": min(kv_heads, 8), "d": min(d, 128), "forks": rng.choice([1, 2, 4, 5])}
    if op == "pages_compact":
        kv_heads, d, page = min(kv_heads, 8), min(d, 128), min(page, 16)
        return {"op": op, "rows": _log(rng, 1, 128), "width": _log(rng, 2, 64), "page": page,
                "kv_heads": kv_heads, "d": d, "free": rng.choice([0.05, 0.2, 0.5, 0.9])}
    return {"op": op, "count": _log(rng, 1, 1000), "page": min(page, 32),
            "kv_heads": min(kv_heads, 8), "d": min(d, 128)}


# ---- sizes that follow from a case alone -----------------------------------

def _lengths(case):
    """The rows' lengths: the longest first, then spread evenly below it."""
    n, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    return [max(1, math.ceil(longest * (1.0 - (0.6180339887498949 * i) % 1.0))) for i in range(n)]


def _visible(case, length):
    """Keys that the newest token of a row of `length` keys sees."""
    w = case["window"]
    if w <= 0 or w >= length:
        return length
    return w + min(case["sinks"], length - w)


def _pairs(case):
    """Query-key pairs of a windowed prompt."""
    total = 0
    w, s, n = case["window"], case["sinks"], case["q_len"]
    for p in (case["start"] + i for i in range(n)):
        total += p + 1 if p + 1 <= w else w + min(s, p + 1 - w)
    return total


def _ceil(a, b):
    return (a + b - 1) // b


def _normal(gen, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * sigma).to(dtype)


def _pool(gen, shape, cache, dtype):
    """A pool of pages; an 8-bit one holds codes of N(0, 1) values over a scale."""
    if cache == "fp8":
        return _normal(gen, shape, torch.float32, 40.0).clamp_(-448, 448).to(TYPE["fp8"])
    return _normal(gen, shape, TYPE[cache])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- inputs ----------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"decode": _prepare_decode, "window": _prepare_window, "append": _prepare_append,
            "pages_step": _prepare_step, "pages_compact": _prepare_compact,
            "pages_copy": _prepare_copy}[case["op"]](case, gen)


def _prepare_decode(case, gen):
    lengths, ps, b = _lengths(case), case["page"], case["batch"]
    hkv, d, dt = case["kv_heads"], case["d"], TYPE[case["dtype"]]
    pages = [_ceil(n, ps) for n in lengths]
    width, num = max(pages), sum(pages) + 7
    ids = torch.randperm(num, generator=gen, device=DEV).to(torch.int32)
    held = torch.arange(width, device=DEV)[None, :] < _ints(pages)[:, None]
    tables = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
    tables[held] = ids[:sum(pages)]
    fp8 = case["cache"] == "fp8"
    return {"case": case, "q": _normal(gen, (b, hkv * case["group"], d), dt),
            "k": _pool(gen, (num, hkv, ps, d), case["cache"], dt),
            "v": _pool(gen, (num, hkv, ps, d), case["cache"], dt),
            "tables": tables, "lengths": _ints(lengths),
            "scale": d ** -0.5, "k_scale": 1 / 32 if fp8 else 1.0, "v_scale": 1 / 40 if fp8 else 1.0,
            "o": torch.zeros((b, hkv * case["group"], d), dtype=dt, device=DEV),
            "workspace": torch.zeros(WORKSPACE, dtype=torch.uint8, device=DEV)}


def _prepare_window(case, gen):
    b, hkv, d, dt = case["batch"], case["kv_heads"], case["d"], TYPE[case["dtype"]]
    n_kv = case["start"] + case["q_len"]
    q = _normal(gen, (b, hkv * case["group"], case["q_len"], d), dt)
    return {"case": case, "q": q, "k": _normal(gen, (b, hkv, n_kv, d), dt),
            "v": _normal(gen, (b, hkv, n_kv, d), dt), "o": torch.zeros_like(q), "scale": d ** -0.5}


def _prepare_append(case, gen):
    rows, each, hkv, d, ps = (case[x] for x in ("rows", "each", "kv_heads", "d", "page"))
    heads = hkv * (case["group"] + 2)
    # the fused projection's rows: the query heads, then K's, then V's
    qkv = _normal(gen, (rows * each, heads * d), TYPE[case["dtype"]])
    # every row has some tokens already, another count each
    lengths = [37 * i % 50 for i in range(rows)]
    width = _ceil(max(lengths) + each, ps)
    num = rows * width + 3
    tables = torch.randperm(num, generator=gen, device=DEV)[:rows * width].to(torch.int32)
    row = torch.arange(rows, device=DEV, dtype=torch.int32).repeat_interleave(each)
    pos = _ints(lengths).repeat_interleave(each) + torch.arange(each, device=DEV, dtype=torch.int32).repeat(rows)
    fp8 = case["cache"] == "fp8"
    return {"case": case, "qkv": qkv, "row": row, "pos": pos, "tables": tables.reshape(rows, width),
            "k": _pool(gen, (num, hkv, ps, d), case["cache"], None),
            "v": _pool(gen, (num, hkv, ps, d), case["cache"], None),
            "k_scale": 1 / 32 if fp8 else 1.0, "v_scale": 1 / 40 if fp8 else 1.0}


def _held_pages(case, gen, fill):
    """Tables of rows whose page counts run up to the width (a share `fill` of it
    at most), their pages in random places of the pool."""
    rows, width = case["rows"], case["width"]
    pages = [1 + int((width - 1) * fill * ((0.6180339887498949 * (i + 1)) % 1.0)) for i in range(rows)]
    return pages, torch.arange(width, device=DEV)[None, :] < _ints(pages)[:, None]


def _prepare_step(case, gen):
    rows, width, ps, hkv, d = (case[x] for x in ("rows", "width", "page", "kv_heads", "d"))
    pages, held = _held_pages(case, gen, 0.9)
    used = sum(pages)
    num = used + 2 * rows + 11
    ids = torch.randperm(num, generator=gen, device=DEV).to(torch.int32)
    tables = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
    tables[held] = ids[:used]
    refs = torch.zeros(num, dtype=torch.int32, device=DEV)
    refs[ids[:used].long()] = 1
    last = torch.randint(1, ps + 1, (rows,), generator=gen, device=DEV, dtype=torch.int32)
    lengths = (_ints(pages) - 1) * ps + last
    # one row in 16 has ended; each group of `forks` beams goes on from one of its rows
    drop = (torch.rand(rows, generator=gen, device=DEV) < 1 / 16).to(torch.int32)
    i = torch.arange(rows, device=DEV, dtype=torch.int32)
    pick = torch.randint(0, case["forks"], (rows,), generator=gen, device=DEV, dtype=torch.int32)
    src = torch.clamp(i - i % case["forks"] + pick, max=rows - 1)
    return {"case": case, "tables": tables, "lengths": lengths, "refs": refs, "drop": drop, "src": src,
            "need": torch.ones(rows, dtype=torch.int32, device=DEV),
            "k": _normal(gen, (num, hkv, ps, d), torch.bfloat16),
            "v": _normal(gen, (num, hkv, ps, d), torch.bfloat16),
            "freed": {"tables": torch.zeros_like(tables), "lengths": torch.zeros_like(lengths),
                      "refs": torch.zeros_like(refs)},
            "forked": {"tables": torch.zeros_like(tables), "lengths": torch.zeros_like(lengths),
                       "refs": torch.zeros_like(refs)},
            "out": {"tables": torch.zeros_like(tables), "refs": torch.zeros_like(refs),
                    "granted": torch.zeros_like(lengths)},
            "workspace": torch.zeros(WORKSPACE >> 4, dtype=torch.uint8, device=DEV)}


def _prepare_compact(case, gen):
    rows, width, ps, hkv, d = (case[x] for x in ("rows", "width", "page", "kv_heads", "d"))
    pages, held = _held_pages(case, gen, 1.0)
    used = sum(pages)
    num = max(used + 1, int(used / (1.0 - case["free"])))
    ids = torch.randperm(num, generator=gen, device=DEV).to(torch.int32)
    tables = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
    tables[held] = ids[:used]
    refs = torch.zeros(num, dtype=torch.int32, device=DEV)
    refs[ids[:used].long()] = torch.randint(1, 4, (used,), generator=gen, device=DEV, dtype=torch.int32)
    return {"case": case, "tables": tables, "refs": refs,
            "k": _normal(gen, (num, hkv, ps, d), torch.bfloat16),
            "v": _normal(gen, (num, hkv, ps, d), torch.bfloat16),
            "out": {"tables": torch.zeros_like(tables), "refs": torch.zeros_like(refs),
                    "used": torch.zeros(1, dtype=torch.int32, device=DEV)},
            "workspace": torch.zeros(WORKSPACE >> 4, dtype=torch.uint8, device=DEV)}


def _prepare_copy(case, gen):
    n, ps, hkv, d = (case[x] for x in ("count", "page", "kv_heads", "d"))
    num = 2 * n + 5
    ids = torch.randperm(num, generator=gen, device=DEV).to(torch.int32)
    return {"case": case, "src": ids[:n].clone(), "dst": ids[n:2 * n].clone(),
            "k": _normal(gen, (num, hkv, ps, d), torch.bfloat16),
            "v": _normal(gen, (num, hkv, ps, d), torch.bfloat16)}


# ---- one pass --------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"decode": _own_decode, "window": _own_window, "append": _own_append,
                "pages_step": _own_step, "pages_compact": _own_compact,
                "pages_copy": _own_copy}[op](state)
    return {"decode": _plain_decode, "window": _plain_window, "append": _plain_append,
            "pages_step": _plain_step, "pages_compact": _plain_compact,
            "pages_copy": _plain_copy}[op](state)


def _plain_softmax(s, dim):
    """exp(s - max) over its sum; a masked score is -inf, a row of them gives zeros."""
    top = s.amax(dim, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _plain_decode(st):
    case, length = st["case"], st["lengths"].long()[:, None]
    longest, w, sinks, ps = case["longest"], case["window"], case["sinks"], case["page"]
    if 0 < w < longest:   # the positions a row sees: the first `sinks`, then the window
        first = torch.clamp(length - w, min=0)
        at = torch.arange(sinks + w, device=DEV)[None, :]
        pos = torch.where(at < sinks, at, first + at - sinks)
        seen = torch.where(at < sinks, at < first, pos < length)
    else:
        pos = torch.arange(longest, device=DEV)[None, :].expand(length.shape[0], longest)
        seen = pos < length
    pos = torch.where(seen, pos, torch.zeros_like(pos))
    page, slot = torch.gather(st["tables"].long(), 1, pos // ps), pos % ps
    if case["cache"] == "fp8":
        k = st["k"].view(torch.uint8)[page, :, slot].view(TYPE["fp8"]).float() * st["k_scale"]
        v = st["v"].view(torch.uint8)[page, :, slot].view(TYPE["fp8"]).float() * st["v_scale"]
    else:
        k, v = st["k"][page, :, slot].float(), st["v"][page, :, slot].float()
    b, hkv, d = length.shape[0], case["kv_heads"], case["d"]
    k, v = k.permute(0, 2, 1, 3).contiguous(), v.permute(0, 2, 1, 3).contiguous()   # [b, hkv, keys, d]
    q = st["q"].float().reshape(b, hkv, case["group"], d).transpose(2, 3).contiguous()
    s = torch.matmul(k, q) * st["scale"]                                            # [b, hkv, keys, group]
    s = torch.where(seen[:, None, :, None], s, torch.full_like(s, -math.inf))
    p = _plain_softmax(s, 2)
    o = torch.matmul(p.transpose(2, 3).contiguous(), v)
    return o.reshape(st["q"].shape).to(st["q"].dtype)


def _plain_window(st):
    case = st["case"]
    b, hkv, g, d, n = (case[x] for x in ("batch", "kv_heads", "group", "d", "q_len"))
    q = st["q"].float().reshape(b, hkv, g * n, d)
    k, v = st["k"].float().transpose(2, 3).contiguous(), st["v"].float()
    s = (torch.matmul(q, k) * st["scale"]).reshape(b, hkv, g, n, -1)
    pos = case["start"] + torch.arange(n, device=DEV)[:, None]
    key = torch.arange(s.shape[-1], device=DEV)[None, :]
    seen = (key <= pos) & ((key > pos - case["window"]) | (key < case["sinks"]))
    s.masked_fill_(~seen, -math.inf)
    p = _plain_softmax(s, 4)
    o = torch.matmul(p.reshape(b, hkv, g * n, -1), v)
    return o.reshape(st["q"].shape).to(st["q"].dtype)


def _kv_of(st):
    case = st["case"]
    d, hkv, qs = case["d"], case["kv_heads"], case["group"] * case["kv_heads"]
    k = st["qkv"][:, qs * d:(qs + hkv) * d]
    v = st["qkv"][:, (qs + hkv) * d:]
    return k, v


def _plain_append(st):
    case = st["case"]
    page, slot = st["pos"].long() // case["page"], st["pos"].long() % case["page"]
    page = st["tables"].long()[st["row"].long(), page]
    k, v = (x.reshape(-1, case["kv_heads"], case["d"]) for x in _kv_of(st))
    if case["cache"] == "fp8":
        k = (k.float() / st["k_scale"]).clamp(-448, 448).to(TYPE["fp8"]).view(torch.uint8)
        v = (v.float() / st["v_scale"]).clamp(-448, 448).to(TYPE["fp8"]).view(torch.uint8)
        st["k"].view(torch.uint8)[page, :, slot] = k
        st["v"].view(torch.uint8)[page, :, slot] = v
    else:
        st["k"][page, :, slot] = k
        st["v"][page, :, slot] = v
    return {"k": st["k"], "v": st["v"]}


def _plain_count(refs, entries, keep, sign):
    """refs with `sign` added at each page of `entries` where `keep` holds."""
    change = torch.where(keep, sign, 0).to(torch.int32).reshape(-1)
    return refs.index_add(0, entries.clamp(min=0).long().reshape(-1), change)


def _plain_step(st):
    ps, width = st["case"]["page"], st["case"]["width"]
    # drop
    gone = (st["drop"] != 0)[:, None]
    refs = _plain_count(st["refs"], st["tables"], gone & (st["tables"] >= 0), -1)
    tables = torch.where(gone, -1, st["tables"])
    lengths = torch.where(gone[:, 0], 0, st["lengths"])
    # fork
    new = tables[st["src"].long()]
    refs = _plain_count(refs, tables, tables >= 0, -1)
    refs = _plain_count(refs, new, new >= 0, 1)
    lengths = lengths[st["src"].long()]
    # reserve
    first, last = (lengths // ps)[:, None], ((lengths + st["need"] - 1) // ps)[:, None]
    e = torch.arange(width, device=DEV)[None, :]
    wanted = (e >= first) & (e <= last)
    shared = torch.where(new >= 0, refs[new.clamp(min=0).long()], 0)
    fresh = wanted & (shared != 1)
    free = torch.nonzero(refs <= 0).reshape(-1)
    fits = lengths + st["need"] <= width * ps
    demand = torch.where(fits, fresh.sum(1), 0)
    granted = fits & (torch.cumsum(demand, 0) <= free.numel())
    fresh = fresh & granted[:, None]
    rank = torch.cumsum(fresh.reshape(-1).long(), 0).reshape(fresh.shape) - 1
    out = torch.where(fresh, free[rank.clamp(min=0, max=free.numel() - 1)], new.long()).to(torch.int32)
    left = fresh & (shared > 1)
    copied = left & (e == first) & ((lengths % ps)[:, None] != 0)
    src, dst = new[copied].long(), out[copied].long()
    st["k"][dst] = st["k"][src]
    st["v"][dst] = st["v"][src]
    refs = _plain_count(refs, new, left, -1)
    refs = refs.index_add(0, out.clamp(min=0).long().reshape(-1), fresh.to(torch.int32).reshape(-1))
    return {"tables": out, "lengths": lengths, "refs": refs, "granted": granted.to(torch.int32),
            "k": st["k"], "v": st["v"]}


def _plain_compact(st):
    used = st["refs"] > 0
    count = used.sum()
    at = torch.arange(used.shape[0], device=DEV)
    hole, mover = torch.nonzero(~used & (at < count)).reshape(-1), torch.nonzero(used & (at >= count)).reshape(-1)
    to = at.clone()
    to[mover] = hole
    refs = torch.where(used, st["refs"], 0)
    refs[hole] = refs[mover]
    refs[mover] = 0
    st["k"][hole] = st["k"][mover]
    st["v"][hole] = st["v"][mover]
    tables = torch.where(st["tables"] >= 0, to[st["tables"].clamp(min=0).long()].to(torch.int32), st["tables"])
    return {"tables": tables, "refs": refs, "used": count.to(torch.int32).reshape(1),
            "k": st["k"], "v": st["v"]}


def _plain_copy(st):
    src, dst = st["src"].long(), st["dst"].long()
    st["k"][dst] = st["k"][src]
    st["v"][dst] = st["v"][src]
    return {"k": st["k"], "v": st["v"]}


def _hip():
    from sile_amd import _abi
    return _abi


def _code(hip, name):
    return {"f16": hip.F16, "bf16": hip.BF16, "fp8": hip.F8E4M3}[name]


def _own_decode(st):
    hip, case = _hip(), st["case"]
    hq, d = case["kv_heads"] * case["group"], case["d"]
    hip.paged_attn_decode(_code(hip, case["dtype"]), _code(hip, case["cache"]), case["batch"], hq,
                          case["kv_heads"], d, st["q"].data_ptr(), hq * d, st["k"].data_ptr(),
                          st["v"].data_ptr(), st["k"].shape[0], case["page"],
                          case["kv_heads"] * case["page"] * d, st["tables"].data_ptr(),
                          st["tables"].shape[1], st["lengths"].data_ptr(), st["o"].data_ptr(), hq * d,
                          st["scale"], st["k_scale"], st["v_scale"], case["window"], case["sinks"],
                          st["workspace"].data_ptr(), st["workspace"].numel())
    return st["o"]


def _own_window(st):
    hip, case = _hip(), st["case"]
    hip.flash_attn_window_fwd(_code(hip, case["dtype"]), case["batch"],
                              case["kv_heads"] * case["group"], case["kv_heads"], case["q_len"],
                              st["k"].shape[2], case["d"], st["q"].data_ptr(), st["k"].data_ptr(),
                              st["v"].data_ptr(), st["o"].data_ptr(), st["scale"], case["start"],
                              case["window"], case["sinks"])
    return st["o"]


def _own_append(st):
    hip, case = _hip(), st["case"]
    k, v = _kv_of(st)
    hip.kv_append(_code(hip, case["dtype"]), _code(hip, case["cache"]), k.shape[0],
                  case["kv_heads"], case["d"], k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                  st["row"].data_ptr(), st["pos"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(),
                  st["k"].shape[0], case["page"], case["kv_heads"] * case["page"] * case["d"],
                  st["tables"].data_ptr(), case["rows"], st["tables"].shape[1], st["k_scale"],
                  st["v_scale"])
    return {"k": st["k"], "v": st["v"]}


def _pools(st):
    bytes_ = st["k"][0].numel() * st["k"].element_size()
    return [st["k"].data_ptr(), st["v"].data_ptr()], bytes_, bytes_


def _own_step(st):
    hip, case = _hip(), st["case"]
    rows, width, num = case["rows"], case["width"], st["refs"].shape[0]
    freed, forked, out = st["freed"], st["forked"], st["out"]
    hip.kv_free(rows, width, st["drop"].data_ptr(), st["tables"].data_ptr(),
                freed["tables"].data_ptr(), st["lengths"].data_ptr(), freed["lengths"].data_ptr(),
                num, st["refs"].data_ptr(), freed["refs"].data_ptr())
    hip.kv_fork(rows, rows, width, st["src"].data_ptr(), freed["tables"].data_ptr(),
                forked["tables"].data_ptr(), freed["lengths"].data_ptr(), forked["lengths"].data_ptr(),
                num, freed["refs"].data_ptr(), forked["refs"].data_ptr())
    hip.kv_reserve(rows, width, case["page"], forked["lengths"].data_ptr(), st["need"].data_ptr(),
                   forked["tables"].data_ptr(), out["tables"].data_ptr(), num,
                   forked["refs"].data_ptr(), out["refs"].data_ptr(), out["granted"].data_ptr(),
                   *_pools(st), st["workspace"].data_ptr(), st["workspace"].numel())
    return {"tables": out["tables"], "lengths": forked["lengths"], "refs": out["refs"],
            "granted": out["granted"], "k": st["k"], "v": st["v"]}


def _own_compact(st):
    hip, case, out = _hip(), st["case"], st["out"]
    hip.kv_compact(case["rows"], case["width"], st["tables"].data_ptr(), out["tables"].data_ptr(),
                   st["refs"].shape[0], st["refs"].data_ptr(), out["refs"].data_ptr(),
                   out["used"].data_ptr(), *_pools(st), st["workspace"].data_ptr(),
                   st["workspace"].numel())
    return {"tables": out["tables"], "refs": out["refs"], "used": out["used"], "k": st["k"], "v": st["v"]}


def _own_copy(st):
    hip = _hip()
    hip.kv_copy_pages(*_pools(st), st["k"].shape[0], st["case"]["count"], st["src"].data_ptr(),
                      st["dst"].data_ptr())
    return {"k": st["k"], "v": st["v"]}


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    op, d = case["op"], case["d"]
    hkv = case["kv_heads"]
    if op == "decode":
        keys = sum(_visible(case, n) for n in _lengths(case))
        q = case["batch"] * hkv * case["group"] * d * SIZE[case["dtype"]]
        return {"bytes": 2 * keys * hkv * d * SIZE[case["cache"]] + 2 * q,
                "flops": 4 * keys * hkv * case["group"] * d}
    if op == "window":
        heads, n_kv = case["batch"] * hkv, case["start"] + case["q_len"]
        seen = min(n_kv, case["q_len"] + case["window"] + case["sinks"])
        return {"bytes": 2 * 2 * heads * d * (case["group"] * case["q_len"] + seen),
                "flops": 4 * d * heads * case["group"] * _pairs(case)}
    if op == "append":
        values = 2 * case["rows"] * case["each"] * hkv * d
        return {"bytes": values * (SIZE[case["dtype"]] + SIZE[case["cache"]]), "flops": values}
    page = 2 * 2 * hkv * case["page"] * d   # K's and V's page, bytes
    if op == "pages_copy":
        return {"bytes": 2 * case["count"] * page, "flops": 0}
    pages = sum(_held_counts(case, 0.9 if op == "pages_step" else 1.0))
    entries = 4 * case["rows"] * case["width"]
    if op == "pages_step":
        # a row copies its part-filled last page if another of its group goes on from
        # the same row
        copies = case["rows"] * (1 - (1 - 1 / case["forks"]) ** (case["forks"] - 1))
        return {"bytes": int(copies * 2 * page) + 2 * entries + 8 * pages, "flops": 2 * case["rows"] * case["width"]}
    num = max(pages + 1, int(pages / (1.0 - case["free"])))
    moved = pages * (num - pages) / num
    return {"bytes": int(moved * 2 * page) + 2 * entries + 8 * num, "flops": 2 * num}


def _held_counts(case, fill):
    return [1 + int((case["width"] - 1) * fill * ((0.6180339887498949 * (i + 1)) % 1.0))
            for i in range(case["rows"])]


# ---- the definitions in 64 bits ----------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"decode": _exact_decode, "window": _exact_window, "append": _exact_append,
            "pages_step": _exact_step, "pages_compact": _exact_compact,
            "pages_copy": _exact_copy}[case["op"]](case, st)


def _exact_decode(case, st):
    if sum(_visible(case, n) for n in _lengths(case)) * case["kv_heads"] * case["d"] > 1 << 28:
        return None
    o = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    hkv, g, d, ps = case["kv_heads"], case["group"], case["d"], case["page"]
    for b, n in enumerate(_lengths(case)):
        ids = st["tables"][b, :_ceil(n, ps)].long()
        k, v = (st[x][ids].double().transpose(0, 1).reshape(hkv, -1, d)[:, :n] for x in ("k", "v"))
        if 0 < case["window"] < n:
            lo = n - case["window"]
            keep = torch.cat([torch.arange(min(case["sinks"], lo), device=DEV),
                              torch.arange(lo, n, device=DEV)])
            k, v = k[:, keep], v[:, keep]
        q = st["q"][b].double().reshape(hkv, g, d)
        for h in range(hkv):
            w = torch.softmax((q[h] @ k[h].t().contiguous()) * (st["k_scale"] * st["scale"]), 1)
            o[b, h * g:(h + 1) * g] = w @ v[h] * st["v_scale"]
    return o


def _exact_window(case, st):
    n, g, start = case["q_len"], case["group"], case["start"]
    o = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    n_kv = start + n
    for b in range(case["batch"]):
        for h in range(case["kv_heads"] * g):
            q, k, v = (t.double() for t in (st["q"][b, h], st["k"][b, h // g], st["v"][b, h // g]))
            for at in range(0, n, 2048):
                some = torch.arange(at, min(n, at + 2048), device=DEV)
                lo = max(0, start + at - case["window"] + 1)
                lo = 0 if lo <= case["sinks"] else lo
                hi = start + int(some[-1]) + 1
                key = torch.arange(lo, hi, device=DEV)
                if lo > 0:
                    key = torch.cat([torch.arange(case["sinks"], device=DEV), key])
                age = (some[:, None] + start) - key[None, :]
                s = (q[some] @ k[key].t().contiguous()) * st["scale"]
                s[(age < 0) | ((age >= case["window"]) & (key[None, :] >= case["sinks"]))] = -math.inf
                o[b, h, some] = torch.softmax(s, 1) @ v[key]
    return o


def _exact_append(case, st):
    d, hkv, ps = case["d"], case["kv_heads"], case["page"]
    x = st["qkv"].double().reshape(-1, hkv * (case["group"] + 2), d)
    flat = st["tables"].long()[st["row"].long(), st["pos"].long().div(ps, rounding_mode="floor")] * ps
    flat = flat + st["pos"].long().remainder(ps)
    out = {}
    for name, at in (("k", case["group"] * hkv), ("v", (case["group"] + 1) * hkv)):
        pool = st[name].double().transpose(1, 2).contiguous()     # [page, slot, head, d]
        pool.view(-1, hkv, d)[flat] = (x[:, at:at + hkv] / st[name + "_scale"]).clamp(-448, 448) \
            if case["cache"] == "fp8" else x[:, at:at + hkv]
        out[name] = pool.transpose(1, 2).contiguous()
    return out


def _exact_step(case, st):
    ps, width, rows = case["page"], case["width"], case["rows"]
    tables, lengths, refs = (st[x].tolist() for x in ("tables", "lengths", "refs"))
    for i, gone in enumerate(st["drop"].tolist()):
        if gone:
            for p in tables[i]:
                if p >= 0:
                    refs[p] -= 1
            tables[i], lengths[i] = [-1] * width, 0
    new = [list(tables[s]) for s in st["src"].tolist()]
    lengths = [lengths[s] for s in st["src"].tolist()]
    for table, sign in ((tables, -1), (new, 1)):
        for row in table:
            for p in row:
                if p >= 0:
                    refs[p] += sign
    free = [p for p, r in enumerate(refs) if r <= 0]
    before, granted, copies = list(refs), [], []
    taken = full = 0
    for i in range(rows):
        n, need = lengths[i], 1
        if n + need > width * ps:
            granted.append(0)
            continue
        want = [e for e in range(n // ps, (n + need - 1) // ps + 1)
                if new[i][e] < 0 or before[new[i][e]] != 1]
        full += len(want)
        granted.append(int(full <= len(free)))
        for e in want if granted[-1] else []:
            old, p = new[i][e], free[taken]
            taken += 1
            if old >= 0 and before[old] > 1:
                refs[old] -= 1
                if e == n // ps and n % ps:
                    copies.append((old, p))
            refs[p] += 1
            new[i][e] = p
    k, v = st["k"].double(), st["v"].double()
    for pool in (k, v):
        if copies:
            a, b = (torch.tensor(x, device=DEV) for x in zip(*copies))
            pool[b] = pool[a]
    return {"tables": _ints(new), "lengths": _ints(lengths), "refs": _ints(refs),
            "granted": _ints(granted), "k": k, "v": v}


def _exact_compact(case, st):
    refs, tables = st["refs"].tolist(), st["tables"].tolist()
    used = [p for p, r in enumerate(refs) if r > 0]
    holes = [p for p, r in enumerate(refs) if r <= 0 and p < len(used)]
    moves = dict(zip([p for p in used if p >= len(used)], holes))
    to = [0] * len(refs)
    for p in used:
        to[moves.get(p, p)] = refs[p]
    k, v = st["k"].double(), st["v"].double()
    if moves:
        a = torch.tensor(list(moves), device=DEV)
        b = torch.tensor(list(moves.values()), device=DEV)
        k[b], v[b] = k[a], v[a]
    return {"tables": _ints([[moves.get(p, p) for p in row] for row in tables]), "refs": _ints(to),
            "used": _ints([len(used)]), "k": k, "v": v}


def _exact_copy(case, st):
    out = {}
    for name in ("k", "v"):
        pool = st[name].double()
        for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
            pool[b] = st[name][a].double()
        out[name] = pool
    return out
