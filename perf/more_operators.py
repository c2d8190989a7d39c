"""The workloads of a serving step over prompts in pieces and single tokens at once:
the step's token list, the normalisation in front of a projection, rotary positions
on the way into the paged cache, the attention of the new tokens over the pages, and
the log probabilities of what was answered.

Each case is one pass of one operator on operands that are resident on the GPU.
With `own` false, run() computes it in elementary torch operations in 32 bits;
with `own` true it makes the calls of sile_amd a serving program makes.

Layouts: pages [num_pages, kv_heads, page, d]; page tables int32 [rows, width];
tokens in a row each, [tokens, (q_heads + 2 kv_heads) d] out of a fused projection,
those of one sequence together, in order.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
        "fp8": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}
TOP = 448.0           # the largest e4m3 value
LOWEST = 2.0 ** -100  # a group's maximum counts as at least this


def listed():
    return [
        # a step's token list: 256 conversations, every eighth with a piece of a prompt
        {"name": "slots_256", "op": "slots", "rows": 256, "piece": 300, "every": 8, "spare": 100,
         "refused": 0.05},
        # the list of a large batch of prompts
        {"name": "slots_4000x65", "op": "slots", "rows": 4000, "piece": 65, "every": 1, "spare": 0,
         "refused": 0.0},
        # the norm before a projection, one token of each of 64 conversations
        {"name": "norm_bf16_64x8192", "op": "norm", "dtype": "bf16", "out": "bf16", "rows": 64,
         "cols": 8192, "residual": True, "weight": True, "group": 0, "pad": 0},
        # prompts' tokens, made ready for an 8-bit projection, a scale for each 128 columns
        {"name": "norm_bf16_fp8_8000x8192", "op": "norm", "dtype": "bf16", "out": "fp8",
         "rows": 8000, "cols": 8192, "residual": True, "weight": True, "group": 128, "pad": 0},
        # one token of each of 64 conversations, rotated and into the cache
        {"name": "rope_append_bf16_64", "op": "rope_append", "dtype": "bf16", "cache": "bf16",
         "layout": "half", "rows": 64, "each": 1, "start": 20000, "kv_heads": 8, "group": 4,
         "d": 128, "rot": 128, "base": 500000.0, "factor": 8.0, "page": 16},
        # two prompts of 8191 tokens into an 8-bit cache
        {"name": "rope_append_fp8_2x8191", "op": "rope_append", "dtype": "bf16", "cache": "fp8",
         "layout": "half", "rows": 2, "each": 8191, "start": 100000, "kv_heads": 8, "group": 4,
         "d": 128, "rot": 128, "base": 500000.0, "factor": 8.0, "page": 32},
        # a quarter of each head rotated, pairs side by side, keys kept contiguous
        {"name": "rope_f16_5000_rot32", "op": "rope", "dtype": "f16", "layout": "pairs", "rows": 1,
         "each": 5000, "start": 0, "kv_heads": 32, "group": 1, "d": 128, "rot": 32,
         "base": 10000.0, "factor": 1.0},
        # drafts of up to 8 tokens looked at in one step, conversations of all lengths to 8192
        {"name": "chunk_bf16_32x8_8192", "op": "chunk", "dtype": "bf16", "cache": "bf16",
         "rows": 32, "new": 8, "singles": 0, "longest": 8192, "ragged": True, "kv_heads": 8,
         "group": 4, "d": 128, "page": 16, "window": 0, "sinks": 0, "pad": 0},
        # a long prompt's last piece: 2048 tokens behind 30000 cached ones
        {"name": "chunk_f16_2048_32048", "op": "chunk", "dtype": "f16", "cache": "f16",
         "rows": 1, "new": 2048, "singles": 0, "longest": 32048, "ragged": False, "kv_heads": 8,
         "group": 4, "d": 128, "page": 64, "window": 0, "sinks": 0, "pad": 0},
        # a mixed step over an 8-bit cache: pieces of three prompts beside 48 single tokens
        {"name": "chunk_bf16_fp8_3x700_48", "op": "chunk", "dtype": "bf16", "cache": "fp8",
         "rows": 3, "new": 700, "singles": 48, "longest": 4000, "ragged": True, "kv_heads": 8,
         "group": 4, "d": 128, "page": 32, "window": 0, "sinks": 0, "pad": 9},
        # the answers of one step: 64 rows of a large vocabulary, 20 alternatives
        {"name": "logprobs_bf16_64x131072_k20", "op": "logprobs", "dtype": "bf16", "rows": 64,
         "cols": 131072, "top": 20, "scale": 1.0, "masked": 0.0, "pad": 0},
        # a scored prompt: 2000 rows of a vocabulary of no round size, at a temperature
        {"name": "logprobs_f32_2000x32001_k5", "op": "logprobs", "dtype": "f32", "rows": 2000,
         "cols": 32001, "top": 5, "scale": 1.25, "masked": 0.3, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["slots", "norm", "norm", "rope", "rope_append", "rope_append", "chunk",
                     "chunk", "chunk", "logprobs", "logprobs"])
    kv_heads, group = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([1, 2, 3, 4, 4, 5, 8])
    d, page = rng.choice([64, 80, 96, 128, 128, 128, 256]), rng.choice([8, 16, 16, 32, 64, 128])
    if op == "slots":
        rows = _log(rng, 1, 8192)
        return {"op": op, "rows": rows, "piece": _log(rng, 1, max(2, 260000 // rows)),
                "every": rng.choice([1, 2, 8, 30]), "spare": rng.choice([0, 1, 500]),
                "refused": rng.choice([0.0, 0.1])}
    if op == "norm":
        cols = rng.choice([_log(rng, 1, 16384), 16 * _log(rng, 4, 1024), 128 * _log(rng, 1, 128)])
        dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
        out = rng.choice([dtype, "fp8"])
        group = rng.choice([0, cols, 128 if cols % 128 == 0 else cols,
                            64 if cols % 64 == 0 else cols]) if out == "fp8" else 0
        return {"op": op, "dtype": dtype, "out": out, "rows": _log(rng, 1, max(2, min(1 << 16, (1 << 25) // cols))),
                "cols": cols, "residual": rng.random() < 0.7, "weight": rng.random() < 0.9,
                "group": group, "pad": rng.choice([0, 0, 8, 1])}
    if op in ("rope", "rope_append"):
        d = rng.choice([d, 72]) if op == "rope" else d
        rows = _log(rng, 1, 256)
        rot = rng.choice([d, d, d // 2, d // 4])
        case = {"op": op, "dtype": rng.choice(["f16", "bf16"] + (["f32"] if op == "rope" else [])),
                "layout": rng.choice(["half", "pairs"]), "rows": rows,
                "each": _log(rng, 1, max(2, (1 << 24) // (rows * kv_heads * (group + 2) * d))),
                "start": rng.choice([0, 1000, 200000]), "kv_heads": kv_heads, "group": group,
                "d": d, "rot": rot - rot % 2, "base": rng.choice([10000.0, 500000.0]),
                "factor": rng.choice([1.0, 4.0, 8.0])}
        if op == "rope_append":
            case["cache"], case["page"] = rng.choice([case["dtype"], "fp8"]), page
        return case
    if op == "chunk":
        dtype = rng.choice(["f16", "bf16"])
        rows, singles = _log(rng, 1, 32), rng.choice([0, 0, 1, 20, 60])
        longest = _log(rng, 1, max(2, min(65536, (1 << 26) // ((rows + singles) * kv_heads * d))))
        # (query-key pairs x dims a head: below those of the long prompt's piece)
        new = _log(rng, 1, max(2, min(2048, (1 << 37) // (rows * kv_heads * group * d * longest))))
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        return {"op": op, "dtype": dtype, "cache": rng.choice([dtype, dtype, "fp8"]), "rows": rows,
                "new": new, "singles": singles, "longest": longest, "ragged": rng.random() < 0.7,
                "kv_heads": kv_heads, "group": group, "d": d, "page": page, "window": window,
                "sinks": rng.choice([0, 1, 4, 40]) if window else 0, "pad": rng.choice([0, 0, 5])}
    cols = rng.choice([_log(rng, 1, 262144), 8 * _log(rng, 100, 20000)])
    return {"op": op, "dtype": rng.choice(["f16", "bf16", "f32"]),
            "rows": _log(rng, 1, max(2, min(1 << 14, (1 << 25) // cols))), "cols": cols,
            "top": rng.choice([0, 1, 5, 20, 50]), "scale": rng.choice([1.0, 0.7, 2.0]),
            "masked": rng.choice([0.0, 0.0, 0.5, 0.99]), "pad": rng.choice([0, 0, 8, 3])}


# ---- sizes that follow from a case alone -----------------------------------

def _ceil(a, b):
    return (a + b - 1) // b


def _spread(i):
    """A share in (0, 1]: 1 first, then all over the range."""
    return 1.0 - (0.6180339887498949 * i) % 1.0


def _pieces(case):
    """New tokens of the rows of a step's list: one each, or a piece of a prompt."""
    return [max(1, math.ceil(case["piece"] * _spread(i))) if i % case["every"] == 0 else 1
            for i in range(case["rows"])]


def _chunks(case):
    """(new tokens, length with them) of the rows of a step's attention."""
    out = []
    for i in range(case["rows"] + case["singles"]):
        share = _spread(i) if case["ragged"] else 1.0
        new = max(1, math.ceil(case["new"] * _spread(i + 3))) if case["ragged"] else case["new"]
        new = 1 if i >= case["rows"] else min(new, case["longest"])
        out.append((new, max(new, math.ceil(case["longest"] * share))))
    return out


def _pairs(case, new, length):
    """Query-key pairs of a row."""
    w, s, total = case["window"], case["sinks"], 0
    if w <= 0:
        return new * (length - new) + new * (new + 1) // 2
    for p in range(length - new, length):
        total += p + 1 if p + 1 <= w else w + min(s, p + 1 - w)
    return total


def _normal(gen, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * sigma).to(dtype)


def _pool(gen, shape, cache):
    """A pool of pages; an 8-bit one holds codes of N(0, 1) values over a scale."""
    if cache == "fp8":
        return _normal(gen, shape, torch.float32, 40.0).clamp_(-TOP, TOP).to(TYPE["fp8"])
    return _normal(gen, shape, TYPE[cache])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _turns(case):
    """Turns a position of each pair; with a factor, pairs that turn less than 4 times
    over 8192 positions are slowed down by it, gradually from there to once."""
    out = []
    for j in range(case["rot"] // 2):
        t = case["base"] ** (-2.0 * j / case["rot"]) / (2.0 * math.pi)
        w = min(max((8192 * t - 1.0) / 3.0, 0.0), 1.0)
        out.append(t * (w + (1.0 - w) / case["factor"]))
    return out


# ---- inputs ----------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"slots": _prepare_slots, "norm": _prepare_norm, "rope": _prepare_rope,
            "rope_append": _prepare_rope, "chunk": _prepare_chunk,
            "logprobs": _prepare_logprobs}[case["op"]](case, gen)


def _prepare_slots(case, gen):
    rows, need = case["rows"], _pieces(case)
    tokens = sum(need) + case["spare"]
    lengths = torch.randint(0, 8192, (rows,), generator=gen, device=DEV, dtype=torch.int32)
    granted = (torch.rand(rows, generator=gen, device=DEV) >= case["refused"]).to(torch.int32)
    empty = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)   # noqa: E731
    return {"case": case, "tokens": tokens, "lengths": lengths, "need": _ints(need),
            "granted": granted, "starts": empty(rows + 1), "rows": empty(tokens),
            "positions": empty(tokens), "lengths_out": empty(rows)}


def _prepare_norm(case, gen):
    rows, cols, dt = case["rows"], case["cols"], TYPE[case["dtype"]]
    ld = cols + case["pad"]
    # the residual stream has grown over the layers and has a few large channels
    channel = 1.0 + 20.0 * (torch.rand(ld, generator=gen, device=DEV) > 0.998)
    st = {"case": case, "ld": ld, "eps": 1e-5, "x": _normal(gen, (rows, ld), dt),
          "residual": (torch.randn((rows, ld), generator=gen, device=DEV) * channel).to(dt)
          if case["residual"] else None,
          "weight": (1.0 + 0.2 * torch.randn(cols, generator=gen, device=DEV)).to(dt)
          if case["weight"] else None,
          "sum": torch.zeros((rows, cols), dtype=dt, device=DEV) if case["residual"] else None,
          "y": torch.zeros((rows, cols), dtype=TYPE[case["out"]], device=DEV),
          "scale": 1 / 32, "scales": None}
    if case["group"]:
        st["scales"] = torch.zeros((rows, cols // case["group"]), dtype=torch.float32, device=DEV)
    return st


def _prepare_rope(case, gen):
    rows, each, hkv, d = (case[x] for x in ("rows", "each", "kv_heads", "d"))
    n, hq, dt = rows * each, hkv * case["group"], TYPE[case["dtype"]]
    # every row has some tokens already, another count each
    lengths = [case["start"] + 37 * i % 50 for i in range(rows)]
    positions = _ints(lengths).repeat_interleave(each) + torch.arange(each, device=DEV, dtype=torch.int32).repeat(rows)
    st = {"case": case, "n": n, "hq": hq, "qkv": _normal(gen, (n, (hq + 2 * hkv) * d), dt),
          "positions": positions, "turns": torch.tensor(_turns(case), dtype=torch.float64, device=DEV),
          "magnitude": 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0,
          "q": torch.zeros((n, hq * d), dtype=dt, device=DEV)}
    if case["op"] == "rope":
        st["k"] = torch.zeros((n, hkv * d), dtype=dt, device=DEV)
        return st
    ps = case["page"]
    # (of the tokens before these only the last page is held here)
    width, used = _ceil(max(lengths) + each, ps), _ceil(50 + each, ps) + 1
    first = _ints(lengths) // ps
    num = rows * used + 3
    ids = torch.randperm(num, generator=gen, device=DEV)[:rows * used].to(torch.int32).reshape(rows, used)
    tables = torch.full((rows, width + used), -1, dtype=torch.int32, device=DEV)
    tables.scatter_(1, first[:, None].long() + torch.arange(used, device=DEV)[None, :], ids)
    st["rows"] = torch.arange(rows, device=DEV, dtype=torch.int32).repeat_interleave(each)
    st["tables"] = tables[:, :width].contiguous()
    st["k"] = _pool(gen, (num, hkv, ps, d), case["cache"])
    st["v"] = _pool(gen, (num, hkv, ps, d), case["cache"])
    fp8 = case["cache"] == "fp8"
    st["k_scale"], st["v_scale"] = (1 / 32, 1 / 40) if fp8 else (1.0, 1.0)
    return st


def _prepare_chunk(case, gen):
    rows, ps, hkv, d, dt = _chunks(case), case["page"], case["kv_heads"], case["d"], TYPE[case["dtype"]]
    hq = hkv * case["group"]
    pages = [_ceil(length, ps) for _, length in rows]
    width, num = max(pages), sum(pages) + 7
    ids = torch.randperm(num, generator=gen, device=DEV).to(torch.int32)
    held = torch.arange(width, device=DEV)[None, :] < _ints(pages)[:, None]
    tables = torch.full((len(rows), width), -1, dtype=torch.int32, device=DEV)
    tables[held] = ids[:sum(pages)]
    starts = [0]
    for new, _ in rows:
        starts.append(starts[-1] + new)
    n = starts[-1] + case["pad"]
    fp8 = case["cache"] == "fp8"
    st = {"case": case, "n": n, "hq": hq, "qkv": _normal(gen, (n, (hq + 2 * hkv) * d), dt),
          "k": _pool(gen, (num, hkv, ps, d), case["cache"]),
          "v": _pool(gen, (num, hkv, ps, d), case["cache"]), "tables": tables,
          "starts": _ints(starts), "lengths": _ints([length for _, length in rows]),
          "scale": d ** -0.5, "k_scale": 1 / 32 if fp8 else 1.0, "v_scale": 1 / 40 if fp8 else 1.0,
          "o": torch.zeros((n, hq, d), dtype=dt, device=DEV), "workspace": None}
    if own:
        bytes_ = _hip().paged_attn_chunk_workspace(len(rows), n, hq, hkv, d)
        st["workspace"] = torch.zeros(bytes_, dtype=torch.uint8, device=DEV)
    return st


def _prepare_logprobs(case, gen):
    rows, cols, top = case["rows"], case["cols"], case["top"]
    ld = cols + case["pad"]
    # a few tokens stand out of each row
    x = torch.randn((rows, ld), generator=gen, device=DEV) * 2.0
    some = torch.randint(0, cols, (rows, 8), generator=gen, device=DEV)
    x.scatter_add_(1, some, 6.0 + 3.0 * torch.randn((rows, 8), generator=gen, device=DEV))
    if case["masked"]:
        x.masked_fill_(torch.rand((rows, ld), generator=gen, device=DEV) < case["masked"], -math.inf)
        x.scatter_(1, some[:, :1], 8.0)   # (the first of them is never masked)
    st = {"case": case, "ld": ld, "x": x.to(TYPE[case["dtype"]]),
          "targets": some[:, 0].to(torch.int32).contiguous(),
          "logp": torch.zeros(rows, dtype=torch.float32, device=DEV),
          "entropy": torch.zeros(rows, dtype=torch.float32, device=DEV),
          "top_logp": torch.zeros((rows, top), dtype=torch.float32, device=DEV),
          "top_ids": torch.zeros((rows, top), dtype=torch.int32, device=DEV), "workspace": None}
    if own:
        bytes_ = _hip().logprobs_workspace(rows, cols, top)
        st["workspace"] = torch.zeros(bytes_, dtype=torch.uint8, device=DEV)
    return st


# ---- one pass --------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"slots": _own_slots, "norm": _own_norm, "rope": _own_rope,
                "rope_append": _own_rope_append, "chunk": _own_chunk,
                "logprobs": _own_logprobs}[op](state)
    return {"slots": _plain_slots, "norm": _plain_norm, "rope": _plain_rope,
            "rope_append": _plain_rope_append, "chunk": _plain_chunk,
            "logprobs": _plain_logprobs}[op](state)


def _plain_slots(st):
    tokens = st["tokens"]
    n = torch.where(st["granted"] != 0, st["need"].clamp(min=0), 0).long()
    ends = torch.cumsum(n, 0).clamp(max=tokens)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), ends])
    t = torch.arange(tokens, device=DEV)
    row = torch.searchsorted(ends, t, right=True)
    there = row < n.shape[0]
    row = torch.where(there, row, 0)
    position = st["lengths"].long()[row] + t - starts[row]
    return {"starts": starts.to(torch.int32), "rows": torch.where(there, row, -1).to(torch.int32),
            "positions": torch.where(there, position, -1).to(torch.int32),
            "lengths": (st["lengths"] + (starts[1:] - starts[:-1])).to(torch.int32)}


def _plain_norm(st):
    case, cols = st["case"], st["case"]["cols"]
    s = st["x"][:, :cols].float()
    if case["residual"]:
        s = s + st["residual"][:, :cols].float()
    y = s * torch.rsqrt((s * s).mean(1, keepdim=True) + st["eps"])
    if case["weight"]:
        y = y * st["weight"].float()
    out = {}
    if case["residual"]:
        out["sum"] = s.to(st["x"].dtype)
    if case["group"]:
        y = y.reshape(case["rows"], -1, case["group"])
        scales = y.abs().amax(2).clamp(min=LOWEST) / TOP
        y = (y / scales[:, :, None]).reshape(case["rows"], cols)
        out["scales"] = scales
    elif case["out"] == "fp8":
        y = y / st["scale"]
    out["y"] = y.clamp(-TOP, TOP).to(TYPE["fp8"]) if case["out"] == "fp8" else y.to(st["x"].dtype)
    return out


def _plain_rotate(x, st):
    """[tokens, heads, d] in 32 bits; the angles in 64, taken modulo a turn."""
    case, h = st["case"], st["case"]["rot"] // 2
    turns = st["positions"].double()[:, None] * st["turns"][None, :]
    angle = (turns - torch.floor(turns)) * (2.0 * math.pi)
    c = (torch.cos(angle) * st["magnitude"]).float()[:, None, :]
    s = (torch.sin(angle) * st["magnitude"]).float()[:, None, :]
    out = x.clone()
    if case["layout"] == "half":
        a, b = x[:, :, :h], x[:, :, h:2 * h]
        out[:, :, :h], out[:, :, h:2 * h] = a * c - b * s, b * c + a * s
    else:
        a, b = x[:, :, 0:2 * h:2], x[:, :, 1:2 * h:2]
        out[:, :, 0:2 * h:2], out[:, :, 1:2 * h:2] = a * c - b * s, b * c + a * s
    return out


def _heads(st):
    """q's, k's and v's [tokens, heads, d] of the fused projection."""
    case, hq = st["case"], st["hq"]
    x = st["qkv"].reshape(st["n"], hq + 2 * case["kv_heads"], case["d"])
    return x[:, :hq], x[:, hq:hq + case["kv_heads"]], x[:, hq + case["kv_heads"]:]


def _plain_rope(st):
    q, k, _ = _heads(st)
    return {"q": _plain_rotate(q.float(), st).to(q.dtype).reshape(st["n"], -1),
            "k": _plain_rotate(k.float(), st).to(k.dtype).reshape(st["n"], -1)}


def _plain_rope_append(st):
    case = st["case"]
    q, k, v = _heads(st)
    page, slot = st["positions"].long() // case["page"], st["positions"].long() % case["page"]
    page = st["tables"].long()[st["rows"].long(), page]
    k, v = _plain_rotate(k.float(), st), v.float()
    for name, x in (("k", k), ("v", v)):
        if case["cache"] == "fp8":
            x = (x / st[name + "_scale"]).clamp(-TOP, TOP).to(TYPE["fp8"]).view(torch.uint8)
            st[name].view(torch.uint8)[page, :, slot] = x
        else:
            st[name][page, :, slot] = x.to(q.dtype)
    return {"q": _plain_rotate(q.float(), st).to(q.dtype).reshape(st["n"], -1), "k": st["k"],
            "v": st["v"]}


def _seen(case, new, length):
    p = torch.arange(length - new, length, device=DEV)[:, None]
    j = torch.arange(length, device=DEV)[None, :]
    seen = j <= p
    if case["window"] > 0:
        seen &= (j > p - case["window"]) | (j < case["sinks"])
    return seen


def _plain_chunk(st):
    case, o = st["case"], st["o"]
    hkv, g, d, ps = (case[x] for x in ("kv_heads", "group", "d", "page"))
    q_all, at = _heads(st)[0], 0
    for r, (new, length) in enumerate(_chunks(case)):
        ids = st["tables"][r, :_ceil(length, ps)].long()
        k, v = (st[x].view(torch.uint8)[ids].view(TYPE["fp8"]) if case["cache"] == "fp8" else st[x][ids]
                for x in ("k", "v"))
        k, v = (x.float().transpose(0, 1).reshape(hkv, -1, d)[:, :length] for x in (k, v))
        q = q_all[at:at + new].float().reshape(new, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * new, d)
        unseen = ~_seen(case, new, length)
        s = torch.matmul(q, (k * (st["k_scale"] * st["scale"])).transpose(1, 2).contiguous())
        s.view(hkv, g, new, length).masked_fill_(unseen, -math.inf)
        s -= s.amax(2, keepdim=True)
        s.exp_()
        s /= s.sum(2, keepdim=True)
        x = torch.matmul(s, v.contiguous() * st["v_scale"])
        o[at:at + new] = x.reshape(hkv, g, new, d).permute(2, 0, 1, 3).reshape(new, hkv * g, d).to(o.dtype)
        at += new
    return o


def _plain_logprobs(st):
    case, cols, top = st["case"], st["case"]["cols"], st["case"]["top"]
    x = st["x"][:, :cols].float()
    t = x * case["scale"]
    t = t - t.amax(1, keepdim=True)
    p = torch.exp(t)
    total = p.sum(1, keepdim=True)
    lse = torch.log(total)
    entropy = (lse - torch.where(p > 0, p * t, 0.0).sum(1, keepdim=True) / total)[:, 0]
    logp = (torch.gather(t, 1, st["targets"].long()[:, None]) - lse)[:, 0]
    # the top ones by value, then the lower index: one whole number that orders so
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 31) - torch.arange(cols, device=DEV)
    ids = torch.topk(key, min(top, cols), 1).indices
    lp = torch.gather(t, 1, ids) - lse
    ids = torch.where(lp == -math.inf, -1, ids)
    if top > cols:
        ids = torch.nn.functional.pad(ids, (0, top - cols), value=-1)
        lp = torch.nn.functional.pad(lp, (0, top - cols), value=-math.inf)
    return {"logp": logp, "entropy": entropy, "top_logp": lp, "top_ids": ids.to(torch.int32)}


def _hip():
    from sile_amd import _abi
    return _abi


def _code(hip, name):
    return {"f32": hip.F32, "f16": hip.F16, "bf16": hip.BF16, "fp8": hip.F8E4M3}[name]


def _ptr(x):
    return 0 if x is None else x.data_ptr()


def _own_slots(st):
    hip = _hip()
    hip.kv_slots(st["case"]["rows"], st["lengths"].data_ptr(), st["need"].data_ptr(),
                 st["granted"].data_ptr(), st["tokens"], st["starts"].data_ptr(),
                 st["rows"].data_ptr(), st["positions"].data_ptr(), st["lengths_out"].data_ptr())
    return {"starts": st["starts"], "rows": st["rows"], "positions": st["positions"],
            "lengths": st["lengths_out"]}


def _own_norm(st):
    hip, case = _hip(), st["case"]
    hip.rmsnorm_rows(_code(hip, case["dtype"]), _code(hip, case["out"]), case["rows"], case["cols"],
                     st["x"].data_ptr(), st["ld"], _ptr(st["residual"]), st["ld"], _ptr(st["sum"]),
                     case["cols"], _ptr(st["weight"]), st["eps"], st["y"].data_ptr(), case["cols"],
                     st["scale"], _ptr(st["scales"]), case["group"])
    out = {"y": st["y"]}
    if case["residual"]:
        out["sum"] = st["sum"]
    if case["group"]:
        out["scales"] = st["scales"]
    return out


def _layout(hip, case):
    return hip.ROPE_HALF if case["layout"] == "half" else hip.ROPE_PAIRS


def _own_rope(st):
    hip, case = _hip(), st["case"]
    q, k, _ = _heads(st)
    hip.rope(_code(hip, case["dtype"]), _layout(hip, case), st["n"], st["hq"], case["kv_heads"],
             case["d"], case["rot"], q.data_ptr(), q.stride(0), st["q"].data_ptr(),
             st["q"].stride(0), k.data_ptr(), k.stride(0), st["k"].data_ptr(), st["k"].stride(0),
             st["positions"].data_ptr(), st["turns"].data_ptr(), st["magnitude"])
    return {"q": st["q"], "k": st["k"]}


def _own_rope_append(st):
    hip, case = _hip(), st["case"]
    q, k, v = _heads(st)
    hip.rope_append(_code(hip, case["dtype"]), _code(hip, case["cache"]), _layout(hip, case), st["n"],
                    st["hq"], case["kv_heads"], case["d"], case["rot"], q.data_ptr(), q.stride(0),
                    st["q"].data_ptr(), st["q"].stride(0), k.data_ptr(), k.stride(0), v.data_ptr(),
                    v.stride(0), st["rows"].data_ptr(), st["positions"].data_ptr(),
                    st["turns"].data_ptr(), st["magnitude"], st["k"].data_ptr(), st["v"].data_ptr(),
                    st["k"].shape[0], case["page"], case["kv_heads"] * case["page"] * case["d"],
                    st["tables"].data_ptr(), case["rows"], st["tables"].shape[1], st["k_scale"],
                    st["v_scale"])
    return {"q": st["q"], "k": st["k"], "v": st["v"]}


def _own_chunk(st):
    hip, case = _hip(), st["case"]
    hq, d, q = st["hq"], case["d"], st["qkv"]
    hip.paged_attn_chunk(_code(hip, case["dtype"]), _code(hip, case["cache"]), st["lengths"].shape[0],
                         st["n"], hq, case["kv_heads"], d, q.data_ptr(), q.stride(0),
                         st["starts"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(),
                         st["k"].shape[0], case["page"], case["kv_heads"] * case["page"] * d,
                         st["tables"].data_ptr(), st["tables"].shape[1], st["lengths"].data_ptr(),
                         st["o"].data_ptr(), hq * d, st["scale"], st["k_scale"], st["v_scale"],
                         case["window"], case["sinks"], st["workspace"].data_ptr(),
                         st["workspace"].numel())
    return st["o"]


def _own_logprobs(st):
    hip, case = _hip(), st["case"]
    hip.logprobs_rows(_code(hip, case["dtype"]), case["rows"], case["cols"], st["x"].data_ptr(),
                      st["ld"], case["scale"], st["targets"].data_ptr(), st["logp"].data_ptr(),
                      st["entropy"].data_ptr(), case["top"], st["top_logp"].data_ptr(),
                      st["top_ids"].data_ptr(), st["workspace"].data_ptr(), st["workspace"].numel())
    return {"logp": st["logp"], "entropy": st["entropy"], "top_logp": st["top_logp"],
            "top_ids": st["top_ids"]}


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    op = case["op"]
    if op == "slots":
        tokens = sum(_pieces(case)) + case["spare"]
        return {"bytes": 4 * (5 * case["rows"] + 2 * tokens), "flops": 3 * tokens}
    if op == "norm":
        n = case["rows"] * case["cols"]
        es = SIZE[case["dtype"]]
        bytes_ = n * (es * (3 if case["residual"] else 1) + SIZE[case["out"]])
        if case["group"]:
            bytes_ += 4 * n // case["group"]
        return {"bytes": bytes_ + (es * case["cols"] if case["weight"] else 0), "flops": 5 * n}
    if op in ("rope", "rope_append"):
        tokens, d, hkv = case["rows"] * case["each"], case["d"], case["kv_heads"]
        hq, es = hkv * case["group"], SIZE[case["dtype"]]
        if op == "rope":
            return {"bytes": tokens * (2 * (hq + hkv) * d * es + 4),
                    "flops": 3 * tokens * (hq + hkv) * case["rot"]}
        return {"bytes": tokens * (2 * hq * d * es + 2 * hkv * d * (es + SIZE[case["cache"]]) + 12),
                "flops": 3 * tokens * (hq + hkv) * case["rot"]}
    if op == "chunk":
        hkv, g, d = case["kv_heads"], case["group"], case["d"]
        tokens = sum(new for new, _ in _chunks(case))
        w, keys, pairs = case["window"], 0, 0
        for new, length in _chunks(case):
            keys += length if w <= 0 else min(length, new + w - 1 + case["sinks"])
            pairs += _pairs(case, new, length)
        return {"bytes": 2 * keys * hkv * d * SIZE[case["cache"]] + 4 * tokens * hkv * g * d,
                "flops": 4 * pairs * hkv * g * d}
    n = case["rows"] * case["cols"]
    return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}


# ---- the definitions in 64 bits ----------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"slots": _exact_slots, "norm": _exact_norm, "rope": _exact_rope,
            "rope_append": _exact_rope, "chunk": _exact_chunk,
            "logprobs": _exact_logprobs}[case["op"]](case, st)


def _exact_slots(case, st):
    starts, rows, positions, lengths = [0], [], [], []
    for r, (n, need, ok) in enumerate(zip(*(st[x].tolist() for x in ("lengths", "need", "granted")))):
        take = min(need if ok else 0, st["tokens"] - starts[-1])
        rows += [r] * take
        positions += range(n, n + take)
        lengths.append(n + take)
        starts.append(starts[-1] + take)
    fill = [-1] * (st["tokens"] - len(rows))
    return {"starts": _ints(starts), "rows": _ints(rows + fill), "positions": _ints(positions + fill),
            "lengths": _ints(lengths)}


def _exact_norm(case, st):
    cols, out = case["cols"], {}
    s = st["x"][:, :cols].double()
    if case["residual"]:
        out["sum"] = s = s + st["residual"][:, :cols].double()
    y = s / torch.sqrt(torch.sum(s ** 2, 1, keepdim=True) / cols + st["eps"])
    if case["weight"]:
        y = y * st["weight"].double()
    if case["out"] == "fp8":
        scale = torch.full_like(y, st["scale"])
        if case["group"]:
            out["scales"] = torch.stack([y[:, i:i + case["group"]].abs().max(1).values.clamp(min=LOWEST) / TOP
                                         for i in range(0, cols, case["group"])], 1)
            scale = out["scales"].repeat_interleave(case["group"], 1)
        y = torch.clamp(y / scale, -TOP, TOP)
    out["y"] = y
    return out


def _exact_rope(case, st):
    d, h, hq, hkv = case["d"], case["rot"] // 2, st["hq"], case["kv_heads"]
    x = st["qkv"].double().reshape(-1, hq + 2 * hkv, d)
    # positions are whole, so the angle is exact in 64 bits but for its last few
    a = torch.remainder(st["positions"].double()[:, None] * st["turns"], 1.0) * (2.0 * math.pi)
    z = torch.polar(torch.full_like(a, st["magnitude"]), a)[:, None, :]
    i = torch.arange(h, device=DEV)
    first, second = (i, i + h) if case["layout"] == "half" else (2 * i, 2 * i + 1)
    turned = x.clone()
    w = torch.complex(x[:, :hq + hkv, first], x[:, :hq + hkv, second]) * z
    turned[:, :hq + hkv, first], turned[:, :hq + hkv, second] = w.real, w.imag
    out = {"q": turned[:, :hq].reshape(-1, hq * d)}
    if case["op"] == "rope":
        out["k"] = turned[:, hq:hq + hkv].reshape(-1, hkv * d)
        return out
    ps = case["page"]
    flat = st["tables"].long()[st["rows"].long(), st["positions"].long().div(ps, rounding_mode="floor")] * ps
    flat = flat + st["positions"].long().remainder(ps)
    for name, at in (("k", hq), ("v", hq + hkv)):
        pool = st[name].double().transpose(1, 2).contiguous()     # [page, slot, head, d]
        new = turned[:, at:at + hkv]
        pool.view(-1, hkv, d)[flat] = (new / st[name + "_scale"]).clamp(-TOP, TOP) \
            if case["cache"] == "fp8" else new
        out[name] = pool.transpose(1, 2).contiguous()
    return out


def _exact_chunk(case, st):
    hkv, g, d, ps = case["kv_heads"], case["group"], case["d"], case["page"]
    o = torch.zeros((st["n"], hkv * g, d), dtype=torch.float64, device=DEV)
    x = st["qkv"].reshape(st["n"], -1, d)
    at = 0
    for r, (new, length) in enumerate(_chunks(case)):
        ids = st["tables"][r, :_ceil(length, ps)].long()
        unseen = _seen(case, new, length).logical_not()
        for h in range(hkv):
            k, v = (st[name][ids, h].double().reshape(-1, d)[:length] for name in ("k", "v"))
            for u in range(g):
                q = x[at:at + new, h * g + u].double()
                s = (q @ k.t().contiguous()) * (st["k_scale"] * st["scale"])
                o[at:at + new, h * g + u] = torch.softmax(s.masked_fill(unseen, -math.inf), 1) @ v * st["v_scale"]
        at += new
    return o


def _exact_logprobs(case, st):
    rows, cols, top = case["rows"], case["cols"], case["top"]
    out = {"logp": torch.zeros(rows, dtype=torch.float64, device=DEV),
           "entropy": torch.zeros(rows, dtype=torch.float64, device=DEV),
           "top_logp": torch.full((rows, top), -math.inf, dtype=torch.float64, device=DEV),
           "top_ids": torch.full((rows, top), -1, dtype=torch.int32, device=DEV)}
    for a in range(0, rows, 256):
        x = st["x"][a:a + 256, :cols].double()
        lp = torch.log_softmax(x * case["scale"], 1)
        p = lp.exp()
        out["entropy"][a:a + 256] = -(p * lp.masked_fill(p == 0, 0.0)).sum(1)
        out["logp"][a:a + 256] = lp.gather(1, st["targets"][a:a + 256, None].long())[:, 0]
        if top:
            order = torch.sort(x, dim=1, descending=True, stable=True)
            n = min(top, cols)
            there = order.values[:, :n] > -math.inf
            ids = order.indices[:, :n]
            out["top_ids"][a:a + 256, :n] = torch.where(there, ids, -1).to(torch.int32)
            out["top_logp"][a:a + 256, :n] = torch.where(there, lp.gather(1, ids), -math.inf)
    return out
