"""The paged cache's operators in numpy: the attention in 64 bits with the error a
kernel may have, the bookkeeping in whole numbers."""
from __future__ import annotations

import numpy as np

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step of the subnormals


def seen_keys(length, window, sinks):
    j = np.arange(length)
    if window <= 0:
        return j
    return j[(j >= length - window) | (j < sinks)]


def attention(q, k, v, scale):
    """One query [d] over keys [n, d]: softmax(q . k * scale) v in 64 bits, and
    sum_j p_j |v_j| and the largest sum_t |q_t k_t| * |scale| for the error bound."""
    if len(k) == 0:
        z = np.zeros(v.shape[1])
        return z, z, 0.0
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    with np.errstate(invalid="ignore", over="ignore"):
        s = (k @ q) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        return p @ v, p @ np.abs(v), float(np.max(np.abs(k) @ np.abs(q)) * abs(scale))


def error_bound(ref, spread, size, dtype, d, keys, p_error):
    """How far a result may be from `ref`, by arithmetic alone:
      half a step of the result's type;
      the scores: d products added in fp32 and scaled, each step 2^-24 of at most `size`
        (and once more for the product with log2 e, at most 2 size), exp2 to 2^-22:
        as a relative error of every p, counted twice (the sum of p has it too);
      p_error: the relative error of a probability as the product takes it;
      the sums over the keys: fp32, at most `keys` additions, numerator and denominator.
    The last three weigh sum p |v| (`spread`)."""
    score = (d + 4) * 2.0 ** -24 * 2.0 * size + 2.0 ** -22
    rel = 2.0 * (score + p_error) + 2.0 * (keys + 8) * 2.0 ** -24
    return HALF[dtype] * np.abs(ref) + (1 + HALF[dtype]) * rel * spread + TINY[dtype]


def reserve(page_size, num_pages, lengths, need, tables, refs):
    """(tables, refs, granted, copies) after handing out pages."""
    tables, width = [list(t) for t in tables], len(tables[0]) if len(tables) else 0
    before, refs = list(refs), list(refs)
    free = [p for p in range(num_pages) if before[p] <= 0]
    granted, copies, taken, asked = [], [], 0, 0
    for r, (n, m) in enumerate(zip(lengths, need)):
        cap = width * page_size
        n = min(max(n, 0), cap)
        if m <= 0:
            granted.append(1)
            continue
        if n + m > cap:
            granted.append(0)
            continue
        count = lambda p: before[p] if 0 <= p < num_pages else 0  # noqa: E731
        want = [e for e in range(n // page_size, (n + m - 1) // page_size + 1)
                if count(tables[r][e]) != 1]
        asked += len(want)
        granted.append(int(not want or asked <= len(free)))
        for e in want if granted[-1] else []:
            old, page = tables[r][e], free[taken]
            taken += 1
            if count(old) > 1:
                refs[old] -= 1
                if e == n // page_size and n % page_size:
                    copies.append((old, page))
            refs[page] = 1
            tables[r][e] = page
    return tables, refs, granted, copies


def compact(num_pages, tables, refs):
    """(tables, refs, used, moves) after closing the pool up."""
    live = [p for p in range(num_pages) if refs[p] > 0]
    u = len(live)
    moves = dict(zip([p for p in live if p >= u],
                     [p for p in range(u) if refs[p] <= 0]))
    out = [0] * num_pages
    for p in live:
        out[moves.get(p, p)] = refs[p]
    return [[moves.get(p, p) for p in t] for t in tables], out, u, moves
