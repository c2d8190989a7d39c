"""A serving step's operators in numpy, in 64 bits, with the error that a kernel of fp32
arithmetic may have: EPS is half a step of fp32, HALF and TINY those of the result's type."""
from __future__ import annotations

import numpy as np

from oracle import cpuref
from tests.helpers import bf16_round, f16_round

EPS = 2.0 ** -24
HALF = {"f32": EPS, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp8": 2.0 ** -4}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134, "fp8": 2.0 ** -10}
NP = {"f32": np.float32, "f16": np.uint16, "bf16": np.uint16, "fp8": np.uint8}
CODE = {"f32": 0, "f16": 1, "bf16": 2, "fp8": 3}


def rounded(x, dtype):
    """(bits, values in fp32) of x in that type."""
    if dtype == "f32":
        x = np.asarray(x, np.float32)
        return x, x
    return f16_round(x) if dtype == "f16" else bf16_round(x)


def values(bits, dtype):
    if dtype == "f32":
        return bits
    if dtype == "fp8":
        return cpuref.e4m3_decode(bits, 1.0)
    return bits.view(np.float16).astype(np.float32) if dtype == "f16" else cpuref.f32_from_bf16(bits)


def rounding(ref, dtype):
    """How far rounding alone may take a result from ref."""
    return np.maximum(HALF[dtype] * np.abs(ref), TINY[dtype])


def within(got, ref, err, dtype, what=""):
    """got is ref, computed with an error of at most err and then rounded to dtype."""
    got, ref = got.astype(np.float64), np.asarray(ref, np.float64)
    if dtype == "fp8":
        ref = np.clip(ref, -448.0, 448.0)
    # (rounding works on ref +- err)
    bound = rounding(np.abs(ref) + err, dtype) + err
    with np.errstate(invalid="ignore"):   # inf - inf: handled below
        off = np.abs(got - ref)
    good = (off <= bound) | ((got == ref) & ~np.isfinite(ref)) | (np.isnan(got) & np.isnan(ref))
    assert good.all(), (what, int((~good).sum()), good.size, np.argwhere(~good)[:3].tolist(),
                        got[~good][:3], ref[~good][:3], float(np.nanmax(off / bound)))


# ---- the token list ---------------------------------------------------------

def slots(lengths, need, granted, max_tokens):
    starts, rows, positions, out = [0], [], [], []
    for r, (n, m) in enumerate(zip(lengths, need)):
        n = max(n, 0)
        m = min(max(m, 0) if granted is None or granted[r] else 0, 2 ** 31 - 1 - n, max_tokens - starts[-1])
        rows += [r] * m
        positions += range(n, n + m)
        out.append(n + m)
        starts.append(starts[-1] + m)
    fill = [-1] * (max_tokens - len(rows))
    return tuple(np.array(x, np.int32) for x in (starts, rows + fill, positions + fill, out))


# ---- rotary positions -------------------------------------------------------

def turns(scaling, rot, base, factor=1.0, original=0.0, low=0.0, high=0.0):
    j = np.arange(rot // 2, dtype=np.float64)
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    t = base ** (-2.0 * j / max(rot, 1)) / (2 * np.pi)
    if scaling == "linear":
        t = t / factor
    if scaling == "turns":
        keep = np.clip((original * t - low) / (high - low), 0, 1)
        t = t * (keep + (1 - keep) / factor)
    if scaling == "dims":
        pair = lambda n: rot * np.log(original / (n * 2 * np.pi)) / (2 * np.log(base))   # noqa: E731
        first, last = max(np.floor(pair(high)), 0), min(np.ceil(pair(low)), rot - 1)
        last = first + 0.001 if last <= first else last
        keep = 1 - np.clip((j - first) / (last - first), 0, 1)
        t = t * (keep + (1 - keep) / factor)
    return t


def rope(x, positions, t, magnitude, layout):
    """x [tokens, heads, d] rotated, and the error of fp32 arithmetic: the angle's product in
    64 bits (2^-53 of it), its rounding to fp32 as at most an eighth of a turn, the sums of the sine and
    cosine, the magnitude, two products and a sum: at most 10 half steps of |a| + |b|."""
    x = x.astype(np.float64)
    h = len(t)
    full = positions.astype(np.float64)[:, None] * t[None, :]
    angle = 2 * np.pi * np.mod(full, 1.0)[:, None, :]
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    i = np.arange(h)
    i, j = (i, i + h) if layout == "half" else (2 * i, 2 * i + 1)
    out, err = x.copy(), np.zeros_like(x)
    a, b = x[:, :, i], x[:, :, j]
    out[:, :, i], out[:, :, j] = a * c - b * s, b * c + a * s
    e = (np.abs(a) + np.abs(b)) * abs(magnitude) * (10 * EPS + 4 * np.pi * 2.0 ** -53 * np.abs(full)[:, None, :])
    err[:, :, i] = err[:, :, j] = e
    return out, err


# ---- the row norm -----------------------------------------------------------

def rmsnorm(x, residual, weight, eps):
    """(s, y, relative error of y): s rounded once, the sum of squares of at most max(64,
    cols / 256) + 24 additions (half of it after the root), six roundings more."""
    s = x.astype(np.float64) + (0 if residual is None else residual.astype(np.float64))
    with np.errstate(invalid="ignore"):
        y = s / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
        if weight is not None:
            y = y * weight.astype(np.float64)
    chain = max(64, x.shape[-1] // 256) + 24
    return s, y, (0.5 * chain + 7) * EPS


# ---- log probabilities ------------------------------------------------------

def logprobs(x, scale, targets, top):
    """logp, entropy, top_logp, top_ids, and the errors of logp (of a column with logit x) and
    of the entropy.  A term's exponent x c - m, c = scale log2 e rounded twice: 2 EPS of |x c|, and one of
    the difference; exp2 to 4 EPS; the sums of a lane's elements (32 of each chunk of 8192) and of
    the lanes, parts and waves (at most 24 joins, of 6 EPS)."""
    x = x.astype(np.float64)
    rows, cols = x.shape
    t = x * scale
    with np.errstate(invalid="ignore", divide="ignore"):
        m = t.max(1, keepdims=True) if cols else np.full((rows, 1), -np.inf)
        m = np.where(m == -np.inf, 0, m)
        p = np.exp(t - m)
        total = p.sum(1, keepdims=True)
        lse = m + np.log(total)
        lp = t - lse
        p = p / total
        entropy = -np.where(p > 0, p * lp, 0).sum(1)
    entropy = np.where(total[:, 0] == 0, 0.0, entropy)
    lp = np.where(x == -np.inf, np.where(np.isnan(lse), np.nan, -np.inf), lp)
    there = (targets >= 0) & (targets < cols)
    logp = np.where(there, lp[np.arange(rows), np.where(there, targets, 0)] if cols else 0.0, 0.0)
    ids = np.full((rows, top), -1, np.int32)
    tlp = np.full((rows, top), -np.inf)
    for r in range(rows):
        at = np.nonzero(x[r] > -np.inf)[0]
        at = at[np.argsort(-x[r][at], kind="stable")][:top]
        ids[r, :len(at)], tlp[r, :len(at)] = at, lp[r, at]
    with np.errstate(invalid="ignore"):
        size = np.where(np.isfinite(t), np.abs(t), 0).max(1) if cols else np.zeros(rows)
        e_exp = 3 * EPS * size + EPS * np.abs(np.where(np.isfinite(t), t - m, 0)).max(1) * 2 if cols else np.zeros(rows)
    e_sum = (32 * -(-cols // 8192) + 150) * EPS
    e_lse = e_exp + 4 * EPS + e_sum
    return (logp, entropy, tlp, ids, lambda v: (e_lse + e_exp)[:, None] + 4 * EPS * np.abs(np.where(np.isfinite(v), v, 0)),
            (e_lse + e_exp) * (2 * np.abs(np.nan_to_num(entropy)) + 4))
