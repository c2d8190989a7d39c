"""GPU: log probabilities and entropies of rows where one column has nearly all of the mass, against
64 bits with a bound relative to the result: both are then small, and come from the other columns alone."""
import numpy as np
import pytest

from tests import serving_ref as ref
from tests.helpers import rng, say
from tests.test_gpu_serving_rows import Logits

pytestmark = pytest.mark.gpu


def expected(x, scale, targets, ids):
    """logp of the targets and of the columns ids, the entropy, and their errors in fp32, with
    u = sum p of all columns but one that has the maximum (d = t - max, EPS half a step):
      p = 2^(c (x - max)): the difference, c (two roundings) and the product, 4 EPS |d|, and exp2 to 4 EPS
      sums: 32 additions of a lane's chunk of 8192, 6 + 4 + 10 of lanes, waves and parts; a growing
      maximum scales what there is, for each chunk and 4 joins, at 12 EPS each; a sum of at least 1.25 with
      the maximum's 1 in it loses, less that, a factor of 5
      log1p to 4 EPS; (x - max) * scale to 2 EPS; the last sums and quotient to 4 EPS"""
    t = x.astype(np.float64) * np.float64(np.float32(scale))
    n = np.arange(len(t))
    d = t - t.max(1, keepdims=True)
    p = np.exp(d)
    seen, dd = p > 0, np.where(p > 0, d, 0.0)
    others = p.copy()
    others[n, t.argmax(1)] = 0.0
    sums = 5 * (100 + 12 * -(-x.shape[1] // 8192)) * ref.EPS
    tiny = x.shape[1] * 2.0 ** -120   # (exp2 below 2^-126 is 0)
    u = others.sum(1)
    e_u = (others * (4 * np.abs(dd) + 4)).sum(1) * ref.EPS + u * sums + tiny
    s = -(others * dd).sum(1)
    e_s = (others * np.abs(dd) * (4 * np.abs(dd) + 6)).sum(1) * ref.EPS + s * sums + tiny
    log, e_log = np.log1p(u), e_u / (1 + u) + 4 * ref.EPS * np.log1p(u)
    entropy = log + s / (1 + u)
    e_entropy = e_log + e_s / (1 + u) + s * e_u / (1 + u) ** 2 + 4 * ref.EPS * entropy

    def of(cols):
        at = dd[n[:, None], cols]
        v = np.where(seen[n[:, None], cols], at, d[n[:, None], cols]) - log[:, None]
        with np.errstate(invalid="ignore"):
            return v, e_log[:, None] + np.where(np.isfinite(v), np.abs(v), 0) * 4 * ref.EPS

    (logp, e_logp), (top, e_top) = of(targets[:, None]), of(ids)
    return (logp[:, 0], e_logp[:, 0]), (entropy, e_entropy), (top, e_top)


def check(hip, dtype, x, targets, scale, top, what):
    say(what)
    c = Logits(hip, 1, dtype, len(x), x.shape[1], top, scale=scale, x=x, targets=targets)
    c.run()
    logp, entropy, tlp, ids = c.results()
    want = ref.logprobs(c.x, np.float32(scale), c.targets, top)[3]
    assert np.array_equal(ids, want), what
    for name, got, (w, err) in zip(("logp", "entropy", "top"), (logp, entropy, tlp),
                                   expected(c.x, scale, c.targets, np.maximum(ids, 0))):
        there = np.isfinite(w) if name != "top" else (ids >= 0) & np.isfinite(w)
        with np.errstate(invalid="ignore"):   # inf - inf: not there
            off = np.abs(got.astype(np.float64) - w)
        assert (off[there] <= err[there]).all(), (what, name, got[there][:4], w[there][:4], float((off[there] / err[there]).max()))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(7, 40), (7, 5000), (7, 50000), (7, 131072), (1, 200001), (1200, 8200)])
def test_sharp(hip, dtype, rows, cols):
    """One column far above N(0, 1) ones, by 2 to 60, also the first, the last and past the whole vectors."""
    r = rng(cols)
    x = r.normal(size=(rows, cols)).astype(np.float32)
    at = r.integers(0, cols, rows)
    at[0], at[-1] = 0, cols - 1
    x[np.arange(rows), at] = np.tile([16.0, 30.0, 10.0, 6.0, 60.0, 20.0, 12.0], rows // 7 + 1)[:rows]
    check(hip, dtype, x, at.astype(np.int32), 1.0, 3, f"sharp {dtype} {rows} x {cols}")
    # another column's, which is far from 0
    check(hip, dtype, x, ((at + 1) % cols).astype(np.int32), 0.8, 0, f"sharp {dtype} {rows} x {cols}, another target")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [300, 5000, 70000])
def test_mostly_masked(hip, dtype, cols):
    """99 % of the columns at -inf, scaled by 2: logp around -1e-3."""
    r = rng(cols + 1)
    x = (r.normal(size=(50, cols)) * 2).astype(np.float32)
    x[r.random(x.shape) < 0.99] = -np.inf
    at = r.integers(0, cols, 50).astype(np.int32)
    x[np.arange(50), at] = 8.0
    check(hip, dtype, x, at, 2.0, 4, f"masked {dtype} {cols}")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("cols", [64, 9000, 150000])
def test_several_maxima(hip, dtype, cols):
    """The maximum twice in a lane's columns, in two lanes, waves and parts, in every column, and in a
    rising row, whose maximum is new in each chunk."""
    r = rng(cols + 2)
    x = r.normal(size=(6, cols)).astype(np.float32)
    for row, at in enumerate(((3, 4), (5, cols // 2), (0, cols - 1), (cols - 2, cols - 1))):
        x[row, list(at)] = 25.0
    x[4] = 1.5
    x[5] = np.linspace(-8, 8, cols)
    check(hip, dtype, x, np.array([3, 5, 0, cols - 1, 7, cols - 1], np.int32), 1.0, 5, f"several maxima {dtype} {cols}")
