"""GPU: the token list, the row norm and the log probabilities, against numpy in 64 bits with
bounds counted in roundings (tests/serving_ref.py)."""
import numpy as np
import pytest

from tests import serving_ref as ref
from tests.helpers import rng, say

pytestmark = pytest.mark.gpu


def up(hip, x):
    return hip.DeviceBuffer.from_array(x)


def filled(hip, nbytes, byte=0x5A):
    b = hip.DeviceBuffer(max(nbytes, 16))
    b.fill_bytes(byte)
    return b


# ---- the token list ---------------------------------------------------------

def run_slots(hip, lengths, need, granted, cap, stream=None):
    n = len(lengths)
    ins = [up(hip, np.array(x if len(x) else [0], np.int32)) for x in (lengths, need)]
    g = None if granted is None else up(hip, np.array(granted if n else [0], np.int32))
    outs = [filled(hip, 4 * (k + 1)) for k in (n + 1, cap, cap, n)]
    hip.kv_slots(n, ins[0].ptr, ins[1].ptr, g.ptr if g else 0, cap, *(o.ptr for o in outs), stream)
    hip.synchronize()
    got = []
    for o, k in zip(outs, (n + 1, cap, cap, n)):
        x = o.download(np.int32, (k + 1,))
        assert x[k] == 0x5A5A5A5A, "wrote past the array"
        got.append(x[:k])
    return got


@pytest.mark.parametrize("n,most,cap", [(0, 0, 0), (0, 0, 70), (1, 1, 1), (1, 5000, 5000), (3, 0, 10), (64, 1, 64),
                                        (255, 7, 900), (256, 40, 3000), (257, 40, 12000), (1000, 3, 1024),
                                        (5000, 30, 100000), (65536, 2, 70000), (40, 3000, 1025)])
def test_slots(hip, n, most, cap):
    say(f"slots {n} rows, up to {most}, list of {cap}")
    r = rng(n + most)
    lengths = r.integers(-3, 5000, n)
    need = np.where(r.random(n) < 0.3, 0, r.integers(-2, most + 1, n))
    for granted in (None, (r.random(n) < 0.8).astype(np.int32) * 7):
        want = ref.slots(lengths.tolist(), need.tolist(), granted, cap)
        for got, w in zip(run_slots(hip, lengths, need, granted, cap), want):
            assert np.array_equal(got, w)


def test_slots_at_the_last_positions(hip):
    top = 2 ** 31 - 1
    lengths, need = [top - 3, top, -5, top - 1], [10, 4, 2, top]
    for got, w in zip(run_slots(hip, lengths, need, None, 20), ref.slots(lengths, need, None, 20)):
        assert np.array_equal(got, w)
    # more tokens asked for than 32 bits count
    lengths, need = [0] * 300, [top] * 300
    for got, w in zip(run_slots(hip, lengths, need, None, 2000), ref.slots(lengths, need, None, 2000)):
        assert np.array_equal(got, w)


# ---- the row norm -----------------------------------------------------------

class Norm:
    def __init__(self, hip, seed, dtype, out, rows, cols, residual=True, weight=True, group=0, pad=0, scale=0.03,
                 store=True, shift=0, x=None):
        r = rng(seed)
        self.a = (dtype, out, rows, cols, group)
        self.hip, self.ld, self.scale, self.shift, self.store = hip, cols + pad, scale, shift, store
        self.eps = 1e-5
        draw = lambda shape: ref.rounded(r.normal(size=shape).astype(np.float32) * 2, dtype)   # noqa: E731
        xb, self.x = draw((rows, self.ld)) if x is None else ref.rounded(x, dtype)
        rb, self.r = draw((rows, self.ld))
        wb, self.w = draw((cols,))
        es = 4 if dtype == "f32" else 2
        self.es = es
        # (shifted by `shift` elements from a 16-byte boundary)
        self.dx, self.dr, self.dw = (up(hip, np.concatenate([np.zeros(shift, b.dtype), b.reshape(-1)])) for b in (xb, rb, wb))
        self.residual, self.weight = residual, weight
        ys = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}[out]
        self.dy, self.ds = filled(hip, (rows + 1) * self.ld * ys), filled(hip, (rows + 1) * self.ld * es)
        self.dsc = filled(hip, (rows + 1) * max(1, cols // group if group else 1) * 4)

    def run(self, stream=None, sum_to=None, y_to=None):
        dtype, out, rows, cols, group = self.a
        off = self.shift * self.es
        s = self.ds.ptr if sum_to is None else sum_to
        self.hip.rmsnorm_rows(ref.CODE[dtype], ref.CODE[out], rows, cols, self.dx.ptr + off, self.ld,
                              self.dr.ptr + off if self.residual else 0, self.ld, s if self.store else 0, self.ld,
                              self.dw.ptr + off if self.weight else 0, self.eps, self.dy.ptr if y_to is None else y_to,
                              self.ld, self.scale, self.dsc.ptr if group else 0, group, stream)

    def check(self, ds=None, dy=None):
        dtype, out, rows, cols, group = self.a
        self.hip.synchronize()
        s, y, e = ref.rmsnorm(self.x[:, :cols], self.r[:, :cols] if self.residual else None,
                              self.w if self.weight else None, self.eps)
        if self.store and ds is not False:
            got = (ds or self.ds).download(ref.NP[dtype], (rows, self.ld))
            ref.within(ref.values(got[:, :cols], dtype), s, EPS_OF(s), dtype, "sum")
            if ds is None:
                assert (got[:, cols:].view(np.uint8) == 0x5A).all(), "wrote past the row"
        err = np.abs(y) * e
        if out == "fp8":
            scale = np.full((rows, 1), self.scale)
            if group:
                top = np.maximum(np.abs(y).reshape(rows, -1, group).max(2), 2.0 ** -100)
                got = self.dsc.download(np.float32, (rows + 1, cols // group))
                assert (got[rows].view(np.uint32) == 0x5A5A5A5A).all(), "wrote past the scales"
                assert (np.abs(got[:rows] - top / 448) <= top / 448 * (e + 2 * ref.EPS)).all()
                scale = (top / 448).repeat(group, 1)
            y, err = y / scale, np.abs(y / scale) * (2 * e + 4 * ref.EPS)
        got = (dy or self.dy).download(ref.NP[out], (rows, self.ld))
        ref.within(ref.values(got[:, :cols], out), y, err, out, "y")
        if dy is None:
            assert (got[:, cols:].view(np.uint8) == 0x5A).all(), "wrote past the row"


def EPS_OF(s):
    return np.abs(s) * ref.EPS


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 7, 2), (5, 8, 0), (9, 64, 8), (33, 504, 8), (7, 512, 0), (4, 520, 0),
                                           (3, 2048, 0), (3, 2056, 8), (6, 4096, 0), (2, 5000, 0), (2, 8192, 8),
                                           (2, 8200, 0), (2, 16384, 0), (2, 16392, 0), (3, 1001, 0), (2, 1024, 3),
                                           (70, 40, 0)])
def test_norm(hip, dtype, rows, cols, pad):
    say(f"norm {dtype} {rows} x {cols} pitch +{pad}")
    for residual, weight in ((True, True), (False, True), (True, False)):
        c = Norm(hip, rows + cols, dtype, dtype, rows, cols, residual, weight, pad=pad)
        c.run()
        c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,group", [(2, 1, 0), (2, 1, 1), (3, 64, 0), (5, 64, 64), (5, 64, 8), (9, 256, 16), (3, 384, 128),
                                             (3, 2048, 512), (3, 4096, 4096), (2, 8192, 128), (2, 16384, 32), (4, 21, 7),
                                             (3, 999, 333), (3, 1000, 1000), (2, 1536, 768), (2, 17000, 1000)])
def test_norm_into_codes(hip, dtype, rows, cols, group):
    say(f"norm {dtype} -> e4m3 {rows} x {cols}, groups of {group}")
    c = Norm(hip, rows + cols, dtype, "fp8", rows, cols, group=group)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype,cols", [("bf16", 2048), ("bf16", 2047), ("f32", 512), ("f16", 9)])
def test_norm_in_place(hip, dtype, cols):
    """The sum over the residual, and over x; the result over either."""
    for where in ("residual", "x"):
        c = Norm(hip, 3, dtype, dtype, 6, cols)
        b = c.dr if where == "residual" else c.dx
        c.run(sum_to=b.ptr)
        c.check(ds=b)
        c = Norm(hip, 4, dtype, dtype, 6, cols, store=False)
        b = c.dr if where == "residual" else c.dx
        c.run(y_to=b.ptr)
        c.check(dy=b)


@pytest.mark.parametrize("shift", [1, 3, 4])
def test_norm_unaligned(hip, shift):
    for dtype in ("f32", "bf16"):
        for out, group in ((dtype, 0), ("fp8", 64)):
            c = Norm(hip, shift, dtype, out, 3, 1024, group=group, shift=shift)
            c.run()
            c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [3, 511, 513, 2047, 5001, 8193, 16383])
def test_norm_of_part_vectors(hip, dtype, cols):
    """Rows that end inside a vector and begin anywhere; nothing behind them is written."""
    for shift, pad in ((0, 1), (1, 5), (3, 0)):
        for out, group in ((dtype, 0), ("fp8", 0), ("fp8", cols)):
            c = Norm(hip, shift + cols, dtype, out, 3, cols, group=group, pad=pad, shift=shift)
            c.run()
            c.check()


def test_norm_of_zeros_and_extremes(hip):
    """A row of zeros, one whose maximum is below the least, rows with Inf and NaN."""
    for cols in (256, 255):
        x = rng(1).normal(size=(5, cols)).astype(np.float32)
        x[0] = 0
        x[1] = 2.0 ** -120
        x[2, 3] = np.inf
        x[3, 5] = np.nan
        for out, group in (("f32", 0), ("fp8", cols), ("fp8", 0)):
            c = Norm(hip, 2, "f32", out, 5, cols, residual=False, weight=False, group=group, x=x)
            c.run()
            hip.synchronize()
            y = ref.values(c.dy.download(ref.NP[out], (5, cols)), out)
            assert (y[0] == 0).all() and np.isnan(y[3]).all()
            assert np.isnan(y[2, 3]) and (np.delete(y[2], 3) == 0).all()
            if group:
                s = c.dsc.download(np.float32, (5, 1))[:, 0]
                assert (s[[0, 2, 3]] == np.float32(2.0 ** -100) / np.float32(448)).all() and np.isfinite(s).all()


# ---- log probabilities ------------------------------------------------------

class Logits:
    def __init__(self, hip, seed, dtype, rows, cols, top, scale=1.0, pad=0, x=None, shift=0, targets=None):
        r = rng(seed)
        self.hip, self.a = hip, (dtype, rows, cols, top, scale)
        self.ld, self.shift, self.es = cols + pad, shift, 4 if dtype == "f32" else 2
        x = r.normal(size=(rows, self.ld)).astype(np.float32) * 4 if x is None else x
        bits, v = ref.rounded(x, dtype)
        self.x = v.reshape(rows, self.ld)[:, :cols]
        self.targets = r.integers(0, max(cols, 1), rows).astype(np.int32) if targets is None else np.array(targets, np.int32)
        self.dx = up(hip, np.concatenate([np.zeros(shift + 1, bits.dtype), bits.reshape(-1)])[1:] if bits.size else np.zeros(4, bits.dtype))
        self.dt = up(hip, self.targets)
        self.outs = [filled(hip, 4 * (n + 1)) for n in (rows, rows, rows * top, rows * top)]
        self.n = (rows, rows, rows * top, rows * top)
        need = hip.logprobs_workspace(rows, cols, top)
        self.ws = filled(hip, need, 0xFF)
        self.need = need

    def run(self, stream=None):
        dtype, rows, cols, top, scale = self.a
        o = self.outs
        self.hip.logprobs_rows(ref.CODE[dtype], rows, cols, self.dx.ptr + self.shift * self.es, self.ld, scale,
                               self.dt.ptr, o[0].ptr, o[1].ptr, top, o[2].ptr, o[3].ptr, self.ws.ptr, self.need, stream)

    def results(self):
        self.hip.synchronize()
        got = []
        for o, n, t in zip(self.outs, self.n, (np.float32, np.float32, np.float32, np.int32)):
            x = o.download(t, (n + 1,))
            assert x[n:].view(np.uint32)[0] == 0x5A5A5A5A, "wrote past the array"
            got.append(x[:n])
        rows, top = self.a[1], self.a[3]
        return got[0], got[1], got[2].reshape(rows, top), got[3].reshape(rows, top)

    def check(self, what=""):
        dtype, rows, cols, top, scale = self.a
        logp, entropy, tlp, ids = self.results()
        w_logp, w_entropy, w_tlp, w_ids, e, e_entropy = ref.logprobs(self.x, np.float32(scale), self.targets, top)
        assert np.array_equal(ids, w_ids), (what, ids[(ids != w_ids).any(1)][:2], w_ids[(ids != w_ids).any(1)][:2])
        ref.within(logp[:, None], w_logp[:, None], e(w_logp[:, None]), "f32", what + " logp")
        ref.within(tlp, w_tlp, e(w_tlp), "f32", what + " top")
        ref.within(entropy, w_entropy, e_entropy, "f32", what + " entropy")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,top,pad", [(1, 1, 1, 0), (1, 1, 0, 0), (3, 2, 5, 1), (2, 63, 64, 0), (5, 100, 20, 4), (4, 1000, 64, 3),
                                               (3, 8191, 10, 0), (3, 8192, 64, 0), (2, 8193, 20, 0), (2, 32001, 50, 0),
                                               (300, 500, 3, 0), (1, 200000, 40, 1), (2, 131072, 64, 0), (1100, 17000, 2, 0)])
def test_logprobs(hip, dtype, rows, cols, top, pad):
    say(f"logprobs {dtype} {rows} x {cols} top {top}")
    c = Logits(hip, cols, dtype, rows, cols, top, scale=0.8, pad=pad)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [700, 9000, 100000])
def test_logprobs_ties(hip, dtype, cols):
    """Rows of equal logits, of two values, of few values, rising and falling, with +0 and -0."""
    r = rng(cols)
    x = np.stack([np.full(cols, 1.5), np.where(r.random(cols) < 0.5, 1.0, 2.0), np.round(r.normal(size=cols) * 2),
                  np.arange(cols) / 256.0, -np.arange(cols) / 256.0, np.where(r.random(cols) < 0.5, 0.0, -0.0)]).astype(np.float32)
    for top in (1, 20, 64):
        c = Logits(hip, 1, dtype, len(x), cols, top, x=x)
        c.run()
        c.check(f"ties {cols} {top}")


@pytest.mark.parametrize("cols", [40, 8192, 70000])
def test_logprobs_masked(hip, cols):
    """-inf nearly everywhere, everywhere, or at the type's lowest value."""
    r = rng(cols)
    x = r.normal(size=(6, cols)).astype(np.float32)
    x[0] = -np.inf
    x[1, 1:] = -np.inf
    x[2, :-1] = -np.inf
    x[3, r.random(cols) < 0.99] = -np.inf
    x[3, 7] = 0
    x[4, r.random(cols) < 0.9] = np.finfo(np.float32).min
    x[5] = np.finfo(np.float32).min
    c = Logits(hip, 1, "f32", 6, cols, 12, x=x, targets=[3, 0, cols - 1, 7, 2, 9])
    c.run()
    c.check("masked")


@pytest.mark.parametrize("cols", [50, 9000, 100000])
def test_logprobs_not_finite(hip, cols):
    """NaN or +inf: numbers NaN, the columns by comparison (NaN never)."""
    x = rng(3).normal(size=(3, cols)).astype(np.float32)
    x[0, 5] = np.nan
    x[1, cols - 2] = np.inf
    x[2] = np.nan
    c = Logits(hip, 1, "f32", 3, cols, 4, x=x)
    c.run()
    logp, entropy, tlp, ids = c.results()
    assert np.isnan(logp).all() and np.isnan(entropy).all()
    _, _, _, want, _, _ = ref.logprobs(np.where(np.isnan(x), -np.inf, x), 1.0, c.targets, 4)
    assert np.array_equal(ids, want)
    assert np.isnan(tlp[ids >= 0]).all()


def test_logprobs_targets_outside_and_parts_left_out(hip):
    c = Logits(hip, 5, "f16", 4, 300, 3, targets=[-1, 300, 299, 0])
    c.run()
    c.check()
    d = Logits(hip, 5, "f16", 4, 300, 3, targets=[-1, 300, 299, 0])
    hip.logprobs_rows(hip.F16, 4, 300, d.dx.ptr, 300, 1.0, 0, 0, d.outs[1].ptr, 0, 0, 0)
    got = d.results()
    assert np.array_equal(got[1], c.results()[1]) and (got[0].view(np.uint32) == 0x5A5A5A5A).all()


@pytest.mark.parametrize("dtype,shift", [("bf16", 1), ("f16", 3), ("f32", 1)])
def test_logprobs_unaligned(hip, dtype, shift):
    c = Logits(hip, 9, dtype, 3, 20001, 7, shift=shift)
    c.run()
    c.check()


def test_logprobs_sharp_rows(hip):
    """One token with nearly all the mass: logp near 0 and a small entropy keep their digits."""
    x = rng(8).normal(size=(3, 50000)).astype(np.float32)
    x[0, 40000], x[1, 3], x[2, 49999] = 30.0, 60.0, 1000.0
    c = Logits(hip, 1, "f32", 3, 50000, 2, x=x, targets=[40000, 3, 49999])
    c.run()
    c.check("sharp")
    # the third row's rest is below 2^-1000: what is left are the roundings of exp2 (4 half steps),
    # of its logarithm and of the quotient
    logp, entropy, _, _ = c.results()
    assert abs(logp[2]) <= 16 * ref.EPS and 0 <= entropy[2] <= 16 * ref.EPS and 0 < entropy[0] < 1e-4


# ---- streams and graphs -----------------------------------------------------

def test_rows_in_a_graph(hip):
    """Norm and log probabilities captured, replayed between other work, as the plain calls."""
    n = Norm(hip, 7, "bf16", "fp8", 9, 2048, group=128)
    c = Logits(hip, 7, "bf16", 5, 60000, 10)
    n.run()
    c.run()
    hip.synchronize()
    want = [n.dy.download(np.uint8, (9, 2048)), c.results()]
    lengths, need = np.arange(50), np.ones(50, np.int64)
    st = hip.Stream()
    with hip.Graph(st) as g:
        n.run(st)
        c.run(st)
    for _ in range(3):
        n.dy.fill_bytes(0)
        for o in c.outs[:3]:
            o.fill_bytes(0x5A)
        hip.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(n.dy.download(np.uint8, (9, 2048)), want[0])
        for a, b in zip(c.results(), want[1]):
            assert np.array_equal(a, b)
        run_slots(hip, lengths, need, None, 64)
    n.check()
    g.close()
    st.close()
