"""GPU: rotary positions, into memory and into the paged cache, against numpy in 64 bits with
bounds counted in roundings (tests/serving_ref.py)."""
import numpy as np
import pytest

from tests import serving_ref as ref
from tests.helpers import rng, say

pytestmark = pytest.mark.gpu


class Rope:
    """Tokens of a fused projection [tokens, (hq + 2 hkv) d + pad]; q to memory; k to memory, or, with
    `cache`, k and v into pages."""

    def __init__(self, hip, seed, dtype, layout, n, hq, hkv, d, rot, positions=None, magnitude=1.1, cache=None,
                 page=16, pad=0, shift=0, base=10000.0, n_rows=3, far=0, spare=2, pad_page=0):
        r = rng(seed)
        self.hip, self.dtype, self.layout, self.n, self.hq, self.hkv, self.d, self.rot = hip, dtype, layout, n, hq, hkv, d, rot
        self.cache, self.page, self.magnitude, self.shift = cache, page, magnitude, shift
        self.es = 4 if dtype == "f32" else 2
        self.ld = (hq + 2 * hkv) * d + pad
        bits, self.x = ref.rounded(r.normal(size=(n, self.ld)).astype(np.float32), dtype)
        self.bits = bits
        self.dx = hip.DeviceBuffer.from_array(np.concatenate([np.zeros(shift, bits.dtype), bits.reshape(-1)]))
        self.t = ref.turns("none", rot, base)
        self.dt = hip.DeviceBuffer.from_array(self.t if rot else np.zeros(1))
        self.rows = np.sort(r.integers(0, n_rows, n)).astype(np.int32)
        if positions is None:   # each row's tokens one behind the other, from anywhere
            first = r.integers(0, 40, n_rows) + far
            seen, positions = {}, []
            for row in self.rows:
                positions.append(first[row] + seen.get(row, 0))
                seen[row] = seen.get(row, 0) + 1
        self.positions = np.array(positions, np.int32)
        self.dp, self.dr = (hip.DeviceBuffer.from_array(x) for x in (self.positions, self.rows))
        self.ldo = max(hq * d, hkv * d, 1) + 8
        self.dq = hip.DeviceBuffer((n + 1) * self.ldo * self.es)
        self.dk = hip.DeviceBuffer((n + 1) * self.ldo * self.es)
        self.dq.fill_bytes(0x5A)
        self.dk.fill_bytes(0x5A)
        if cache:
            self.width = -(-(int(self.positions.max(initial=0)) + 1) // page) + 1
            self.num = n_rows * self.width + spare
            self.stride = hkv * page * d + pad_page
            self.n_rows = n_rows
            self.tables = r.permutation(self.num)[:n_rows * self.width].astype(np.int32).reshape(n_rows, self.width)
            self.dtab = hip.DeviceBuffer.from_array(self.tables)
            self.cs = 1 if cache == "fp8" else 2
            self.pools = [hip.DeviceBuffer(self.num * self.stride * self.cs) for _ in "kv"]
            for p in self.pools:
                p.fill_bytes(0x5A)
            self.scales = (0.031, 0.027) if cache == "fp8" else (1.0, 1.0)

    def run(self, stream=None, in_place=False, with_rows=True):
        h, es = self.hip, self.es
        q = self.dx.ptr + self.shift * es
        k, v = q + self.hq * self.d * es, q + (self.hq + self.hkv) * self.d * es
        lay = h.ROPE_HALF if self.layout == "half" else h.ROPE_PAIRS
        t = ref.CODE[self.dtype]
        qo, lq = (q, self.ld) if in_place else (self.dq.ptr, self.ldo)
        ko, lk = (k, self.ld) if in_place else (self.dk.ptr, self.ldo)
        if self.cache:
            h.rope_append(t, ref.CODE[self.cache], lay, self.n, self.hq, self.hkv, self.d, self.rot, q, self.ld, qo,
                          lq, k, self.ld, v, self.ld, self.dr.ptr if with_rows else 0, self.dp.ptr, self.dt.ptr, self.magnitude, self.pools[0].ptr,
                          self.pools[1].ptr, self.num, self.page, self.stride, self.dtab.ptr, self.n_rows, self.width,
                          self.scales[0], self.scales[1], stream)
        else:
            h.rope(t, lay, self.n, self.hq, self.hkv, self.d, self.rot, q if self.hq else 0, self.ld, qo if self.hq else 0, lq,
                   k if self.hkv else 0, self.ld, ko if self.hkv else 0, lk, self.dp.ptr, self.dt.ptr, self.magnitude, stream)

    def heads(self):
        x = self.x[:, :(self.hq + 2 * self.hkv) * self.d].reshape(self.n, -1, self.d)
        return x[:, :self.hq], x[:, self.hq:self.hq + self.hkv], x[:, self.hq + self.hkv:]

    def check_out(self, buf, x, what):
        """Tokens at positions below 0, and what lies behind a token, as they were."""
        w = x.shape[1] * self.d
        got = buf.download(ref.NP[self.dtype], (self.n + 1, self.ldo))
        assert (got[:, w:].view(np.uint8) == 0x5A).all() and (got[self.n].view(np.uint8) == 0x5A).all(), "wrote past"
        left = self.positions < 0
        assert (got[:self.n][left].view(np.uint8) == 0x5A).all(), "wrote a token that is left out"
        want, err = ref.rope(x[~left], self.positions[~left], self.t, self.magnitude, self.layout)
        ref.within(ref.values(got[:self.n][~left][:, :w], self.dtype).reshape(want.shape), want, err, self.dtype, what)
        stays = ref.values(got[:self.n][~left][:, :w], self.dtype).reshape(want.shape)[:, :, self.rot:]
        assert np.array_equal(stays, x[~left][:, :, self.rot:]), "dims past rot changed"

    def check(self, left_out=()):
        self.hip.synchronize()
        q, k, v = self.heads()
        if self.hq:
            self.check_out(self.dq, q, "q")
        if not self.cache:
            if self.hkv:
                self.check_out(self.dk, k, "k")
            return
        for name, x, pool, scale in (("k", k, self.pools[0], self.scales[0]), ("v", v, self.pools[1], self.scales[1])):
            got = pool.download(ref.NP[self.cache], (self.num, self.stride))
            touched = np.zeros(got.shape, bool)
            view = got[:, :self.hkv * self.page * self.d].reshape(self.num, self.hkv, self.page, self.d)
            mark = touched[:, :self.hkv * self.page * self.d].reshape(view.shape)
            if name == "k":
                x, err = ref.rope(x, self.positions, self.t, self.magnitude, self.layout)
            else:
                x, err = x.astype(np.float64), np.zeros(x.shape)
            if self.cache == "fp8":
                x, err = x / scale, (err + np.abs(x) * 2 * ref.EPS) / scale
            keep = [i for i in range(self.n) if i not in left_out]
            page = self.tables[self.rows[keep], self.positions[keep] // self.page]
            slot = self.positions[keep] % self.page
            ref.within(ref.values(view[page, :, slot], self.cache), x[keep], err[keep], self.cache, name)
            mark[page, :, slot] = True
            assert (got[~touched].view(np.uint8) == 0x5A).all(), "wrote elsewhere in the pool"


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,hq,hkv,d,rot,pad", [(1, 1, 1, 2, 2, 0), (5, 4, 2, 64, 64, 0), (7, 3, 1, 80, 80, 8), (33, 8, 2, 128, 32, 0),
                                                (3, 2, 2, 72, 72, 0), (4, 5, 1, 96, 48, 8), (2, 40, 8, 128, 128, 0),
                                                (3, 2, 1, 7, 6, 0), (3, 2, 1, 9, 4, 1), (2, 1, 0, 256, 256, 0), (2, 0, 3, 64, 0, 0),
                                                (1, 100, 10, 256, 64, 0), (2, 1, 1, 2048, 2048, 0), (3000, 1, 1, 16, 16, 0)])
def test_rope(hip, dtype, layout, n, hq, hkv, d, rot, pad):
    say(f"rope {dtype} {layout} {n} tokens {hq}+{hkv} heads of {d}, {rot} turned, pitch +{pad}")
    c = Rope(hip, n + d, dtype, layout, n, hq, hkv, d, rot, pad=pad)
    c.run()
    c.check()


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "fp8"), ("bf16", "fp8")])
@pytest.mark.parametrize("n,hq,hkv,d,rot,page,pad_page", [(1, 4, 1, 64, 64, 16, 0), (50, 8, 2, 128, 128, 16, 0), (20, 3, 3, 80, 40, 8, 16),
                                                          (9, 2, 1, 96, 96, 1, 0), (300, 4, 2, 64, 32, 128, 0),
                                                          (5, 0, 2, 128, 128, 32, 0), (4, 2, 2, 256, 20, 16, 0), (3, 5, 2, 112, 24, 4, 32)])
def test_rope_append(hip, dtype, cache, layout, n, hq, hkv, d, rot, page, pad_page):
    say(f"rope_append {dtype} -> {cache} {layout} {n} tokens {hq}+{hkv} heads of {d}, {rot} turned, pages of {page}")
    c = Rope(hip, n + d, dtype, layout, n, hq, hkv, d, rot, cache=cache, page=page, pad_page=pad_page)
    c.run()
    c.check()


@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_rope_far_positions(hip, layout):
    """Angles are as good at the last position as at the first: fp32 results at 2^31 - 1."""
    p = [0, 1, 1000, 131071, 10 ** 6, 2 ** 24 + 1, 2 ** 30 + 12345, 2 ** 31 - 1, -1, -(2 ** 31)]
    c = Rope(hip, 1, "f32", layout, len(p), 2, 1, 128, 128, positions=p, base=500000.0)
    c.run()
    c.check()


def test_rope_turned_back(hip):
    """Negative turns undo a rotation, in place."""
    c = Rope(hip, 2, "f32", "half", 40, 3, 1, 64, 64, magnitude=1.0, far=5000)
    c.run(in_place=True)
    back = hip.DeviceBuffer.from_array(-c.t)
    c.dt = back
    c.run(in_place=True)
    hip.synchronize()
    got = c.dx.download(np.float32, (40, c.ld))[:, :4 * 64]
    # two rotations, each off by at most 10 half steps of |a| + |b| <= sqrt 2 |(a, b)|, and rounded
    x = c.x[:, :4 * 64].reshape(40, 4, 64)
    size = np.sqrt(x[:, :, :32] ** 2 + x[:, :, 32:] ** 2)
    err = np.abs(got.reshape(x.shape) - x)
    assert (err <= np.concatenate([size, size], 2) * 2 * (10 * np.sqrt(2) + 2) * ref.EPS).all()


@pytest.mark.parametrize("dtype,d,rot", [("bf16", 128, 128), ("f16", 72, 40), ("bf16", 9, 4)])
def test_rope_in_place(hip, dtype, d, rot):
    a, b = (Rope(hip, 3, dtype, "pairs", 20, 4, 2, d, rot) for _ in range(2))
    a.run()
    b.run(in_place=True)
    hip.synchronize()
    es = ref.NP[dtype]
    got = b.dx.download(es, (20, b.ld))
    q, k = a.dq.download(es, (21, a.ldo)), a.dk.download(es, (21, a.ldo))
    assert np.array_equal(got[:, :4 * d], q[:20, :4 * d]) and np.array_equal(got[:, 4 * d:6 * d], k[:20, :2 * d])
    assert np.array_equal(got[:, 6 * d:], b.bits[:, 6 * d:])


@pytest.mark.parametrize("dtype,shift", [("f32", 1), ("bf16", 1), ("f16", 4)])
def test_rope_unaligned(hip, dtype, shift):
    c = Rope(hip, 4, dtype, "half", 6, 3, 2, 64, 64, shift=shift)
    c.run()
    c.check()


def test_rope_append_leaves_out(hip):
    """Rows, positions and pages that do not exist: nothing stored; the queries still turn where
    the position is one."""
    c = Rope(hip, 6, "bf16", "half", 6, 2, 1, 64, 64, cache="bf16")
    c.positions[1] = -1
    c.positions[2] = c.width * c.page
    rows = c.rows.copy()
    rows[3], rows[4] = -1, c.n_rows
    c.tables[c.rows[5], c.positions[5] // c.page] = c.num   # a page outside the pool
    c.dtab = hip.DeviceBuffer.from_array(c.tables)
    c.dr, c.dp = hip.DeviceBuffer.from_array(rows), hip.DeviceBuffer.from_array(c.positions)
    c.run()
    gone = {i for i in range(6) if i in (1, 2, 3, 4) or c.tables[c.rows[i], min(c.positions[i] // c.page, c.width - 1)] == c.num}
    c.check(left_out=gone)


def test_rope_append_rows_null(hip):
    c = Rope(hip, 8, "f16", "pairs", 5, 2, 1, 64, 64, cache="f16", n_rows=5)
    c.rows = np.arange(5, dtype=np.int32)
    c.positions = np.array([0, 3, 9, 1, 17], np.int32) % (c.width * c.page)
    c.dp = hip.DeviceBuffer.from_array(c.positions)
    c.run(with_rows=False)
    c.check()


def test_rope_append_is_rope_then_append(hip):
    """One launch gives what the two calls give, where the cache has the tokens' type."""
    a, b = (Rope(hip, 9, "bf16", "half", 60, 4, 2, 128, 64, cache="bf16") for _ in range(2))
    a.run()
    b.cache, cache = None, b.cache
    b.run()
    b.cache = cache
    hip.kv_append(hip.BF16, hip.BF16, b.n, b.hkv, b.d, b.dk.ptr, b.ldo, b.dx.ptr + (b.hq + b.hkv) * b.d * 2, b.ld, b.dr.ptr,
                  b.dp.ptr, b.pools[0].ptr, b.pools[1].ptr, b.num, b.page, b.stride, b.dtab.ptr, b.n_rows, b.width)
    hip.synchronize()
    for x, y in ((a.dq, b.dq), (a.pools[0], b.pools[0]), (a.pools[1], b.pools[1])):
        assert np.array_equal(x.download(np.uint8, (x.nbytes,)), y.download(np.uint8, (y.nbytes,)))


def test_rope_in_a_graph(hip):
    c = Rope(hip, 11, "bf16", "half", 30, 4, 2, 64, 64, cache="fp8")
    st = hip.Stream()
    with hip.Graph(st) as g:
        c.run(st)
    for _ in range(3):
        c.dq.fill_bytes(0x5A)
        for p in c.pools:
            p.fill_bytes(0x5A)
        hip.synchronize()
        g.launch()
        st.synchronize()
        c.check()
    g.close()
    st.close()
