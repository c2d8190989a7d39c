"""GPU: attention over a sliding window with sinks, against numpy in 64 bits with a bound
derived from the arithmetic (paged_ref.error_bound)."""
import numpy as np
import pytest

from oracle import cpuref
from tests import paged_ref
from tests.helpers import bf16_round, f16_round, rng, say

pytestmark = pytest.mark.gpu

# half a step of a probability in 16 bits; the sum is of the rounded ones
P_ERROR = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def rounded(x, dtype):
    return f16_round(x) if dtype == "f16" else bf16_round(x)


def as_f64(bits, dtype):
    return (bits.view(np.float16) if dtype == "f16" else cpuref.f32_from_bf16(bits)).astype(np.float64)


class Case:
    def __init__(self, seed, dtype, b, hq, hkv, n, d, window, sinks=0, start=0, kv_len=None, scale=None):
        r = rng(seed)
        self.dtype, self.b, self.hq, self.hkv, self.n, self.d = dtype, b, hq, hkv, n, d
        self.window, self.sinks, self.start = window, sinks, start
        self.kv_len = start + n if kv_len is None else kv_len
        self.scale = d ** -0.5 if scale is None else scale
        self.qb, self.q = rounded(r.normal(size=(b, hq, n, d)).astype(np.float32), dtype)
        self.kb, self.k = rounded(r.normal(size=(b, hkv, self.kv_len, d)).astype(np.float32), dtype)
        self.vb, self.v = rounded(r.normal(size=(b, hkv, self.kv_len, d)).astype(np.float32), dtype)

    def mask(self):
        p = self.start + np.arange(self.n)[:, None]
        j = np.arange(self.kv_len)[None]
        return (j <= p) & ((j > p - self.window) | (j < self.sinks))

    def run(self, hip, stream=None, offset=0):
        """The output's bits; `offset` bytes off the operands' 16-byte boundaries."""
        say(f"window {self.dtype} {self.b}x{self.hq}/{self.hkv} q={self.n}+{self.start} kv={self.kv_len} d={self.d} "
            f"w={self.window} s={self.sinks}")
        bufs = []
        for x in (self.qb, self.kb, self.vb):
            buf = hip.DeviceBuffer(x.nbytes + 64)
            if x.nbytes:
                hip.call("sile_hip_memcpy_htod", buf.ptr + offset, np.ascontiguousarray(x).ctypes.data, x.nbytes)
            bufs.append(buf)
        o = hip.DeviceBuffer(self.qb.nbytes + 64)
        o.fill_bytes(0x5A)
        hip.synchronize()
        hip.flash_attn_window_fwd(hip.F16 if self.dtype == "f16" else hip.BF16, self.b, self.hq, self.hkv, self.n,
                                  self.kv_len, self.d, *(x.ptr + offset for x in bufs), o.ptr + offset, self.scale,
                                  self.start, self.window, self.sinks, stream)
        hip.synchronize()
        all_ = o.download(np.uint16, (self.qb.size + 32,))
        got = all_[offset // 2:offset // 2 + self.qb.size].reshape(self.qb.shape)
        assert (all_[:offset // 2] == 0x5A5A).all() and (all_[offset // 2 + self.qb.size:] == 0x5A5A).all()
        return got

    def check(self, got, rows=None, p_error=None):
        val = as_f64(got, self.dtype)
        mask = self.mask()
        for b in range(self.b):
            for h in range(self.hq):
                k, v = (x[b, h // (self.hq // self.hkv)] for x in (self.k, self.v))
                for i in range(self.n) if rows is None else rows:
                    at = mask[i]
                    ref, spread, size = paged_ref.attention(self.q[b, h, i], k[at], v[at], self.scale)
                    bound = paged_ref.error_bound(ref, spread, size, self.dtype, self.d, int(at.sum()),
                                                  P_ERROR[self.dtype] if p_error is None else p_error)
                    err = np.abs(val[b, h, i] - ref)
                    same_nan = np.isnan(ref) & np.isnan(val[b, h, i])
                    assert ((err <= bound) | same_nan).all(), (b, h, i, float(np.nanmax(err / bound)),
                                                               val[b, h, i][:4], ref[:4])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 104, 128, 136, 192, 200, 256])
def test_head_dims(hip, dtype, d):
    c = Case(1, dtype, 1, 2, 1, 150, d, 40, 3)
    c.check(c.run(hip))


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 600])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 0), (64, 4), (100, 70), (1000, 5)])
def test_lengths(hip, n, window, sinks):
    c = Case(2, "f16", 1, 2, 2, n, 64, window, sinks)
    c.check(c.run(hip))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (31, 1), (32, 32), (33, 33), (64, 0), (65, 100),
                                          (128, 4), (200, 300), (511, 1), (512, 0), (10 ** 12, 10 ** 12)])
@pytest.mark.parametrize("d", [64, 128])
def test_windows(hip, window, sinks, d):
    c = Case(3, "bf16", 1, 1, 1, 520, d, window, sinks)
    c.check(c.run(hip))


@pytest.mark.parametrize("start,n,kv", [(1, 1, None), (63, 1, None), (500, 1, None), (500, 40, None), (777, 300, None),
                                        (0, 100, 40), (100, 60, 20), (1000, 50, 30), (50, 300, 200), (5, 40, 0)])
@pytest.mark.parametrize("window,sinks", [(16, 0), (70, 3), (400, 90)])
def test_pieces_of_a_prompt(hip, start, n, kv, window, sinks):
    """Queries behind cached keys; fewer keys than positions: some queries see none."""
    c = Case(4, "f16", 1, 2, 1, n, 72, window, sinks, start, kv)
    got = c.run(hip)
    c.check(got)
    empty = ~c.mask().any(1)
    assert (got[:, :, empty] == 0).all()


@pytest.mark.parametrize("b,hq,hkv", [(2, 6, 2), (3, 3, 3), (1, 12, 1), (9, 2, 1), (2, 20, 5)])
def test_head_groups(hip, b, hq, hkv):
    c = Case(5, "bf16", b, hq, hkv, 90, 64, 30, 2)
    c.check(c.run(hip))


@pytest.mark.parametrize("hq,n,d,window", [(8, 2100, 128, 300), (64, 300, 64, 100), (256, 260, 64, 90), (2, 5000, 64, 1000),
                                           (96, 600, 128, 250), (1, 3000, 256, 500)])
def test_layouts(hip, hq, n, d, window):
    """Shapes that take one, two and four key groups."""
    c = Case(6, "f16", 1, hq, max(1, hq // 4), n, d, window, 4)
    c.check(c.run(hip), rows=sorted({0, 1, 31, 32, 100, 200, n // 2, n - 257, n - 33, n - 2, n - 1} & set(range(n)))
            if hq < 64 else [0, 3, n // 2, n - 1])


@pytest.mark.parametrize("d,offset,scale", [(63, 0, None), (5, 0, None), (130, 0, None), (64, 2, None), (64, 0, -0.3), (40, 0, 0.0)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_row_kernel(hip, dtype, d, offset, scale):
    """Odd head dimensions, unaligned operands, scales that are not positive: fp32
    probabilities."""
    c = Case(7, dtype, 2, 2, 1, 70, d, 20, 2, 9, None, scale)
    c.check(c.run(hip, offset=offset), p_error=0.0)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_masked_keys_do_not_count(hip, d):
    """NaN and Inf in K and V of keys that only some queries see: the others are as without
    them; those that see them are NaN, or what the formula says."""
    c = Case(8, "f16", 1, 1, 1, 300, d, 50, 2)
    for j, x in ((0, 0x7E00), (100, 0x7E00), (101, 0x7C00), (299, 0x7E00)):
        for bits, vals in ((c.kb, c.k), (c.vb, c.v)):
            if j == 101 and bits is c.kb:
                continue
            bits[0, 0, j, 3] = x
            vals[0, 0, j, 3] = np.float16(bits[0, 0, j, 3:4].view(np.float16)[0])
    got = c.run(hip)
    val = as_f64(got, "f16")[0, 0]
    sees = c.mask()
    clean = ~sees[:, [0, 100, 101, 299]].any(1)
    assert not clean.any()   # key 0 is a sink: every query sees it
    c.sinks = 0
    got = c.run(hip)
    val = as_f64(got, "f16")[0, 0]
    sees = c.mask()
    nan_k = sees[:, [0, 100, 299]].any(1)
    assert np.isnan(val[nan_k]).all()
    inf_v = sees[:, 101] & ~nan_k
    assert inf_v.any() and (np.isinf(val[inf_v][:, 3])).all() and np.isfinite(np.delete(val[inf_v], 3, 1)).all()
    clean = np.nonzero(~nan_k & ~sees[:, 101])[0]
    assert len(clean) > 50
    c.check(got, rows=clean)


def test_extreme_scores(hip):
    """Large scores, a growing maximum, and rows whose scores are all -inf (0 / 0)."""
    c = Case(9, "bf16", 1, 1, 1, 400, 64, 60, 0, scale=20.0)
    c.check(c.run(hip))
    c = Case(10, "f16", 1, 1, 1, 400, 64, 300, 1)
    c.q[..., 0], c.k[..., 0] = 8.0, np.float16(np.linspace(0, 60, 400))[None, None]
    c.qb, c.kb = f16_round(c.q)[0], f16_round(c.k)[0]
    c.check(c.run(hip))
    c = Case(11, "f16", 1, 1, 1, 100, 64, 10, 0)
    c.q[:], c.k[..., 0] = 0, -np.inf
    c.q[..., 0] = 1
    c.k[0, 0, 50:, 0] = 1
    c.qb, c.kb = f16_round(c.q)[0], f16_round(c.k)[0]
    c.check(c.run(hip))


def test_far_below_the_maximum(hip):
    """Many keys at 2^-15 of the maximum's weight: f16 probabilities keep their bits."""
    c = Case(12, "f16", 1, 1, 1, 4000, 64, 4000, 0)
    c.q[:], c.k[:] = 0, 0
    c.q[..., 0] = 8
    c.k[0, 0, 0, 0] = 8
    c.scale = 15.3 * np.log(2) / 64
    c.v[:] = 1.0 + (np.arange(64) / 64)
    c.v[0, 0, 0] = -4.0
    c.qb, c.kb, c.vb = (f16_round(x)[0] for x in (c.q, c.k, c.v))
    c.check(c.run(hip), rows=[0, 1, 63, 64, 1000, 3998, 3999])


def test_same_as_causal_attention(hip):
    """A window over everything is the causal kernel's result, within both's rounding."""
    c = Case(13, "f16", 1, 4, 4, 300, 128, 300)
    got = as_f64(c.run(hip), "f16")
    bufs = [hip.DeviceBuffer.from_array(x) for x in (c.qb, c.kb, c.vb)]
    o = hip.DeviceBuffer(c.qb.nbytes)
    hip.flash_attn_fwd(hip.F16, 1, 4, 300, 128, *(x.ptr for x in bufs), o.ptr, c.scale, True)
    hip.synchronize()
    ref = as_f64(o.download(np.uint16, c.qb.shape), "f16")
    c.check(c.run(hip))
    assert np.abs(got - ref).max() <= 4 * 2.0 ** -11 * np.abs(c.v).max()


def test_stream_and_graph(hip):
    c = Case(14, "bf16", 2, 4, 2, 333, 64, 77, 3, 20)
    want = c.run(hip)
    st = hip.Stream()
    assert (c.run(hip, st) == want).all()
    bufs = [hip.DeviceBuffer.from_array(x) for x in (c.qb, c.kb, c.vb)]
    o = hip.DeviceBuffer(c.qb.nbytes)
    args = (hip.BF16, 2, 4, 2, 333, 353, 64, *(x.ptr for x in bufs), o.ptr, c.scale, 20, 77, 3, st)
    with hip.Graph(st) as graph:
        hip.flash_attn_window_fwd(*args)
    for rep in range(3):
        o.fill_bytes(0xFF)
        hip.synchronize()
        graph.launch()
        st.synchronize()
        assert (o.download(np.uint16, c.qb.shape) == want).all(), rep
        c.run(hip)
    graph.close()
    st.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 72, 128])
@pytest.mark.parametrize("hq,hkv,n,window", [
    (48, 16, 700, 100), (32, 16, 1100, 100), (16, 4, 2100, 100),    # one key group; 1, 2 and 4 query heads a workgroup
    (8, 8, 2100, 300), (8, 4, 2100, 300), (8, 2, 2100, 300),        # two
    (2, 2, 777, 500), (4, 2, 500, 400), (3, 1, 900, 700)])          # four; 1, 2 and 1 query heads
def test_every_layout(hip, dtype, d, hq, hkv, n, window):
    """What window_plan chooses on 256 CUs: every number of key groups, with every number
    of query heads a workgroup takes, in each width up to 128; rows at the edges of
    blocks and of the window, in every head."""
    c = Case(15, dtype, 1, hq, hkv, n, d, window, 4)
    at = {0, 1, 31, 32, 33, 63, 64, 65, 127, 128, window - 1, window, window + 1, n // 2, n - 65, n - 33, n - 32, n - 2, n - 1}
    c.check(c.run(hip), rows=sorted(at))


def test_more_rows_than_a_launch_takes(hip):
    """Query rows past 2^25 on the row kernel (an odd head dimension) and past 2^24 blocks on
    the matrix cores: the calls an aligned or a smaller one takes, and every row written."""
    r = rng(16)
    n, d = (1 << 25) + 77, 3
    q = r.integers(-8, 8, (n, d), dtype=np.int16).astype(np.float16)
    say(f"window f16 1x1 q={n} d={d} w=2")
    buf = hip.DeviceBuffer.from_array(q.view(np.uint16))
    o = hip.DeviceBuffer(q.nbytes)
    o.fill_bytes(0xFF)
    hip.flash_attn_window_fwd(hip.F16, 1, 1, 1, n, n, d, buf.ptr, buf.ptr, buf.ptr, o.ptr, 0.25, 0, 2)
    hip.synchronize()
    got = o.download(np.float16, (n, d))
    assert np.isfinite(got).all()
    for i in (0, 1, 2, (1 << 24) - 1, 1 << 24, (1 << 25) - 1, 1 << 25, n - 2, n - 1):
        x = q[max(0, i - 1):i + 1].astype(np.float64)
        ref, spread, size = paged_ref.attention(x[-1], x, x, 0.25)
        assert (np.abs(got[i] - ref) <= paged_ref.error_bound(ref, spread, size, "f16", d, 2, 0.0)).all(), i
    buf.close()
    o.close()
    # one query and one key a head: the result is V's row
    b, d = (1 << 24) + 5, 8
    say(f"window f16 {b}x1 q=1 d={d}")
    bits = r.integers(0, 0x7C00, (1 << 20) * d, dtype=np.uint16)
    v = np.resize(bits, b * d)
    dv, o = hip.DeviceBuffer.from_array(v), hip.DeviceBuffer(v.nbytes)
    o.fill_bytes(0xFF)
    hip.flash_attn_window_fwd(hip.F16, b, 1, 1, 1, 1, d, dv.ptr, dv.ptr, dv.ptr, o.ptr, 1e-4, 0, 1)
    hip.synchronize()
    got = o.download(np.float16, v.shape).astype(np.float32)
    want = v.view(np.float16).astype(np.float32)
    assert (np.abs(got - want) <= 2.0 ** -11 * want + 2.0 ** -25).all()
    dv.close()
    o.close()
