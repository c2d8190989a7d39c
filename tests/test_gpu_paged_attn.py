"""GPU: attention of one new token a row over the paged cache, against numpy in 64
bits with a bound derived from the arithmetic (paged_ref.error_bound).  Every slot
that the token does not see holds NaN, so that a read that counts shows."""
import numpy as np
import pytest

from oracle import cpuref
from tests import paged_ref
from tests.helpers import bf16_round, f16_round, rng, say

pytestmark = pytest.mark.gpu

NAN16 = {"f16": 0x7E00, "bf16": 0x7FC0}
P_ERROR = {"f16": 2.0 ** -21, "bf16": 2.0 ** -17}   # two parts: half a step of half a step


def rounded(x, dtype):
    return f16_round(x) if dtype == "f16" else bf16_round(x)


def as_f32(bits, dtype):
    return bits.view(np.float16).astype(np.float32) if dtype == "f16" else cpuref.f32_from_bf16(bits)


class Case:
    """A cache of random rows and one query token for each, on the host."""

    def __init__(self, seed, dtype, lengths, hq, hkv, d, page, window=0, sinks=0, fp8=False,
                 pad_page=0, ldq_pad=0, scale=None, spare=3, width_pad=1):
        r = rng(seed)
        self.r, self.dtype, self.fp8, self.d, self.page = r, dtype, fp8, d, page
        self.hq, self.hkv, self.window, self.sinks = hq, hkv, window, sinks
        self.lengths, self.b = list(lengths), len(lengths)
        self.scale = d ** -0.5 if scale is None else scale
        self.k_scale, self.v_scale = (0.03125, 0.025) if fp8 else (1.0, 1.0)
        pages = [-(-max(n, 0) // page) for n in self.lengths]
        self.width = max(pages + [1]) + width_pad
        self.num = sum(pages) + spare
        self.stride = hkv * page * d + pad_page
        ids = r.permutation(self.num).astype(np.int32)
        self.tables = np.full((self.b, self.width), -1, np.int32)
        at = 0
        for i, n in enumerate(pages):
            self.tables[i, :n] = ids[at:at + n]
            at += n
        self.ldq = hq * d + ldq_pad
        q = r.normal(size=(self.b, self.ldq)).astype(np.float32)
        self.q_bits, q = rounded(q, dtype)
        self.q = q[:, :hq * d].reshape(self.b, hq, d)
        nan = 0x7F if fp8 else NAN16[dtype]
        self.pools = [np.full((self.num, self.stride), nan, np.uint8 if fp8 else np.uint16) for _ in "kv"]
        self.kv = []   # per row: K, V [hkv, n, d] fp32, as the cache holds them
        for i, n in enumerate(self.lengths):
            n = max(n, 0)
            both = []
            for pool, sc in zip(self.pools, (self.k_scale, self.v_scale)):
                x = r.normal(size=(hkv, n, d)).astype(np.float32)
                if fp8:
                    bits = cpuref.e4m3_encode(x, sc)
                    x = cpuref.e4m3_decode(bits, sc)
                else:
                    bits, x = rounded(x, dtype)
                seen = np.zeros(n, bool)
                seen[paged_ref.seen_keys(n, window, sinks)] = True
                view = pool[:, :hkv * page * d].reshape(self.num, hkv, page, d)
                for j in np.nonzero(seen)[0]:
                    view[self.tables[i, j // page], :, j % page] = bits[:, j]
                both.append(x)
            self.kv.append(both)

    def reference(self, i, h, gone=()):
        """Row i, query head h: value and bound; keys of the pages `gone` (table
        entries) do not count."""
        n = max(self.lengths[i], 0)
        at = [j for j in paged_ref.seen_keys(n, self.window, self.sinks) if j // self.page not in gone]
        k, v = (x[h // (self.hq // self.hkv)][at] for x in self.kv[i])
        ref, spread, size = paged_ref.attention(self.q[i, h], k, v, self.scale)
        return ref, paged_ref.error_bound(ref, spread, size, self.dtype, self.d, len(at), P_ERROR[self.dtype])

    def upload(self, hip):
        b = hip.DeviceBuffer.from_array
        self.dq, self.dk, self.dv = b(self.q_bits), b(self.pools[0]), b(self.pools[1])
        self.dt, self.dl = b(self.tables), b(np.array(self.lengths, np.int32))
        self.ldo = self.hq * self.d + 16
        self.do = hip.DeviceBuffer((self.b + 1) * self.ldo * 2)
        self.do.fill_bytes(0x5A)
        self.ws = hip.DeviceBuffer(hip.paged_attn_workspace(self.b, self.hq, self.hkv, self.d))
        self.ws.fill_bytes(0xFF)

    def run(self, hip, stream=None, **over):
        t = hip.F16 if self.dtype == "f16" else hip.BF16
        a = dict(q=self.dq.ptr, k=self.dk.ptr, v=self.dv.ptr, tables=self.dt.ptr, num=self.num,
                 width=self.width, ws=self.ws.ptr, ws_bytes=self.ws.nbytes)
        a.update(over)
        hip.paged_attn_decode(t, hip.F8E4M3 if self.fp8 else t, self.b, self.hq, self.hkv, self.d, a["q"],
                              self.ldq, a["k"], a["v"], a["num"], self.page, self.stride, a["tables"],
                              a["width"], self.dl.ptr, self.do.ptr, self.ldo, self.scale, self.k_scale,
                              self.v_scale, self.window, self.sinks, a["ws"], a["ws_bytes"], stream)

    def result(self, hip):
        hip.synchronize()
        o = self.do.download(np.uint16, (self.b + 1, self.ldo))
        assert (o[self.b:] == 0x5A5A).all() and (o[:, self.hq * self.d:] == 0x5A5A).all(), "wrote past the rows"
        return o[:self.b, :self.hq * self.d].reshape(self.b, self.hq, self.d)

    def check(self, got, what, gone=None):
        val = as_f32(got, self.dtype).astype(np.float64)
        for i in range(self.b):
            for h in range(self.hq):
                ref, bound = self.reference(i, h, (gone or {}).get(i, ()))
                err = np.abs(val[i, h] - ref)
                assert (err <= bound).all(), (what, i, h, float(np.nanmax(err / bound)), val[i, h][:4], ref[:4])


LENGTHS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 1000]


def run_case(hip, case, what):
    say(what)
    case.upload(hip)
    case.run(hip)
    got = case.result(hip)
    case.check(got, what)
    return got


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 80, 128, 144, 256])
def test_head_dims(hip, dtype, d, fp8):
    run_case(hip, Case(1, dtype, LENGTHS, 4, 2, d, 16, fp8=fp8), f"paged attn {dtype} d={d} fp8={fp8}")


@pytest.mark.parametrize("d", [8, 24, 72, 136, 248])
def test_head_dims_odd_multiples_of_8(hip, d):
    run_case(hip, Case(2, "bf16", LENGTHS, 3, 1, d, 16), f"paged attn bf16 d={d}")


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (5, 1), (16, 1), (17, 1), (32, 2), (33, 1), (70, 2)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_head_groups(hip, hq, hkv, d):
    run_case(hip, Case(3, "f16", [5, 0, 200, 77], hq, hkv, d, 32), f"paged attn heads {hq}/{hkv} d={d}")


@pytest.mark.parametrize("page", [1, 2, 4, 8, 64, 128, 1024])
@pytest.mark.parametrize("fp8", [False, True])
def test_page_sizes(hip, page, fp8):
    run_case(hip, Case(4, "bf16", [1, 40, 0, 333, 129], 4, 2, 64, page, fp8=fp8), f"paged attn page={page} fp8={fp8}")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (32, 0), (33, 31), (100, 40), (100, 500),
                                          (1000, 7), (5000, 3), (64, 64)])
@pytest.mark.parametrize("page", [8, 64])
def test_window_and_sinks(hip, window, sinks, page):
    run_case(hip, Case(5, "f16", LENGTHS, 4, 2, 64, page, window, sinks),
             f"paged attn window={window} sinks={sinks} page={page}")


@pytest.mark.parametrize("hq,hkv", [(4, 2), (16, 1), (17, 1), (33, 1), (40, 2)])
@pytest.mark.parametrize("d,page,fp8", [(64, 16, False), (64, 4, True), (80, 64, False), (128, 32, True), (128, 8, False),
                                        (104, 2, False), (256, 16, False), (176, 128, True)])
def test_rows_split_over_workgroups(hip, hq, hkv, d, page, fp8):
    """Every instance with rows long enough to be dealt out and joined: each page size's
    addressing, one and two query tiles, head groups past them."""
    run_case(hip, Case(20, "bf16", [1500, 0, 3, 700, 129], hq, hkv, d, page, fp8=fp8),
             f"paged attn split {hq}/{hkv} d={d} page={page} fp8={fp8}")


@pytest.mark.parametrize("window,sinks", [(600, 0), (600, 70), (1000, 1), (513, 2000), (2000, 33)])
def test_windows_dealt_out(hip, window, sinks):
    run_case(hip, Case(21, "f16", [0, 5, 599, 600, 601, 700, 1500, 4000], 6, 2, 72, 16, window, sinks),
             f"paged attn dealt window={window} sinks={sinks}")


@pytest.mark.parametrize("batch", [1, 64, 200, 257, 520])
def test_short_rows_a_workgroup_each(hip, batch):
    """A table of 512 keys at most (a workgroup a unit), and one past it."""
    lengths = [int(n) for n in rng(22).integers(0, 300, batch)]
    run_case(hip, Case(22, "f16", lengths, 2, 1, 64, 32), f"paged attn {batch} short rows")
    lengths[batch // 2] = 1100
    run_case(hip, Case(23, "f16", lengths, 2, 1, 64, 32), f"paged attn {batch} rows, one of 1100")


def test_many_rows_and_one_long_one(hip):
    """More rows than a workgroup has threads, most of them short or empty."""
    lengths = [int(n) for n in rng(6).integers(0, 40, 700)]
    lengths[333] = 9000
    run_case(hip, Case(6, "bf16", lengths, 2, 1, 64, 16), "paged attn 700 rows")


def test_long_row_split_over_workgroups(hip):
    """A row of 40001 keys is shared by all workgroups; the same call twice gives the
    same bits."""
    case = Case(7, "f16", [40001], 4, 1, 128, 64)
    got = run_case(hip, case, "paged attn 1 x 40001")
    case.do.fill_bytes(0x5A)
    case.run(hip)
    assert (case.result(hip) == got).all()


def test_strides(hip):
    """Pages further apart than they are long, query rows in a wider pitch."""
    run_case(hip, Case(8, "bf16", [90, 5, 260], 6, 2, 80, 16, pad_page=2 * 16 * 80 + 8, ldq_pad=24),
             "paged attn strides")


def test_negative_scale_and_large_scores(hip):
    run_case(hip, Case(9, "f16", [50, 400], 4, 2, 64, 16, scale=-0.2), "paged attn negative scale")
    run_case(hip, Case(10, "bf16", [50, 400], 4, 2, 64, 16, scale=30.0), "paged attn large scores")


def test_far_below_the_maximum(hip):
    """One key with nearly all the weight and 60000 whose 2^-19th parts add up: they
    keep their precision in 16-bit probabilities."""
    case = Case(11, "f16", [60001], 1, 1, 64, 64)
    k, v = case.kv[0]
    k[:], v[:] = 0, 1.0 + (np.arange(64) / 64)[None, None]
    k[0, 777, 0], v[0, 777] = 8.0, -4.0
    case.q[:] = 0
    case.q[0, 0, 0] = 8.0
    case.scale = 19.2 * np.log(2) / 64
    case.q_bits = f16_round(case.q.reshape(1, -1))[0]
    for pool, x in zip(case.pools, case.kv[0]):
        bits = f16_round(x)[0]
        view = pool[:, :64 * 64].reshape(case.num, 1, 64, 64)
        for j in range(60001):
            view[case.tables[0, j // 64], :, j % 64] = bits[:, j]
    run_case(hip, case, "paged attn far below the maximum")


def test_pages_that_do_not_exist(hip):
    """Entries outside the pool, lengths below zero and past the table: left out."""
    case = Case(12, "f16", [100, 64, 33, 0, 200], 4, 2, 64, 16, width_pad=0)
    case.tables[0, 2], case.tables[0, 6] = -1, case.num
    case.tables[1, :] = [2 ** 31 - 1, -2 ** 31, case.num, -7] + [-1] * (case.width - 4)
    case.tables[2, 0] = -1
    real = list(case.lengths)
    case.lengths = [100, 64, 33, -5, 10 ** 9]
    case.upload(hip)
    say("paged attn bad pages")
    case.run(hip)
    got = case.result(hip)
    case.lengths = real[:4] + [case.width * 16]
    # the last row's length counts as the table's: its keys past 200 lie in entries of -1
    # and in slots of NaN behind key 200 of its last page, which it now sees
    case.lengths[4] = 200
    case.b = 4
    case.check(got, "bad pages", gone={0: (2, 6), 1: (0, 1, 2, 3), 2: (0,)})
    assert (got[1] == 0).all() and (got[3] == 0).all()
    assert np.isnan(as_f32(got[4], "f16")).all()   # 200 = 12.5 pages: slots of NaN are seen


def test_no_page_at_all(hip):
    case = Case(13, "bf16", [7, 0], 2, 1, 64, 16)
    case.upload(hip)
    say("paged attn empty pool")
    case.run(hip, num=0, k=None, v=None)
    assert (case.result(hip) == 0).all()
    case.do.fill_bytes(0x5A)
    case.run(hip, width=0, tables=None)
    assert (case.result(hip) == 0).all()


def test_infinite_scores(hip):
    """All scores of a row -inf: 0 / 0 as the formula says; some: they weigh nothing."""
    case = Case(14, "f16", [40, 40], 1, 1, 64, 16)
    q = np.zeros((2, 64), np.float32)
    q[:, 0] = 1
    case.q_bits, case.q = f16_round(q)[0], q.reshape(2, 1, 64)
    for i, at in ((0, range(40)), (1, range(0, 40, 3))):
        view = case.pools[0].reshape(case.num, 1, 16, 64)
        for j in at:
            view[case.tables[i, j // 16], 0, j % 16, 0] = 0xFC00
            case.kv[i][0][0, j, 0] = -np.inf
    case.upload(hip)
    say("paged attn -inf scores")
    case.run(hip)
    got = case.result(hip)
    assert np.isnan(as_f32(got[0], "f16")).all()
    keep = [j for j in range(40) if j % 3]
    ref, spread, size = paged_ref.attention(case.q[1, 0], case.kv[1][0][0, keep], case.kv[1][1][0, keep], case.scale)
    bound = paged_ref.error_bound(ref, spread, size, "f16", 64, 40, P_ERROR["f16"])
    assert (np.abs(as_f32(got[1, 0], "f16") - ref) <= bound).all()


def test_offsets_past_32_bits(hip):
    """Pages 2^30 bytes apart: the last ones lie past 4 GiB."""
    say("paged attn offsets past 4 GiB")
    case = Case(15, "bf16", [70, 33], 2, 1, 64, 16, spare=1)
    stride = 1 << 29
    big = hip.DeviceBuffer((case.num * stride) * 2 + (1 << 20))
    for i in range(case.num):
        for at, pool in ((0, case.pools[0]), (4096, case.pools[1])):
            hip.call("sile_hip_memcpy_htod", big.ptr + 2 * (i * stride + at), pool[i].ctypes.data, pool[i].nbytes)
    case.upload(hip)
    case.stride = stride
    case.run(hip, k=big.ptr, v=big.ptr + 8192)
    case.check(case.result(hip), "far pages")
    big.close()


def test_other_stream_and_graph(hip):
    """Captured once, replayed with other lengths, tables and cache contents, eager work
    in between; each replay is the eager call's bits."""
    say("paged attn graph")
    st = hip.Stream()
    first = Case(16, "bf16", [300, 0, 77, 12], 8, 2, 128, 16, spare=40, width_pad=20)
    other = Case(17, "bf16", [5, 600, 0, 33], 8, 2, 128, 16, spare=20, width_pad=1)
    first.upload(hip)
    first.run(hip, st)
    st.synchronize()
    first.check(first.result(hip), "on a stream")
    with hip.Graph(st) as graph:
        first.run(hip, st)
    assert other.width <= first.width and other.num <= first.num, (first.width, other.width, first.num, other.num)
    for rep, case in enumerate((first, other, first, other)):
        tables = np.full((4, first.width), -1, np.int32)
        tables[:, :case.width] = case.tables
        first.dt.upload(tables)
        first.dl.upload(np.array(case.lengths, np.int32))
        for buf, pool in ((first.dk, case.pools[0]), (first.dv, case.pools[1])):
            buf.upload(pool[:first.num])
        first.dq.upload(case.q_bits)
        first.do.fill_bytes(0x5A)
        hip.synchronize()
        graph.launch()
        st.synchronize()
        got = first.result(hip)
        case.check(got, f"replay {rep}")
        first.do.fill_bytes(0x5A)
        first.run(hip)
        assert (first.result(hip) == got).all(), f"replay {rep} against eager"
    graph.close()
    st.close()


def test_refusals(hip):
    case = Case(18, "f16", [10], 2, 1, 64, 16)
    case.upload(hip)
    for over, needle in (({"ws_bytes": case.ws.nbytes - 1}, "workspace"), ({"ws": None}, "workspace"),
                         ({"ws": case.ws.ptr + 4}, "aligned"), ({"q": case.dq.ptr + 2}, "aligned"),
                         ({"tables": None}, "NULL")):
        with pytest.raises(hip.SileError, match=needle):
            case.run(hip, **over)
    hip.synchronize()
    assert (case.do.download(np.uint16, (2, case.ldo)) == 0x5A5A).all()


INF16 = {"f16": 0x7C00, "bf16": 0x7F80}


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lengths,hq,hkv,d,page,window,sinks", [
    ([1, 2, 40, 0, 300], 4, 2, 64, 16, 0, 0), ([1, 77], 3, 1, 128, 8, 0, 0), ([1, 200, 33], 20, 1, 80, 32, 0, 0),
    ([500, 65], 6, 2, 256, 16, 60, 3), ([700, 1, 5000, 64], 4, 2, 128, 16, 0, 0), ([3000, 1], 40, 2, 64, 4, 0, 0),
    ([20001], 4, 1, 72, 64, 0, 0), ([4000, 900, 5], 17, 1, 104, 16, 700, 40), ([1500, 2500], 5, 1, 256, 128, 0, 0)])
def test_values_that_are_not_finite(hip, dtype, lengths, hq, hkv, d, page, window, sinks):
    """Inf and NaN in V of keys that the token sees, in rows of one workgroup and in rows
    dealt out and joined: in their own dimension the result is what the formula gives
    (Inf of a sign, or NaN where Inf meets -Inf or NaN is there), and the others are as
    without them."""
    case = Case(24, dtype, lengths, hq, hkv, d, page, window, sinks)
    view = case.pools[1].reshape(case.num, hkv, page, d)
    inf, nan, neg = INF16[dtype], NAN16[dtype], 0x8000
    for i, n in enumerate(lengths):
        at = paged_ref.seen_keys(n, window, sinks)
        if len(at) == 0:
            continue
        mid = at[len(at) // 2]
        for h in range(hkv):
            for j, dim, bits in ((at[0], 3, inf), (at[-1], 5, inf | neg), (mid, 2, inf), (mid, 7, nan),
                                 (at[0], d - 1, inf), (at[-1], d - 1, inf | neg)):
                if h and dim == 3:
                    continue   # another key head: other dimensions
                view[case.tables[i, j // page], h, j % page, dim] = bits
                case.kv[i][1][h, j, dim] = as_f32(np.array([bits], np.uint16), dtype)[0]
    say(f"paged attn Inf in V {dtype} {lengths} {hq}/{hkv} d={d} page={page} window={window}")
    case.upload(hip)
    case.run(hip)
    got = as_f32(case.result(hip), dtype).astype(np.float64)
    for i in range(case.b):
        for h in range(hq):
            with np.errstate(invalid="ignore"):
                ref, bound = case.reference(i, h)
                err = np.abs(got[i, h] - ref)
            same = (got[i, h] == ref) | (np.isnan(got[i, h]) & np.isnan(ref))
            assert (same | (np.isfinite(ref) & (err <= bound))).all(), (i, h, got[i, h][:8], ref[:8])
            assert lengths[i] == 0 or np.isinf(ref).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,page", [(2, 1, 64, 16), (40, 2, 72, 4), (5, 1, 256, 32)])
def test_values_that_are_not_finite_in_some_of_many_rows(hip, dtype, hq, hkv, d, page):
    """Several whole rows a workgroup, every third with an Inf in V, every seventh with a NaN in
    K (which makes all of the row's head NaN), beside one that is dealt out."""
    lengths = [int(n) for n in rng(25).integers(0, 50, 400)]
    lengths[100] = 3000
    case = Case(25, dtype, lengths, hq, hkv, d, page)
    views = [pool.reshape(case.num, hkv, page, d) for pool in case.pools]
    for i, n in enumerate(lengths):
        for which, every, dim, bits in ((1, 3, i % d, INF16[dtype]), (0, 7, 1, NAN16[dtype])):
            if n and i % every == 1:
                h, j = i % hkv, i % n
                views[which][case.tables[i, j // page], h, j % page, dim] = bits
                case.kv[i][which][h, j, dim] = as_f32(np.array([bits], np.uint16), dtype)[0]
    say(f"paged attn Inf in V of some of 400 rows {dtype} {hq}/{hkv} d={d} page={page}")
    case.upload(hip)
    case.run(hip)
    got = as_f32(case.result(hip), dtype).astype(np.float64)
    infs = 0
    for i in range(case.b):
        for h in range(hq):
            with np.errstate(invalid="ignore"):
                ref, bound = case.reference(i, h)
                err = np.abs(got[i, h] - ref)
            same = (got[i, h] == ref) | (np.isnan(got[i, h]) & np.isnan(ref))
            assert (same | (np.isfinite(ref) & (err <= bound))).all(), (i, h, got[i, h][:8], ref[:8])
            infs += int(np.isinf(ref).any())
    assert infs > 100


@pytest.mark.parametrize("lengths", [[1, 40, 300], [3000, 2, 700]])
@pytest.mark.parametrize("page", [8, 32])
def test_nan_codes(hip, lengths, page):
    """An e4m3 cache (which has no Inf): NaN in V stays in its dimension, NaN in K takes its key
    head's row."""
    case = Case(26, "bf16", lengths, 6, 2, 64, page, fp8=True)
    kp, vp = (pool.reshape(case.num, 2, page, 64) for pool in case.pools)
    for i, n in enumerate(lengths):
        j = n // 2
        at = case.tables[i, j // page]
        vp[at, 0, j % page, 5] = 0xFF
        case.kv[i][1][0, j, 5] = np.nan
        if i == 1:
            kp[at, 1, j % page, 9] = 0x7F
    say(f"paged attn NaN codes {lengths} page={page}")
    case.upload(hip)
    case.run(hip)
    got = as_f32(case.result(hip), "bf16").astype(np.float64)
    for i in range(case.b):
        for h in range(6):
            if i == 1 and h >= 3:
                assert np.isnan(got[i, h]).all()
                continue
            ref, bound = case.reference(i, h)
            assert (np.isnan(got[i, h]) == np.isnan(ref)).all() and np.isnan(ref).sum() == (h < 3), (i, h)
            ok = ~np.isnan(ref)
            assert (np.abs(got[i, h] - ref)[ok] <= bound[ok]).all(), (i, h)
