"""GPU: attention of pieces of prompts and single tokens over the paged cache, against numpy in 64
bits with a bound derived from the arithmetic (paged_ref.error_bound, with probabilities of 16
bits).  Slots that no token sees hold NaN, so that a read that counts shows."""
import ctypes

import numpy as np
import pytest

from oracle import cpuref
from tests import paged_ref
from tests.helpers import bf16_round, f16_round, rng, say

pytestmark = pytest.mark.gpu

NAN16 = {"f16": 0x7E00, "bf16": 0x7FC0}
P_ERROR = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def rounded(x, dtype):
    return f16_round(x) if dtype == "f16" else bf16_round(x)


def as_f32(bits, dtype):
    return bits.view(np.float16).astype(np.float32) if dtype == "f16" else cpuref.f32_from_bf16(bits)


class Case:
    """Sequences of (new tokens, keys with them), their cache and their queries, on the host."""

    def __init__(self, seed, dtype, seqs, hq, hkv, d, page, window=0, sinks=0, fp8=False, pad_page=0, pad_q=0, scale=None,
                 spare=3, tail=2, width_pad=1, spread=1.0):
        r = rng(seed)
        self.r, self.dtype, self.fp8, self.d, self.page = r, dtype, fp8, d, page
        self.hq, self.hkv, self.window, self.sinks, self.tail = hq, hkv, window, sinks, tail
        self.seqs, self.b = list(seqs), len(seqs)
        self.scale = d ** -0.5 if scale is None else scale
        self.k_scale, self.v_scale = (0.03125, 0.025) if fp8 else (1.0, 1.0)
        lengths = [max(n, 0) for _, n in self.seqs]
        pages = [-(-n // page) for n in lengths]
        self.width = max(pages + [1]) + width_pad
        self.num = sum(pages) + spare
        self.stride = hkv * page * d + pad_page
        ids = r.permutation(self.num).astype(np.int32)
        self.tables = np.full((self.b, self.width), -1, np.int32)
        at = 0
        for i, n in enumerate(pages):
            self.tables[i, :n] = ids[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in self.seqs])]).astype(np.int32)
        self.n = int(self.starts[-1]) + tail
        self.ldq = hq * d + pad_q
        self.q_bits, q = rounded(r.normal(size=(self.n, self.ldq)).astype(np.float32) * spread, dtype)
        self.q = q[:, :hq * d].reshape(self.n, hq, d)
        nan = 0x7F if fp8 else NAN16[dtype]
        self.pools = [np.full((self.num, self.stride), nan, np.uint8 if fp8 else np.uint16) for _ in "kv"]
        self.kv = []   # per sequence: K, V [hkv, n, d] fp32, as the cache holds them
        for i, n in enumerate(lengths):
            both = []
            seen = np.zeros(n, bool)
            for p in range(max(n - self.seqs[i][0], 0), n):
                seen[self.keys(p)] = True
            for pool, sc in zip(self.pools, (self.k_scale, self.v_scale)):
                x = r.normal(size=(hkv, n, d)).astype(np.float32)
                if fp8:
                    bits = cpuref.e4m3_encode(x, sc)
                    x = cpuref.e4m3_decode(bits, sc)
                else:
                    bits, x = rounded(x, dtype)
                view = pool[:, :hkv * page * d].reshape(self.num, hkv, page, d)
                j = np.nonzero(seen)[0]
                view[self.tables[i, j // page], :, j % page] = bits[:, j].transpose(1, 0, 2)
                both.append(x)
            self.kv.append(both)

    def keys(self, p):
        j = np.arange(p + 1)
        return j if self.window <= 0 else j[(j > p - self.window) | (j < self.sinks)]

    def upload(self, hip):
        b = hip.DeviceBuffer.from_array
        self.dq, self.dk, self.dv = b(self.q_bits), b(self.pools[0]), b(self.pools[1])
        self.dt, self.dl, self.ds = b(self.tables), b(np.array([n for _, n in self.seqs], np.int32)), b(self.starts)
        self.ldo = self.hq * self.d + 16
        self.do = hip.DeviceBuffer((self.n + 1) * self.ldo * 2)
        self.do.fill_bytes(0x5A)
        self.ws = hip.DeviceBuffer(hip.paged_attn_chunk_workspace(self.b, self.n, self.hq, self.hkv, self.d))
        self.ws.fill_bytes(0xFF)

    def run(self, hip, stream=None, **over):
        t = hip.F16 if self.dtype == "f16" else hip.BF16
        a = dict(q=self.dq.ptr, k=self.dk.ptr, v=self.dv.ptr, tables=self.dt.ptr, num=self.num, width=self.width,
                 stride=self.stride, scale=self.scale)
        a.update(over)
        hip.paged_attn_chunk(t, hip.F8E4M3 if self.fp8 else t, self.b, self.n, self.hq, self.hkv, self.d, a["q"], self.ldq,
                             self.ds.ptr, a["k"], a["v"], a["num"], self.page, a["stride"], a["tables"], a["width"],
                             self.dl.ptr, self.do.ptr, self.ldo, a["scale"], self.k_scale, self.v_scale, self.window,
                             self.sinks, self.ws.ptr, self.ws.nbytes, stream)

    def result(self, hip):
        hip.synchronize()
        o = self.do.download(np.uint16, (self.n + 1, self.ldo))
        assert (o[self.starts[-1]:] == 0x5A5A).all() and (o[:, self.hq * self.d:] == 0x5A5A).all(), "wrote past the rows"
        return o[:self.n, :self.hq * self.d].reshape(self.n, self.hq, self.d)

    def check(self, got, what, gone=None, heads=None, scale=None):
        """gone: {sequence: table entries whose pages do not count}."""
        val = as_f32(got, self.dtype).astype(np.float64)
        scale = self.scale if scale is None else scale
        for i, (new, n) in enumerate(self.seqs):
            n = max(n, 0)
            for t in range(new):
                p = n - new + t
                at = self.keys(p) if p >= 0 else np.zeros(0, int)
                at = np.array([j for j in at if j // self.page not in (gone or {}).get(i, ())], int)
                row = self.starts[i] + t
                for h in (range(self.hq) if heads is None else heads):
                    k, v = (x[h // (self.hq // self.hkv)][at] for x in self.kv[i])
                    ref, spread, size = paged_ref.attention(self.q[row, h], k, v, scale)
                    bound = paged_ref.error_bound(ref, spread, size, self.dtype, self.d, len(at), P_ERROR[self.dtype])
                    if self.dtype == "f16" and len(at):
                        # probabilities below the least f16 step, 2^-25 under a factor 2^7 and with a sum of
                        # at least 1, and once more in that sum
                        bound = bound + 2 * len(at) * 2.0 ** -32 * np.abs(v).max(0)
                    err = np.abs(val[row, h] - ref)
                    assert (err <= bound).all(), (what, i, t, h, float(np.nanmax(err / bound)), val[row, h][:4], ref[:4])


def run_case(hip, case, what, **kw):
    say(what)
    case.upload(hip)
    case.run(hip)
    case.check(case.result(hip), what, **kw)


SEQS = {"one": [(1, 1)], "first": [(5, 5), (33, 33), (1, 64)], "piece": [(70, 300)], "mixed": [(1, 700), (0, 9), (40, 40), (3, 1000), (1, 1)],
        "singles": [(1, n) for n in (1, 31, 32, 33, 64, 65, 100, 127, 128, 500)], "long": [(2, 5000)], "before": [(9, 4), (3, 0), (2, -1), (4, 4)]}


@pytest.mark.parametrize("dtype,fp8", [("f16", False), ("bf16", False), ("f16", True), ("bf16", True)])
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 64), (8, 2, 128), (3, 3, 256)])
@pytest.mark.parametrize("seqs", list(SEQS))
def test_chunk(hip, dtype, fp8, hq, hkv, d, seqs):
    run_case(hip, Case(len(seqs) + d, dtype, SEQS[seqs], hq, hkv, d, 16, fp8=fp8), f"chunk {dtype} fp8={fp8} {hq}/{hkv} x {d} {seqs}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,page", [(5, 1, 80, 16), (6, 2, 96, 32), (2, 2, 8, 16), (24, 1, 72, 8), (1, 1, 120, 64), (10, 2, 136, 16),
                                           (7, 1, 248, 128), (4, 4, 40, 1), (8, 2, 128, 1), (8, 2, 128, 2), (4, 1, 64, 4), (2, 1, 256, 1),
                                           (40, 1, 64, 16), (200, 1, 64, 16)])
def test_chunk_shapes(hip, dtype, hq, hkv, d, page):
    case = Case(hq + d, dtype, [(37, 150), (1, 90), (6, 6)], hq, hkv, d, page, pad_page=64, pad_q=24)
    run_case(hip, case, f"chunk {dtype} {hq}/{hkv} x {d}, pages of {page}")


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 0), (32, 4), (100, 33), (300, 1), (64, 500), (5000, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_chunk_window(hip, fp8, window, sinks, d):
    case = Case(window + sinks, "bf16", [(50, 400), (1, 777), (130, 130), (3, 30)], 4, 2, d, 16, window=window, sinks=sinks, fp8=fp8)
    run_case(hip, case, f"chunk window {window} sinks {sinks} d {d} fp8={fp8}", heads=[0, 3])


@pytest.mark.parametrize("dtype,fp8", [("f16", False), ("bf16", True)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_chunk_over_workgroups(hip, dtype, fp8, d):
    """Long rows whose keys are shared out, beside short ones, and tiles of several pieces."""
    case = Case(d, dtype, [(3, 9000), (1, 20), (60, 4000), (1, 6001)], 4, 1, d, 32, fp8=fp8)
    run_case(hip, case, f"chunk over workgroups {dtype} d {d}")


def test_chunk_many_sequences(hip):
    """More tiles than a workgroup has threads."""
    r = rng(5)
    case = Case(5, "bf16", [(int(r.integers(0, 4)), int(r.integers(4, 60))) for _ in range(700)], 2, 1, 64, 16, width_pad=60)
    run_case(hip, case, "chunk 700 sequences")


def test_chunk_missing_pages(hip):
    """Entries that name no page count as unseen, also in blocks that all rows would see whole."""
    for d, fp8 in ((128, False), (64, True)):
        case = Case(3, "f16", [(40, 900), (2, 200), (5, 20)], 4, 1, d, 16, fp8=fp8)
        gone = {0: {0, 7, 8, 30}, 1: set(range(13)), 2: {1}}
        for i, entries in gone.items():
            for e in entries:
                case.tables[i, e] = (-1, case.num, 2 ** 31 - 1, -(2 ** 31))[e % 4]
        run_case(hip, case, f"chunk missing pages d {d}", gone=gone)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,fp8", [("f16", False), ("bf16", False), ("bf16", True)])
def test_chunk_nan_ahead(hip, dtype, fp8, d):
    """Inf and NaN in K and V of the last tokens: the ones before them do not see it; tokens of a
    key with an Inf in V give Inf there."""
    case = Case(7, dtype, [(60, 300), (20, 2000)], 4, 2, d, 16, fp8=fp8)
    nan, inf = (0x7F, 0x7E) if fp8 else (NAN16[dtype], {"f16": 0x7C00, "bf16": 0x7F80}[dtype])
    for i, (new, n) in enumerate(case.seqs):
        for j, code in ((n - 1, nan), (n - 5, inf)):
            for pool in case.pools:
                view = pool[:, :case.hkv * case.page * d].reshape(case.num, case.hkv, case.page, d)
                if pool is case.pools[0] and code != nan:
                    continue
                view[case.tables[i, j // case.page], :, j % case.page] = code
    say(f"chunk nan ahead {dtype} fp8={fp8} d {d}")
    case.upload(hip)
    case.run(hip)
    got = as_f32(case.result(hip), dtype)
    for i, (new, n) in enumerate(case.seqs):
        rows = got[case.starts[i]:case.starts[i + 1]]
        assert np.isnan(rows[-1]).all(), "the token of the NaN key"
        if not fp8:
            assert (rows[-5:-1] == np.inf).all(), "tokens that see the Inf"
    # the tokens before them
    case.seqs = [(new - 5, n - 5) for new, n in case.seqs]
    case.starts = np.array([0, 60, 80], np.int32)
    case.check(case.do.download(np.uint16, (case.n + 1, case.ldo))[:case.n, :case.hq * d].reshape(case.n, case.hq, d), "nan ahead")


@pytest.mark.parametrize("dtype,fp8", [("f16", False), ("bf16", False), ("bf16", True)])
@pytest.mark.parametrize("d,window", [(64, 0), (80, 0), (128, 0), (128, 700), (208, 0), (256, 500)])
def test_chunk_drafts(hip, dtype, fp8, d, window):
    """A few tokens behind many: the keys of all workgroups' waves joined, with pages that are missing and a NaN that
    only the last token sees (the rows before it are taken again, in parts of their dims)."""
    case = Case(11, dtype, [(6, 3001), (1, 900), (8, 8000), (4, 4)], 4, 1, d, 16, fp8=fp8, window=window, sinks=5 if window else 0)
    gone = {0: {180, 186}, 2: {0, 470, 495}}
    for i, entries in gone.items():
        for e in entries:
            case.tables[i, e] = (-1, case.num)[e % 2]
    for i in (0, 2, 3):
        n = case.seqs[i][1] - 1
        for pool in case.pools:
            view = pool[:, :case.hkv * case.page * d].reshape(case.num, case.hkv, case.page, d)
            view[case.tables[i, n // case.page], :, n % case.page] = 0x7F if fp8 else NAN16[dtype]
    say(f"chunk drafts {dtype} fp8={fp8} d {d} window {window}")
    case.upload(hip)
    case.run(hip)
    got = as_f32(case.result(hip), dtype)
    for i in (0, 2, 3):
        assert np.isnan(got[case.starts[i + 1] - 1]).all(), "the token of the NaN key"
    case.seqs = [(new - (i != 1), n - (i != 1)) for i, (new, n) in enumerate(case.seqs)]
    case.check(case.do.download(np.uint16, (case.n + 1, case.ldo))[:case.n, :case.hq * d].reshape(case.n, case.hq, d),
               "drafts", gone=gone)


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_chunk_scales(hip, scale):
    """No scale (every key alike), a negative one, sharp ones."""
    case = Case(8, "bf16", [(20, 100), (1, 700)], 4, 2, 64, 16, scale=scale)
    run_case(hip, case, f"chunk scale {scale}")


def test_chunk_far_maximum(hip):
    """Scores that grow from block to block, past the lazy maximum, and many keys far below it."""
    for dtype in ("f16", "bf16"):
        case = Case(9, dtype, [(30, 1500)], 2, 1, 64, 16, spread=8.0)
        run_case(hip, case, f"chunk far maximum {dtype}")


def test_chunk_as_decode_and_window(hip):
    """One token a sequence is sliding, like the one-token attention; both within their bounds."""
    case = Case(10, "bf16", [(1, n) for n in (5, 300, 1111, 64)], 8, 2, 128, 16, window=200, sinks=4, tail=0)
    run_case(hip, case, "chunk of single tokens")
    ws = hip.DeviceBuffer(hip.paged_attn_workspace(4, 8, 2, 128))
    got = case.result(hip)
    case.do.fill_bytes(0x5A)
    hip.paged_attn_decode(hip.BF16, hip.BF16, 4, 8, 2, 128, case.dq.ptr, case.ldq, case.dk.ptr, case.dv.ptr, case.num, 16,
                          case.stride, case.dt.ptr, case.width, case.dl.ptr, case.do.ptr, case.ldo, case.scale, 1.0, 1.0, 200, 4,
                          ws.ptr, ws.nbytes)
    one = case.result(hip)
    case.check(one, "decode")
    # each is within its bound of the exact value: 2^-8 of a result's own rounding and 2^-7 of sum p |v|
    a, b = as_f32(got, "bf16"), as_f32(one, "bf16")
    assert np.abs(a - b).max() <= 0.05


@pytest.mark.parametrize("fp8,page", [(False, 16), (False, 2), (True, 16)])
def test_chunk_pages_past_4gib(hip, fp8, page):
    """Pages far apart: offsets past 32 bits in K and V."""
    d, hkv = 64, 1
    case = Case(11, "bf16", [(20, 5 * page + 3)], 2, hkv, d, page, fp8=fp8, spare=0)
    es = 1 if fp8 else 2
    stride = (1 << 30) // es
    pages = [hip.DeviceBuffer((case.num - 1) * stride * es + case.stride * es) for _ in "kv"]
    assert pages[0].nbytes > 1 << 32
    say(f"chunk pages past 4 GiB fp8={fp8}")
    case.upload(hip)
    for big, pool in zip(pages, case.pools):
        for i in range(case.num):
            row = np.ascontiguousarray(pool[i])
            hip.call("sile_hip_memcpy_htod", ctypes.c_void_p(big.ptr + i * stride * es), row.ctypes.data, row.nbytes)
    case.run(hip, k=pages[0].ptr, v=pages[1].ptr, stride=stride)
    case.check(case.result(hip), "past 4 GiB")
    for b in pages:
        b.close()


def test_chunk_repeats_and_graph(hip):
    """The same call gives the same bits, plain, on a stream and replayed, between other work."""
    case = Case(12, "bf16", [(30, 2000), (1, 3000), (100, 100)], 4, 1, 128, 16)
    case.upload(hip)
    case.run(hip)
    want = case.result(hip)
    case.check(want, "graph")
    st = hip.Stream()
    with hip.Graph(st) as g:
        case.run(hip, stream=st)
    other = Case(13, "bf16", [(7, 900)], 4, 1, 128, 16)
    other.upload(hip)
    for _ in range(3):
        case.do.fill_bytes(0x5A)
        hip.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(case.result(hip), want)
        other.run(hip)
    g.close()
    st.close()


def test_chunk_empty_calls(hip):
    """No sequences with tokens, no pages at all, nothing to do."""
    case = Case(14, "f16", [(0, 5), (0, 0)], 2, 1, 64, 16)
    run_case(hip, case, "no tokens")
    case = Case(15, "f16", [(3, 40)], 2, 1, 64, 16)
    case.upload(hip)
    case.run(hip, num=0, k=None, v=None)
    assert (case.result(hip)[:3] == 0).all()
    case.do.fill_bytes(0x5A)
    case.run(hip, tables=None, width=0)
    assert (case.result(hip)[:3] == 0).all()


def test_chunk_refused_on_the_device_side(hip):
    case = Case(16, "f16", [(3, 40)], 2, 1, 64, 16)
    case.upload(hip)
    for kw in (dict(ws=0), ):
        with pytest.raises(hip.SileError):
            hip.paged_attn_chunk(hip.F16, hip.F16, 1, 3, 2, 1, 64, case.dq.ptr, 128, case.ds.ptr, case.dk.ptr, case.dv.ptr, case.num, 16,
                                 case.stride, case.dt.ptr, case.width, case.dl.ptr, case.do.ptr, 128, 0.1, workspace=kw["ws"],
                                 workspace_bytes=1 << 30)
    with pytest.raises(hip.SileError):
        hip.paged_attn_chunk(hip.F16, hip.F16, 1, 3, 2, 1, 64, case.dq.ptr, 128, case.ds.ptr, case.dk.ptr, case.dv.ptr, case.num, 16,
                             case.stride, case.dt.ptr, case.width, case.dl.ptr, case.do.ptr, 128, 0.1, workspace=case.ws.ptr,
                             workspace_bytes=16)
