"""GPU: the paged cache's bookkeeping against plain Python (whole numbers and copies:
equal to the last one), and a run of it as a serving program's steps."""
import numpy as np
import pytest

from oracle import cpuref
from tests import paged_ref
from tests.helpers import bf16_round, f16_round, rng, say

pytestmark = pytest.mark.gpu


def ints(hip, x):
    return hip.DeviceBuffer.from_array(np.asarray(x, np.int32))


def down(buf, shape):
    return buf.download(np.int32, shape)


class State:
    """Random rows over a pool: rows share pages (counts above 1), some pages are free,
    some entries name no page."""

    def __init__(self, seed, rows, width, page=16, spare=20, shared=0.3, page_bytes=64, pools=2,
                 stride=None, extra=0):
        r = rng(seed)
        self.r, self.rows, self.width, self.page = r, rows, width, page
        counts = r.integers(0, width + 1, rows)
        self.num = int(counts.sum()) + spare
        ids = r.permutation(self.num).astype(np.int32)
        self.tables = np.full((rows, width), -1, np.int32)
        at = 0
        for i, c in enumerate(counts):
            self.tables[i, :c] = ids[at:at + c]
            at += c
        for i in range(1, rows):   # some rows go on from the row before
            if r.random() < shared:
                self.tables[i] = self.tables[i - 1]
                counts[i] = counts[i - 1]
        self.lengths = np.array([r.integers((c - 1) * page + 1, c * page + 1) if c else 0 for c in counts], np.int32)
        self.refs = np.zeros(self.num, np.int32)
        for p in self.tables[self.tables >= 0]:
            self.refs[p] += 1
        if extra:   # pages held from elsewhere too
            for p in r.choice(self.num, extra):
                self.refs[p] += 1
        self.page_bytes, self.stride = page_bytes, stride or page_bytes
        self.pools = [r.integers(0, 256, (self.num, self.stride), dtype=np.uint8) for _ in range(pools)]

    def upload(self, hip):
        self.dt, self.dl, self.dr = ints(hip, self.tables), ints(hip, self.lengths), ints(hip, self.refs)
        self.dp = [hip.DeviceBuffer.from_array(p) for p in self.pools]
        self.ws = hip.DeviceBuffer(max(16, hip.kv_workspace(self.rows, self.num)))
        self.ws.fill_bytes(0xA5)
        return self

    def pool_args(self):
        return [p.ptr for p in self.dp], self.page_bytes, self.stride

    def check_pools(self, moves, what):
        for p, buf in zip(self.pools, self.dp):
            want = p.copy()
            for a, b in moves:
                want[b, :self.page_bytes] = p[a, :self.page_bytes]
            assert (buf.download(np.uint8, p.shape) == want).all(), what


def counts_of(tables, num, start):
    refs = np.array(start, np.int64)
    for p in np.asarray(tables).ravel():
        if 0 <= p < num:
            refs[p] += 1
    return refs


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 1), (7, 5), (40, 300), (1500, 9)])
def test_free(hip, rows, width, in_place):
    say(f"kv free {rows} x {width} in_place={in_place}")
    s = State(1, rows, width).upload(hip)
    drop = (s.r.random(rows) < 0.4).astype(np.int32) * s.r.integers(1, 9, rows).astype(np.int32)
    out = (s.dt, s.dl, s.dr) if in_place else (ints(hip, s.tables * 0 + 77), ints(hip, s.lengths), ints(hip, s.refs * 0))
    dd = ints(hip, drop)
    hip.kv_free(rows, width, dd.ptr, s.dt.ptr, out[0].ptr, s.dl.ptr, out[1].ptr, s.num, s.dr.ptr, out[2].ptr)
    hip.synchronize()
    gone = drop != 0
    assert (down(out[0], s.tables.shape) == np.where(gone[:, None], -1, s.tables)).all()
    assert (down(out[1], rows) == np.where(gone, 0, s.lengths)).all()
    freed = counts_of(s.tables[gone], s.num, np.zeros(s.num))
    assert (down(out[2], s.num) == s.refs - freed).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n_in,n_out,width", [(1, 1, 1), (6, 9, 4), (300, 40, 20), (40, 1300, 70), (5, 0, 3), (0, 4, 3)])
def test_fork(hip, n_in, n_out, width, in_place):
    say(f"kv fork {n_in} -> {n_out} x {width} counts in_place={in_place}")
    s = State(2, max(n_in, 1), width, extra=5)
    s.tables, s.lengths = s.tables[:n_in], s.lengths[:n_in]
    s.upload(hip)
    src = s.r.integers(-2, n_in + 2, n_out).astype(np.int32)
    ds, new_t, new_l = ints(hip, src), ints(hip, np.full((n_out, width), 55)), ints(hip, np.full(n_out, 66))
    refs = s.dr if in_place else ints(hip, s.refs * 0 - 9)
    hip.kv_fork(n_in, n_out, width, ds.ptr, s.dt.ptr, new_t.ptr, s.dl.ptr, new_l.ptr, s.num, s.dr.ptr, refs.ptr)
    hip.synchronize()
    ok = (src >= 0) & (src < n_in)
    want = np.full((n_out, width), -1)
    want[ok] = s.tables[src[ok]]
    assert (down(new_t, (n_out, width)) == want).all()
    assert (down(new_l, n_out) == [s.lengths[x] if o else 0 for x, o in zip(src, ok)]).all()
    before = s.refs - counts_of(s.tables, s.num, np.zeros(s.num))
    assert (down(refs, s.num) == counts_of(want, s.num, before)).all()


@pytest.mark.parametrize("mode", ["out", "in", "mixed"])
@pytest.mark.parametrize("rows,width,page,spare,most", [(1, 1, 16, 1, 1), (9, 6, 16, 30, 40), (64, 40, 8, 200, 30),
                                                        (64, 40, 8, 20, 30), (1200, 6, 4, 3000, 9), (3, 300, 1, 700, 200),
                                                        (20, 10, 16, 6000, 50)])
def test_reserve(hip, rows, width, page, spare, most, mode):
    """Enough pages and too few, needs of none to many pages, rows past their table."""
    say(f"kv reserve {rows} x {width} page={page} spare={spare} {mode}")
    s = State(3, rows, width, page, spare, extra=3, stride=80).upload(hip)
    need = s.r.integers(-1, most + 1, rows).astype(np.int32)
    dn, dg = ints(hip, need), ints(hip, np.full(rows, 9))
    t = s.dt if mode != "out" else ints(hip, s.tables * 0 + 5)
    f = s.dr if mode == "in" else ints(hip, s.refs * 0 + 5)
    hip.kv_reserve(rows, width, page, s.dl.ptr, dn.ptr, s.dt.ptr, t.ptr, s.num, s.dr.ptr, f.ptr, dg.ptr,
                   *s.pool_args(), s.ws.ptr, s.ws.nbytes)
    hip.synchronize()
    tables, refs, granted, copies = paged_ref.reserve(page, s.num, s.lengths.tolist(), need.tolist(),
                                                      s.tables.tolist(), s.refs.tolist())
    assert (down(dg, rows) == granted).all()
    assert (down(t, s.tables.shape) == tables).all()
    assert (down(f, s.num) == refs).all()
    assert (down(s.dl, rows) == s.lengths).all()
    s.check_pools(copies, "copies")


def test_reserve_bad_state(hip):
    """Lengths below zero and past the table, entries outside the pool, counts of zero and
    below for pages that a table names."""
    say("kv reserve bad state")
    s = State(4, 30, 8, 16, 60)
    s.lengths[:6] = [-3, 10 ** 9, 8 * 16, 2 ** 31 - 1, -2 ** 31, 17]
    s.tables[5, :] = [s.num, -9, 2 ** 31 - 1, -2 ** 31, 0, 1, 2, 3]
    s.refs[s.r.choice(s.num, 10)] = -2
    s.refs[s.r.choice(s.num, 10)] = 0
    s.upload(hip)
    need = np.full(30, 20, np.int32)
    need[7] = 2 ** 31 - 1
    dn, dg = ints(hip, need), ints(hip, np.full(30, 9))
    hip.kv_reserve(30, 8, 16, s.dl.ptr, dn.ptr, s.dt.ptr, s.dt.ptr, s.num, s.dr.ptr, s.dr.ptr, dg.ptr,
                   *s.pool_args(), s.ws.ptr, s.ws.nbytes)
    hip.synchronize()
    tables, refs, granted, copies = paged_ref.reserve(16, s.num, s.lengths.tolist(), need.tolist(),
                                                      s.tables.tolist(), s.refs.tolist())
    assert (down(dg, 30) == granted).all() and (down(s.dt, s.tables.shape) == tables).all()
    assert (down(s.dr, s.num) == refs).all()
    s.check_pools(copies, "copies")


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows,width,spare,page_bytes", [(1, 1, 0, 16), (5, 9, 30, 48), (50, 30, 0, 64), (60, 200, 9000, 32),
                                                         (4, 3, 20, 40000)])
def test_compact(hip, rows, width, spare, page_bytes, in_place):
    say(f"kv compact {rows} x {width} spare={spare} bytes={page_bytes} in_place={in_place}")
    s = State(5, rows, width, 16, spare, page_bytes=page_bytes, stride=page_bytes + 16, extra=2)
    s.refs[s.r.choice(s.num, min(3, s.num))] -= 3   # below zero counts as free
    if rows > 3:
        s.tables[2, 0] = s.num + 5
    s.upload(hip)
    t, f = (s.dt, s.dr) if in_place else (ints(hip, s.tables * 0), ints(hip, s.refs * 0 + 9))
    used = ints(hip, [-1])
    hip.kv_compact(rows, width, s.dt.ptr, t.ptr, s.num, s.dr.ptr, f.ptr, used.ptr, *s.pool_args(), s.ws.ptr, s.ws.nbytes)
    hip.synchronize()
    tables, refs, u, moves = paged_ref.compact(s.num, s.tables.tolist(), s.refs.tolist())
    assert down(used, 1)[0] == u
    assert (down(t, s.tables.shape) == tables).all()
    assert (down(f, s.num) == refs).all()
    s.check_pools(list(moves.items()), "moves")


@pytest.mark.parametrize("n,page_bytes,stride,pools", [(1, 16, 16, 1), (30, 4096, 4096, 3), (17, 50000, 50016, 2),
                                                       (200, 48, 64, 128)])
def test_copy_pages(hip, n, page_bytes, stride, pools):
    say(f"kv copy {n} pages of {page_bytes}")
    r = rng(6)
    num = 2 * n + 4
    host = [r.integers(0, 256, (num, stride), dtype=np.uint8) for _ in range(pools)]
    dev = [hip.DeviceBuffer.from_array(p) for p in host]
    ids = r.permutation(num)[:2 * n]
    src, dst = ids[:n].copy(), ids[n:].copy()
    pairs = [(a, b) for a, b in zip(src, dst)]
    if n > 3:   # outside the pool, and onto itself: left out
        src[0], dst[1], src[2] = num, -1, dst[2]
        pairs = pairs[3:]
    ds, dd = ints(hip, src), ints(hip, dst)
    hip.kv_copy_pages([p.ptr for p in dev], page_bytes, stride, num, n, ds.ptr, dd.ptr)
    hip.synchronize()
    for h, d in zip(host, dev):
        want = h.copy()
        for a, b in pairs:
            want[b, :page_bytes] = h[a, :page_bytes]
        assert (d.download(np.uint8, h.shape) == want).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,hkv,d,page", [(1, 1, 16, 1), (37, 2, 64, 16), (5, 3, 80, 4), (300, 8, 128, 32), (9, 1, 256, 64)])
def test_append(hip, dtype, fp8, tokens, hkv, d, page):
    """Tokens out of a wider projection; some with a row, position or page that does not
    exist.  Values past e4m3's range, NaN and Inf among them."""
    say(f"kv append {dtype} fp8={fp8} {tokens} x {hkv} x {d} page={page}")
    r = rng(7)
    rows, width = 6, 5
    num, stride = rows * width + 2, hkv * page * d + 32
    tables = r.permutation(num)[:rows * width].reshape(rows, width).astype(np.int32)
    tables[1, 2], tables[2, 0], tables[3, 1] = -1, num, 2 ** 31 - 1
    slots = r.permutation(rows * width * page)[:min(tokens, rows * width * page)]
    tokens = len(slots)
    row, pos = (slots // (width * page)).astype(np.int32), (slots % (width * page)).astype(np.int32)
    if tokens > 4:
        row[0], row[1], pos[2], pos[3] = -1, rows, -1, width * page
    ld = (hkv * 2 + 1) * d
    x = (r.normal(size=(tokens, ld)) * 3).astype(np.float32)
    x.ravel()[::97] *= 1000
    x.ravel()[5::211] = np.nan
    x.ravel()[7::223] = np.inf
    bits, x = (f16_round if dtype == "f16" else bf16_round)(x)
    scales = (0.02, 0.5) if fp8 else (1.0, 1.0)
    dx, dr_, dp, dt = hip.DeviceBuffer.from_array(bits), ints(hip, row), ints(hip, pos), ints(hip, tables)
    kind = np.uint8 if fp8 else np.uint16
    host = [r.integers(0, 255, (num, stride)).astype(kind) for _ in "kv"]
    dev = [hip.DeviceBuffer.from_array(p) for p in host]
    t = hip.F16 if dtype == "f16" else hip.BF16
    hip.kv_append(t, hip.F8E4M3 if fp8 else t, tokens, hkv, d, dx.ptr + 2 * d, ld, dx.ptr + 2 * d * (hkv + 1), ld,
                  dr_.ptr, dp.ptr, dev[0].ptr, dev[1].ptr, num, page, stride, dt.ptr, rows, width, *scales)
    hip.synchronize()
    for which in range(2):
        want = host[which].copy()
        for i in range(tokens):
            if not (0 <= row[i] < rows and 0 <= pos[i] < width * page):
                continue
            p = tables[row[i], pos[i] // page]
            if not 0 <= p < num:
                continue
            at = slice(d * (1 + hkv * which), d * (1 + hkv * which) + hkv * d)
            with np.errstate(over="ignore"):
                new = cpuref.e4m3_encode(x[i, at], scales[which]) if fp8 else bits[i, at]
            want[p, :hkv * page * d].reshape(hkv, page, d)[:, pos[i] % page] = new.reshape(hkv, d)
        got = dev[which].download(kind, host[which].shape)
        if fp8:   # any NaN code stands for NaN
            got, want = (np.where((y & 0x7F) == 0x7F, 0x7F, y) for y in (got, want))
        assert (got == want).all(), (which, np.argwhere(got != want)[:5], got[got != want][:5], want[got != want][:5])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [1.0, 0.1, 1 / 3, 0.007, 2.0 ** -126, 1e-40, 3e38, -0.3, 1.9999999, 0.0])
def test_append_e4m3_every_value(hip, dtype, scale):
    """Every 16-bit value over a scale: the correctly rounded quotient's nearest code."""
    say(f"kv append {dtype} every value / {scale}")
    bits = np.arange(65536, dtype=np.uint16).reshape(64, 1024)
    x = bits.view(np.float16).astype(np.float32) if dtype == "f16" else cpuref.f32_from_bf16(bits)
    dx, dt = hip.DeviceBuffer.from_array(bits), ints(hip, [[0]])
    dr_, dp = ints(hip, np.zeros(64)), ints(hip, np.arange(64))
    pools = [hip.DeviceBuffer(65536) for _ in "kv"]
    t = hip.F16 if dtype == "f16" else hip.BF16
    hip.kv_append(t, hip.F8E4M3, 64, 4, 256, dx.ptr, 1024, dx.ptr, 1024, dr_.ptr, dp.ptr, pools[0].ptr, pools[1].ptr,
                  1, 64, 65536, dt.ptr, 1, 1, scale, 1.0)
    hip.synchronize()
    for buf, s in zip(pools, (scale, 1.0)):
        got = buf.download(np.uint8, (4, 64, 256)).transpose(1, 0, 2).reshape(64, 1024)
        with np.errstate(all="ignore"):
            y = np.clip(x / np.float32(s), -448, 448)   # (NaN stays)
        want = cpuref.e4m3_encode(y, 1.0)
        nan = np.isnan(y)
        assert ((got & 0x7F)[nan] == 0x7F).all()
        assert (got[~nan] == want[~nan]).all(), (s, x[~nan][got[~nan] != want[~nan]][:5])


def test_pages_past_32_bits(hip):
    """Pages 2^30 bytes apart in a pool of 6 GiB: tokens stored into and pages copied between
    its ends."""
    say("kv pages past 4 GiB")
    r = rng(10)
    num, far, hkv, d, page = 6, 1 << 30, 2, 64, 16
    size = hkv * page * d * 2
    pool = hip.DeviceBuffer((num - 1) * far + 2 * size)
    one = r.integers(0, 65536, size // 2, dtype=np.uint16)
    pages = [one + np.uint16(i) for i in range(num)]
    for i, x in enumerate(pages):
        hip.call("sile_hip_memcpy_htod", pool.ptr + i * far, x.ctypes.data, size)
    bits = f16_round(r.normal(size=(3, 2, hkv, d)))[0]
    dx, table, pos = hip.DeviceBuffer.from_array(bits), ints(hip, [[5, 0, 4]]), ints(hip, [3, 16, 47])
    rows = ints(hip, [0, 0, 0])
    # (V's pages lie behind K's in the same records)
    hip.kv_append(hip.F16, hip.F16, 3, hkv, d, dx.ptr, 2 * hkv * d, dx.ptr + 2 * hkv * d, 2 * hkv * d, rows.ptr, pos.ptr,
                  pool.ptr, pool.ptr + size, num, page, far // 2, table.ptr, 1, 3)
    src, dst = ints(hip, [5, 0]), ints(hip, [1, 3])
    hip.kv_copy_pages([pool.ptr], size, far, num, 2, src.ptr, dst.ptr)
    hip.synchronize()
    want = [x.reshape(hkv, page, d).copy() for x in pages]
    for t, (p, slot) in enumerate(((5, 3), (0, 0), (4, 15))):
        want[p][:, slot] = bits[t, 0]
    want[1], want[3] = want[5], want[0]
    got = np.empty(size // 2, np.uint16)
    for i in range(num):
        hip.call("sile_hip_memcpy_dtoh", got.ctypes.data, pool.ptr + i * far, size)
        assert (got == want[i].ravel()).all(), i
    pool.close()


def test_serving_run(hip):
    """Steps of a serving program, captured where they repeat: prompts stored, a token a
    step, beams forked and dropped, pages made writable, the pool closed up; after each
    the attention over the cache is that over the tokens' own list."""
    say("kv serving run")
    r = rng(8)
    rows, hq, hkv, d, page, width, num = 6, 4, 2, 64, 16, 8, 40
    stride = hkv * page * d
    st = hip.Stream()
    dt = [ints(hip, np.full((rows, width), -1)) for _ in range(2)]
    dl = [ints(hip, np.zeros(rows)) for _ in range(2)]
    dr = ints(hip, np.zeros(num))
    dk, dv = (hip.DeviceBuffer.from_array(np.full((num, stride), 0x7E00, np.uint16)) for _ in "kv")
    ws = hip.DeviceBuffer(hip.kv_workspace(rows, num))
    wa = hip.DeviceBuffer(hip.paged_attn_workspace(rows, hq, hkv, d))
    granted, used = ints(hip, np.zeros(rows)), ints(hip, [0])
    pools = ([dk.ptr, dv.ptr], stride * 2, stride * 2)
    lists = [[[], []] for _ in range(rows)]   # a row's K and V tokens [hkv, d]
    lengths = [0] * rows
    dq, do = hip.DeviceBuffer(rows * hq * d * 2), hip.DeviceBuffer(rows * hq * d * 2)

    def store(tokens):   # {row: count}
        row = np.array([i for i, n in tokens.items() for _ in range(n)], np.int32)
        pos = np.array([lengths[i] + j for i, n in tokens.items() for j in range(n)], np.int32)
        need = np.zeros(rows, np.int32)
        for i, n in tokens.items():
            need[i] = n
        bits, x = f16_round(r.normal(size=(len(row), 2, hkv, d)))
        dx, dn, drow, dpos = hip.DeviceBuffer.from_array(bits), ints(hip, need), ints(hip, row), ints(hip, pos)
        hip.kv_reserve(rows, width, page, dl[0].ptr, dn.ptr, dt[0].ptr, dt[0].ptr, num, dr.ptr, dr.ptr, granted.ptr,
                       *pools, ws.ptr, ws.nbytes, st)
        hip.kv_append(hip.F16, hip.F16, len(row), hkv, d, dx.ptr, 2 * hkv * d, dx.ptr + 2 * hkv * d, 2 * hkv * d,
                      drow.ptr, dpos.ptr, dk.ptr, dv.ptr, num, page, stride, dt[0].ptr, rows, width, stream=st)
        st.synchronize()
        assert (down(granted, rows) == 1).all()
        for i, t in zip(row, range(len(row))):
            lists[i][0].append(x[t, 0])
            lists[i][1].append(x[t, 1])
        for i, n in tokens.items():
            lengths[i] += n
        dl[0].upload(np.array(lengths, np.int32))

    def attend(what):
        qb, q = f16_round(r.normal(size=(rows, hq, d)))
        dq.upload(qb)
        hip.paged_attn_decode(hip.F16, hip.F16, rows, hq, hkv, d, dq.ptr, hq * d, dk.ptr, dv.ptr, num, page, stride,
                              dt[0].ptr, width, dl[0].ptr, do.ptr, hq * d, d ** -0.5, workspace=wa.ptr,
                              workspace_bytes=wa.nbytes, stream=st)
        st.synchronize()
        got = do.download(np.float16, (rows, hq, d)).astype(np.float64)
        for i in range(rows):
            for h in range(hq):
                k = np.array([t[h // 2] for t in lists[i][0]]).reshape(-1, d)
                v = np.array([t[h // 2] for t in lists[i][1]]).reshape(-1, d)
                ref, spread, size = paged_ref.attention(q[i, h], k, v, d ** -0.5)
                bound = paged_ref.error_bound(ref, spread, size, "f16", d, len(k), 2.0 ** -21)
                assert (np.abs(got[i, h] - ref) <= bound).all(), (what, i, h)

    def fork(src):
        ds = ints(hip, src)
        hip.kv_fork(rows, rows, width, ds.ptr, dt[0].ptr, dt[1].ptr, dl[0].ptr, dl[1].ptr, num, dr.ptr, dr.ptr, st)
        st.synchronize()
        dt.reverse()
        dl.reverse()
        lists[:] = [[list(lists[s][0]), list(lists[s][1])] if 0 <= s < rows else [[], []] for s in src]
        lengths[:] = [lengths[s] if 0 <= s < rows else 0 for s in src]

    store({0: 21, 1: 5, 3: 40, 4: 16})
    attend("prompts")
    for step in range(3):
        store({0: 1, 1: 1, 3: 1, 4: 1})
        attend(f"token {step}")
    fork([0, 0, 0, 3, 3, -1])       # row 1's and 4's pages go free
    store({i: 1 for i in range(5)})  # the shared last pages are copied
    attend("forked")
    drop = ints(hip, [0, 1, 0, 0, 1, 0])
    hip.kv_free(rows, width, drop.ptr, dt[0].ptr, dt[0].ptr, dl[0].ptr, dl[0].ptr, num, dr.ptr, dr.ptr, st)
    for i in (1, 4):
        lists[i], lengths[i] = [[], []], 0
    attend("dropped")
    hip.kv_compact(rows, width, dt[0].ptr, dt[0].ptr, num, dr.ptr, dr.ptr, used.ptr, *pools, ws.ptr, ws.nbytes, st)
    attend("closed up")
    refs = down(dr, num)
    u = down(used, 1)[0]
    assert (refs[:u] > 0).all() and (refs[u:] == 0).all()
    assert (counts_of(down(dt[0], (rows, width)), num, np.zeros(num)) == refs).all()
    store({5: 30, 0: 1})
    attend("and on")
    st.close()


@pytest.mark.parametrize("window,sinks", [(1000, 0), (50, 3)])
def test_prompt_then_tokens(hip, window, sinks):
    """A prompt's attention, its tokens stored, then token by token over the cache: one
    sequence's attention, row for row, in one graph per step."""
    say(f"kv prompt then tokens window={window}")
    r = rng(9)
    n, steps, hq, hkv, d, page, width = 90, 12, 4, 2, 64, 16, 8
    total, stride = n + steps, hkv * page * d
    qb, q = f16_round(r.normal(size=(total, hq, d)))
    kb, k = f16_round(r.normal(size=(total, hkv, d)))
    vb, v = f16_round(r.normal(size=(total, hkv, d)))
    st = hip.Stream()
    up = hip.DeviceBuffer.from_array
    heads = lambda x: up(np.ascontiguousarray(x[:n].transpose(1, 0, 2)))  # noqa: E731
    hq_, hk, hv, ho = heads(qb), heads(kb), heads(vb), hip.DeviceBuffer(n * hq * d * 2)
    hip.flash_attn_window_fwd(hip.F16, 1, hq, hkv, n, n, d, hq_.ptr, hk.ptr, hv.ptr, ho.ptr, d ** -0.5, 0, window, sinks, st)
    dq, dk, dv = up(qb), up(kb), up(vb)
    pk, pv = (up(np.full((width, stride), 0x7E00, np.uint16)) for _ in "kv")
    table, refs = ints(hip, np.full((1, width), -1)), ints(hip, np.zeros(width))
    length, need, pos, granted = ints(hip, [0]), ints(hip, [n]), ints(hip, np.arange(n)), ints(hip, [0])
    rows = ints(hip, np.zeros(n))
    ws, wa = hip.DeviceBuffer(hip.kv_workspace(1, width)), hip.DeviceBuffer(hip.paged_attn_workspace(1, hq, hkv, d))
    out = hip.DeviceBuffer(hq * d * 2)
    pools = ([pk.ptr, pv.ptr], 2 * stride, 2 * stride)

    def reserve():
        hip.kv_reserve(1, width, page, length.ptr, need.ptr, table.ptr, table.ptr, width, refs.ptr, refs.ptr, granted.ptr,
                       *pools, ws.ptr, ws.nbytes, st)

    reserve()
    hip.kv_append(hip.F16, hip.F16, n, hkv, d, dk.ptr, hkv * d, dv.ptr, hkv * d, rows.ptr, pos.ptr, pk.ptr, pv.ptr, width,
                  page, stride, table.ptr, 1, width, stream=st)
    st.synchronize()
    got = [x for x in ho.download(np.float16, (hq, n, d)).transpose(1, 0, 2)]
    # a step: the newest token at fixed places, so that one graph serves all steps
    tq, tk, tv = (hip.DeviceBuffer(x.nbytes // total) for x in (qb, kb, vb))
    need.upload(np.array([1], np.int32))
    before = ints(hip, [0])
    with hip.Graph(st) as graph:
        hip.kv_reserve(1, width, page, before.ptr, need.ptr, table.ptr, table.ptr, width, refs.ptr, refs.ptr, granted.ptr,
                       *pools, ws.ptr, ws.nbytes, st)
        hip.kv_append(hip.F16, hip.F16, 1, hkv, d, tk.ptr, hkv * d, tv.ptr, hkv * d, None, before.ptr, pk.ptr, pv.ptr, width,
                      page, stride, table.ptr, 1, width, stream=st)
        hip.paged_attn_decode(hip.F16, hip.F16, 1, hq, hkv, d, tq.ptr, hq * d, pk.ptr, pv.ptr, width, page, stride,
                              table.ptr, width, length.ptr, out.ptr, hq * d, d ** -0.5, window=window, sinks=sinks,
                              workspace=wa.ptr, workspace_bytes=wa.nbytes, stream=st)
    for i in range(n, total):
        for buf, x in ((tq, qb), (tk, kb), (tv, vb)):
            buf.upload(x[i])
        before.upload(np.array([i], np.int32))
        length.upload(np.array([i + 1], np.int32))
        hip.synchronize()
        graph.launch()
        st.synchronize()
        assert down(granted, 1)[0] == 1
        got.append(out.download(np.float16, (hq, d)))
    for i in range(total):
        at = paged_ref.seen_keys(i + 1, window, sinks)
        for h in range(hq):
            ref, spread, size = paged_ref.attention(q[i, h], k[at, h // 2], v[at, h // 2], d ** -0.5)
            p_error = 2.0 ** -11 if i < n else 2.0 ** -21
            bound = paged_ref.error_bound(ref, spread, size, "f16", d, len(at), p_error)
            assert (np.abs(got[i][h].astype(np.float64) - ref) <= bound).all(), (i, h)
    graph.close()
    st.close()


def test_graph_of_a_step(hip):
    """free, fork, reserve and compact captured once: each replay on its own state gives
    what the eager calls give, with eager work in between."""
    say("kv graph")
    rows, width, page = 40, 12, 16
    states = [State(20 + i, rows, width, page, 100) for i in range(3)]
    num = max(s.num for s in states)
    st = hip.Stream()
    dt, tt = ints(hip, np.zeros((rows, width))), ints(hip, np.zeros((rows, width)))
    dl, tl = ints(hip, np.zeros(rows)), ints(hip, np.zeros(rows))
    dr, dd, ds, dn = ints(hip, np.zeros(num)), ints(hip, np.zeros(rows)), ints(hip, np.zeros(rows)), ints(hip, np.zeros(rows))
    dg, du = ints(hip, np.zeros(rows)), ints(hip, [0])
    pool = hip.DeviceBuffer(num * 64)
    ws = hip.DeviceBuffer(hip.kv_workspace(rows, num))

    def calls(stream):
        hip.kv_free(rows, width, dd.ptr, dt.ptr, dt.ptr, dl.ptr, dl.ptr, num, dr.ptr, dr.ptr, stream)
        hip.kv_fork(rows, rows, width, ds.ptr, dt.ptr, tt.ptr, dl.ptr, tl.ptr, num, dr.ptr, dr.ptr, stream)
        hip.kv_reserve(rows, width, page, tl.ptr, dn.ptr, tt.ptr, tt.ptr, num, dr.ptr, dr.ptr, dg.ptr, [pool.ptr], 64, 64,
                       ws.ptr, ws.nbytes, stream)
        hip.kv_compact(rows, width, tt.ptr, tt.ptr, num, dr.ptr, dr.ptr, du.ptr, [pool.ptr], 64, 64, ws.ptr, ws.nbytes, stream)

    def load(s):
        refs = np.zeros(num, np.int32)
        refs[:s.num] = s.refs
        r = rng(99 + s.num)
        for buf, x in ((dt, s.tables), (dl, s.lengths), (dr, refs), (dd, r.integers(0, 2, rows)),
                       (ds, r.integers(-1, rows, rows)), (dn, r.integers(0, 20, rows))):
            buf.upload(np.asarray(x, np.int32))
        pool.upload(r.integers(0, 256, num * 64, dtype=np.uint8))

    def out():
        return [down(tt, (rows, width)), down(tl, rows), down(dr, num), down(dg, rows), down(du, 1),
                pool.download(np.uint8, num * 64)]

    load(states[0])
    with hip.Graph(st) as graph:
        calls(st)
    for s in states + states[:1]:
        load(s)
        hip.synchronize()
        calls(None)
        hip.synchronize()
        want = out()
        load(s)
        hip.synchronize()
        graph.launch()
        st.synchronize()
        for a, b in zip(out(), want):
            assert (a == b).all()
    graph.close()
    st.close()


@pytest.mark.parametrize("in_place", [False, True])
def test_large_pools(hip, in_place):
    """A pool of 100000 pages: the one workgroup that ranks free pages and plans the
    closing up goes on past what it holds in registers."""
    say(f"kv 100000 pages in_place={in_place}")
    s = State(11, 300, 400, 16, 40000, page_bytes=16, pools=1, extra=5).upload(hip)
    assert s.num > 90000, s.num
    need = s.r.integers(0, 3000, 300).astype(np.int32)
    dn, dg, used = ints(hip, need), ints(hip, np.full(300, 9)), ints(hip, [-1])
    t, f = (s.dt, s.dr) if in_place else (ints(hip, s.tables * 0), ints(hip, s.refs * 0))
    hip.kv_reserve(300, 400, 16, s.dl.ptr, dn.ptr, s.dt.ptr, t.ptr, s.num, s.dr.ptr, f.ptr, dg.ptr, *s.pool_args(),
                   s.ws.ptr, s.ws.nbytes)
    hip.synchronize()
    tables, refs, granted, copies = paged_ref.reserve(16, s.num, s.lengths.tolist(), need.tolist(), s.tables.tolist(),
                                                      s.refs.tolist())
    assert 0 < sum(granted) < 300 and (down(dg, 300) == granted).all()
    assert (down(t, s.tables.shape) == tables).all() and (down(f, s.num) == refs).all()
    s.check_pools(copies, "copies")
    # every 20th row goes; what stays is closed up
    s.tables, s.refs = np.array(tables, np.int32), np.array(refs, np.int32)
    s.pools = [p.download(np.uint8, x.shape) for p, x in zip(s.dp, s.pools)]
    s.refs -= counts_of(s.tables[::20], s.num, np.zeros(s.num)).astype(np.int32)
    s.tables[::20] = -1
    dt, dr = ints(hip, s.tables), ints(hip, s.refs)
    t, f = (dt, dr) if in_place else (t, f)
    hip.kv_compact(300, 400, dt.ptr, t.ptr, s.num, dr.ptr, f.ptr, used.ptr, *s.pool_args(), s.ws.ptr, s.ws.nbytes)
    hip.synchronize()
    tables, refs, u, moves = paged_ref.compact(s.num, s.tables.tolist(), s.refs.tolist())
    assert down(used, 1)[0] == u and len(moves) > 1000 and max(moves) > 65536
    assert (down(t, s.tables.shape) == tables).all() and (down(f, s.num) == refs).all()
    s.check_pools(list(moves.items()), "moves")
