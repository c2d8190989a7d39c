"""GPU: rotary positions of many tokens, several of which a workgroup takes (up to 16, from 8 tokens a CU on)."""
import numpy as np
import pytest

from tests.helpers import rng, say
from tests.test_gpu_rope import Rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "fp8"), ("bf16", "fp8")])
@pytest.mark.parametrize("n,hq,hkv,d,rot,page,pad_page", [
    (2100, 4, 2, 64, 64, 16, 0), (2049, 3, 1, 80, 80, 8, 16), (5003, 2, 1, 64, 32, 1, 0), (5000, 5, 3, 96, 40, 32, 0),
    (20001, 1, 1, 32, 32, 128, 0), (17000, 0, 1, 48, 12, 16, 0), (4100, 1, 1, 256, 20, 16, 0), (2300, 8, 2, 128, 128, 16, 0)])
def test_append(hip, dtype, cache, layout, n, hq, hkv, d, rot, page, pad_page):
    say(f"rope_append {dtype} -> {cache} {layout} {n} tokens {hq}+{hkv} heads of {d}, {rot} turned, pages of {page}")
    c = Rope(hip, n + d, dtype, layout, n, hq, hkv, d, rot, cache=cache, page=page, pad_page=pad_page)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("bf16", "fp8")])
def test_append_leaves_out(hip, dtype, cache):
    """Of a workgroup's tokens some without a position, a row or a page."""
    n = 6001
    c = Rope(hip, 5, dtype, "half", n, 3, 2, 64, 48, cache=cache)
    r = rng(7)
    kind = r.integers(0, 12, n)
    rows, positions = c.rows.copy(), c.positions.copy()
    rows[kind == 1] = -1
    rows[kind == 2] = c.n_rows
    positions[kind == 3] = -5
    positions[kind == 4] = c.width * c.page
    gone_pages = [(0, 2), (1, 7), (2, 0)]
    for row, entry in gone_pages:
        c.tables[row, entry] = c.num + 3
    missing = np.array([(int(c.rows[i]), int(c.positions[i]) // c.page) in gone_pages for i in range(n)])
    c.dr, c.dp = hip.DeviceBuffer.from_array(rows), hip.DeviceBuffer.from_array(positions)
    c.dtab = hip.DeviceBuffer.from_array(c.tables)
    c.run()
    hip.synchronize()
    left = set(np.nonzero((kind >= 1) & (kind <= 4) | missing)[0].tolist())
    assert len(left) > 1000
    # the queries turn by the positions they were given; what is stored is checked without them
    q, k, v = c.heads()
    stored, c.positions = c.positions, positions
    c.check_out(c.dq, q, "q")
    c.positions, c.hq, c.heads = stored, 0, lambda: (None, k, v)
    c.check(left_out=left)


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("dtype,n,hq,hkv,d,rot,shift", [("f32", 5000, 2, 1, 64, 64, 0), ("bf16", 20000, 1, 1, 32, 16, 0), ("f16", 4500, 3, 2, 72, 40, 0),
                                                        ("bf16", 9000, 2, 1, 9, 4, 0), ("f32", 2500, 2, 2, 64, 64, 1), ("f16", 3100, 2, 1, 30, 30, 0)])
def test_memory(hip, dtype, layout, n, hq, hkv, d, rot, shift):
    say(f"rope {dtype} {layout} {n} tokens {hq}+{hkv} heads of {d}, {rot} turned, from {shift} elements on")
    c = Rope(hip, n, dtype, layout, n, hq, hkv, d, rot, shift=shift)
    c.run()
    c.check()
    other = Rope(hip, n, dtype, layout, n, hq, hkv, d, rot, shift=shift)
    other.run(in_place=True)
    hip.synchronize()
    words = {"f32": np.uint32}.get(dtype, np.uint16)
    got = other.dx.download(words, (shift + n * other.ld,))[shift:].reshape(n, other.ld)
    q, k = c.dq.download(words, (n + 1, c.ldo)), c.dk.download(words, (n + 1, c.ldo))
    assert np.array_equal(got[:, :hq * d], q[:n, :hq * d]) and np.array_equal(got[:, hq * d:(hq + hkv) * d], k[:n, :hkv * d])
    assert np.array_equal(got[:, (hq + hkv) * d:], other.bits.view(words)[:, (hq + hkv) * d:])
