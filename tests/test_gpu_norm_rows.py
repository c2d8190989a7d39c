"""GPU: the row norm where tests/test_gpu_serving_rows.py does not look: rows whose sum of squares leaves
fp32, and more rows than one launch has workgroups."""
import numpy as np
import pytest

from tests import serving_ref as ref
from tests.helpers import rng, say
from tests.test_gpu_serving_rows import Norm

pytestmark = pytest.mark.gpu


def rows_of(cols, sizes, dtype, seed):
    """A row of N(0, 1) at each size, values held to the type's range."""
    top = 3.3e38 if dtype != "f16" else 6.5e4
    x = rng(seed).normal(size=(len(sizes), cols)) * np.array(sizes)[:, None]
    return np.clip(x, -top, top).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 7, 64, 512, 1000, 2048, 4097, 8192, 16384, 17001])
def test_large_values(hip, dtype, cols):
    """Finite rows past the root of fp32's range, beside ordinary ones: of order 1 all the same."""
    x = rows_of(cols, [1.0, 1e19, 1e25, 1.0, 1e37, 1e38, 2.0, 1e30, 0.0], dtype, cols)
    x[7, 1:] = 1.0   # one large value alone
    for out, group in ((dtype, 0), ("fp8", cols), ("fp8", 64 if cols % 64 == 0 else 0)):
        say(f"norm of large values {dtype} -> {out}, {cols} columns, group {group}")
        for residual in (False, True):
            c = Norm(hip, cols, dtype, out, len(x), cols, residual=residual, weight=residual, group=group, x=x)
            c.run()
            c.check()
            c.run(sum_to=c.dx.ptr)   # (the sum over x)
            c.check(ds=c.dx)


@pytest.mark.parametrize("cols", [1, 40, 512, 2000, 8193, 16384, 20000])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-31, 1e-25, 1e-5])
def test_small_values(hip, cols, eps):
    """Rows whose squares are below fp32's least, with an eps that is no larger, or is."""
    x = rows_of(cols, [1.0, 1e-10, 1e-16, 1e-20, 1e-25, 1e-36, 1e-44], "f32", cols)
    x[x == 0.0] = 2.0 ** -149
    say(f"norm of small values, {cols} columns, eps {eps}")
    for out, group in (("f32", 0), ("fp8", 0)):
        c = Norm(hip, cols, "f32", out, len(x), cols, residual=False, weight=False, group=group, x=x, scale=0.01)
        c.eps = float(np.float32(eps))
        c.run()
        c.check()


@pytest.mark.parametrize("cols", [200, 3000, 16000])
def test_zeros_without_eps(hip, cols):
    """0 / 0: NaN, as the formula; and Inf as it is beside an eps."""
    x = np.zeros((3, cols), np.float32)
    x[1] = 1.0
    x[2], x[2, 5] = 1e38, np.inf
    c = Norm(hip, 1, "f32", "f32", 3, cols, residual=False, weight=False, x=x)
    c.eps = 0.0
    c.run()
    hip.synchronize()
    y = c.dy.download(np.float32, (3, cols))
    assert np.isnan(y[0]).all() and (np.abs(y[1] - 1) <= 50 * ref.EPS).all()
    assert np.isnan(y[2, 5]) and (np.delete(y[2], 5) == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols,group", [(256, 0), (256, 64), (256, 256), (2048, 128), (255, 255), (18000, 1000), (18000, 18000), (18000, 0)])
def test_signs_of_zeros(hip, dtype, cols, group):
    """Codes keep the sign of a zero, and of what rounds to one, whatever the scale is from."""
    x = rng(cols).normal(size=(4, cols)).astype(np.float32)
    x[:, ::3] = 0.0
    x[:, 1::6] = -0.0
    x[:, 2::9] = 1e-7 * np.where(np.arange(len(range(2, cols, 9))) % 2, 1, -1)
    c = Norm(hip, 1, dtype, "fp8", 4, cols, residual=False, weight=False, group=group, x=x)
    c.run()
    c.check()
    code = c.dy.download(np.uint8, (4, cols))
    assert np.array_equal(code >> 7 != 0, np.signbit(c.x))


@pytest.mark.parametrize("dtype,out,rows,cols,group", [
    # a wave a row (8192 rows are one launch's, on 256 CUs), a workgroup of 256 (2048) and of 1024 (512), any width
    ("bf16", "bf16", 17001, 40, 0), ("f32", "f32", 9000, 100, 0), ("f16", "fp8", 9001, 256, 64), ("bf16", "fp8", 20000, 33, 33),
    ("bf16", "bf16", 4500, 1000, 0), ("bf16", "fp8", 6200, 600, 600), ("f32", "fp8", 4200, 1024, 128), ("f16", "f16", 2100, 4097, 0),
    ("bf16", "fp8", 4100, 8192, 8192), ("f32", "fp8", 2050, 3001, 3001),
    ("bf16", "bf16", 1100, 8200, 0), ("f16", "fp8", 1600, 8200, 8200), ("f32", "fp8", 520, 16384, 256),
    ("f32", "f32", 2060, 16386, 0), ("bf16", "fp8", 4500, 999, 333), ("f16", "fp8", 2100, 16400, 16400)])
def test_many_rows(hip, dtype, out, rows, cols, group):
    """Workgroups that go on to further rows, some of which are summed again."""
    say(f"norm {dtype} -> {out} {rows} x {cols}, groups of {group}")
    r = rng(rows + cols)
    x = r.normal(size=(rows, cols)).astype(np.float32) * r.choice([0.01, 1.0, 50.0], rows).astype(np.float32)[:, None]
    if dtype != "f16":
        x[r.random(rows) < 0.2, 0] = 1e25
    c = Norm(hip, rows, dtype, out, rows, cols, weight=cols < 5000, group=group, x=x)
    c.run()
    c.check()
