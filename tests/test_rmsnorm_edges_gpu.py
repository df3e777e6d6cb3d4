"""The root-mean-square norm where rounding decides: against whole numbers and fractions."""
from fractions import Fraction

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from decx_amd import hip as h
    h.init()
    return h


def rint(q):
    """A fraction to the nearest whole number, halves to the even one."""
    low = q.numerator // q.denominator
    rest = q - low
    return low + 1 if rest > Fraction(1, 2) or (rest == Fraction(1, 2) and low % 2) else low


# (top's factors, t's factors): fp32 values whose 127 t / top misses a half by less than the last of 53 bits of either side
NEXT_TO_A_HALF = [(10826011, 12636473, 8806181, 13883497), (15460537, 15476367, 11702938, 16018360), (12190991, 11474615, 9030521, 12258199),
                  (10152001, 16244053, 11760712, 12862774), (11945017, 13029605, 9362068, 15773554), (11300127, 12203409, 6023476, 12889012),
                  (10959887, 10180709, 3832792, 13180533), (16618719, 10210709, 4910714, 8570687)]


@pytest.mark.parametrize("cols", [2, 4, 300, 5001, 40001])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -60, 2.0 ** 70])
def test_codes_of_fp32_rows_next_to_a_half(hip, cols, scale):
    """Products of 48 bits: the sides of the comparison do not fit 64-bit floating point."""
    for a, b, c, d in NEXT_TO_A_HALF:
        left = rint(Fraction(127 * c * d, a * b))
        exactly = Fraction(127 * c * d, a * b) - Fraction(127 * c * d * 2 // (a * b), 2)
        assert min(exactly, Fraction(1, 2) - exactly) < Fraction(1, 1 << 44)
        x, w = np.zeros((2, cols), np.float32), np.ones((1, cols), np.float32)
        at, top = cols // 3, cols - 1
        x[:, top], w[0, top] = a * scale, b
        x[0, at], x[1, at], w[0, at] = c * scale, -c * scale, d
        dx, dw = hip.DeviceMatrix(2, cols, np.float32, data=x), hip.DeviceMatrix(1, cols, np.float32, data=w)
        dy, ds = hip.DeviceMatrix(2, cols, np.int8, pad_value=77), hip.DeviceMatrix(1, 2, np.float32)
        hip.rmsnorm(dx, dw, dy, y_scales=ds)
        hip.sync()
        want = np.zeros((2, cols), np.int8)
        want[:, top], want[0, at], want[1, at] = 127, left, -left
        assert np.array_equal(dy.download(), want), (a, b, c, d)


@pytest.mark.parametrize("cols", [40001, 1 << 20, (1 << 24) + 5])
@pytest.mark.parametrize("value", [0.1, 0.77, 1.7])
def test_long_rows_of_one_value(hip, cols, value):
    """Sums whose roundings all fall to one side.  A sum of 8 squares in fp32 is off by at most 8 2^-24 of itself, the threads'
    sums in 64 bits by next to nothing, rounding them and adding 1024 of them over lanes and wavefronts by 1 + 6 + 16; half of
    that of the root, 6 roundings behind it: 22 2^-24."""
    h = float(np.float16(value))
    row = np.full((1, cols), h, np.float16)
    d, w = hip.DeviceMatrix(1, cols, np.float16, data=row), hip.DeviceMatrix(1, cols, np.float16, data=np.ones((1, cols), np.float16))
    codes, scale, y = hip.DeviceMatrix(1, cols, np.int8), hip.DeviceMatrix(1, 1, np.float32), hip.DeviceMatrix(1, cols, np.float16)
    eps = float(np.float32(1e-5))
    hip.rmsnorm(d, w, codes, y_scales=scale, eps=eps)
    hip.rmsnorm(d, w, y, eps=eps)
    hip.sync()
    rho = 1 / np.sqrt(h * h + eps)
    assert abs(float(scale.download()[0, 0]) / (h * rho / 127) - 1) <= 22 * 2.0 ** -24
    assert (codes.download() == 127).all()
    assert (np.abs(y.download().astype(np.float64) / (h * rho) - 1) <= 2.0 ** -11 + 22 * 2.0 ** -24).all()


@pytest.mark.parametrize("t", [np.float16, np.float32])
@pytest.mark.parametrize("q8", [False, True])
def test_more_rows_than_a_launch_takes(hip, t, q8):
    """2^21 rows a launch: every operand of the second one from its place on; rows behind the last stay as they were."""
    rows, cols = (1 << 21) + 5, 3
    rng = np.random.default_rng(8)
    x, r = (rng.integers(-9, 10, (rows, cols)).astype(t) for _ in range(2))
    x[:, 0], r[:, 0] = 20, 1                              # (no row of zeros)
    w = np.array([[1, 0.5, -2]], t)
    dx, dr, dw = hip.DeviceMatrix(rows, cols, t, 4, x), hip.DeviceMatrix(rows, cols, t, data=r), hip.DeviceMatrix(1, cols, t, data=w)
    dh = hip.DeviceMatrix(rows + 2, cols, t, 5, pad_value=-777.0)
    dy = hip.DeviceMatrix(rows + 2, cols, np.int8 if q8 else t, 4, pad_value=77)
    ds = hip.DeviceMatrix(1, rows + 2, np.float32, data=np.full((1, rows + 2), -5, np.float32)) if q8 else None
    dh.rows = dy.rows = rows
    if q8:
        ds.cols = rows
    hip.rmsnorm(dx, dw, dy, residual=dr, sum_out=dh, y_scales=ds, eps=0.0)
    hip.sync()
    dh.rows = dy.rows = rows + 2
    h = (x + r).astype(np.float64)
    got = dh.download_raw()
    assert np.array_equal(got[:rows, :cols], h) and (got[rows:] == -777.0).all() and (got[:, cols:] == -777.0).all()
    p = h * w.astype(np.float64)
    rho = 1 / np.sqrt((h * h).mean(1))
    got = dy.download_raw()
    assert (got[rows:] == 77).all() and (got[:, cols:] == 77).all()
    if not q8:
        some = p != 0
        assert (np.abs(got[:rows, :cols][some] / (p * rho[:, None])[some] - 1) <= (2.0 ** -11 if t == np.float16 else 0) + 8 * 2.0 ** -24).all()
        return
    top = np.abs(p).max(1)
    exact = 127 * p / top[:, None]                         # quotients of small whole numbers: in 64 bits a half is a half
    assert np.array_equal(got[:rows, :cols], np.rint(exact))
    ds.cols = rows + 2
    s = ds.download()[0]
    assert (s[rows:] == -5).all() and (np.abs(s[:rows] / (top * rho / 127) - 1) <= 8 * 2.0 ** -24).all()
