"""The root-mean-square norm against its definition in 64 bits.

The sum and the 8-bit codes are exact by definition and have to be equal.  Tolerances of the rest, derived: a sum of squares
of n terms in fp32 is off by at most (n / 64 + 24) 2^-24 of itself (a thread adds at most n / 64 of them one after the other,
then at most 24 more meet over lanes and wavefronts; the squares round once each: 1 more), its root by half of that; mean,
eps, root, reciprocal and two products add at most 6 roundings.  fp32 rows are summed in 64 bits: 6 roundings of the result
at most.  fp16 results add half a step, 2^-11 of the value and 2^-25."""
import ctypes

import numpy as np
import pytest

from oracle import q4_reference as ref

pytestmark = pytest.mark.gpu

F = {"f16": np.float16, "f32": np.float32}


@pytest.fixture(scope="module")
def hip():
    from decx_amd import hip as h
    h.init()
    return h


def relative(cols, t):
    return ((cols / 64 + 25) / 2 + 6) * 2.0 ** -24 if t == np.float16 else 6 * 2.0 ** -24


def check(hip, x, residual, weight, eps, q8, keep, pad=0, off=0, in_place=None, stream=None):
    rows, cols = x.shape
    t = x.dtype
    up = lambda a, p, name: None if a is None else hip.DeviceMatrix(a.shape[0], cols, t, cols + p, a, pad_value=np.nan, offset_elems=off)   # noqa: E731
    dx, dr, dw = up(x, pad, "x"), up(residual, 2 * pad, "residual"), up(weight[None], 0, "weight")
    if q8:
        dy = hip.DeviceMatrix(rows, cols, np.int8, cols + 3 * pad, pad_value=77, offset_elems=off)
        ds = hip.DeviceMatrix(1, rows, np.float32)
    else:
        dy, ds = hip.DeviceMatrix(rows, cols, t, cols + 3 * pad, pad_value=-777.0, offset_elems=off), None
    dsum = hip.DeviceMatrix(rows, cols, t, cols + pad, pad_value=-777.0, offset_elems=off) if keep else None
    if in_place == "sum in residual":
        dsum = dr
    elif in_place == "sum in x":
        dsum = dx
    elif in_place == "y in x":
        dy = dx
    print("norm", rows, cols, t, q8, keep, in_place, flush=True)
    hip.rmsnorm(dx, dw, dy, residual=dr, sum_out=dsum, y_scales=ds, eps=eps, stream=stream)
    hip.sync(stream)
    want_sum, want, want_scale = ref.rmsnorm(x, residual, weight, eps, q8)
    if dsum is not None:
        raw = dsum.download_raw()
        assert np.array_equal(raw[:, :cols], want_sum, equal_nan=True)
        if in_place is None:
            assert (raw[:, cols:] == -777.0).all()
    raw = dy.download_raw()
    got = raw[:, :cols]
    if q8:
        assert (raw[:, cols:] == 77).all()
        assert np.array_equal(got, want)
        s = ds.download()[0].astype(np.float64)
        assert np.array_equal(np.isnan(s), np.isnan(want_scale))
        fine = np.isfinite(want_scale)
        assert (np.abs(s - want_scale)[fine] <= (relative(cols, t) + 2.0 ** -23) * want_scale[fine] + 2.0 ** -149).all()
    else:
        assert in_place or (raw[:, cols:] == -777.0).all()
        tol = relative(cols, t) * np.abs(want)
        tol = tol + (2.0 ** -11 * (np.abs(want) + tol) + 2.0 ** -25 if t == np.float16 else 2.0 ** -149)
        fine = np.isfinite(want)
        assert (np.abs(got.astype(np.float64) - want)[fine] <= tol[fine]).all()
    return raw


def rows_of(rng, rows, cols, t, wild=True):
    x = rng.standard_normal((rows, cols)) * (1 + 40 * (rng.random((1, cols)) < 0.02))
    if wild:
        x *= 10.0 ** rng.integers(-3, 2, (rows, 1))
    return x.astype(t)


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (5, 7), (2, 64), (4, 255), (3, 256), (7, 511), (2, 513), (3, 1000), (2, 2049), (5, 4096), (3, 5001), (2, 8192),
                                       (2, 8193), (3, 16385), (2, 32768), (2, 32769), (3, 40001)])
def test_norms_of_all_lengths(hip, t, rows, cols):
    rng = np.random.default_rng([rows, cols])
    x, r, w = rows_of(rng, rows, cols, F[t]), rows_of(rng, rows, cols, F[t]), (1 + rng.standard_normal(cols) * 0.3).astype(F[t])
    check(hip, x, r, w, 1e-5, True, True, pad=1)
    check(hip, x, None, w, 1e-6, False, False, pad=3)
    check(hip, x, r, w, 1e-5, False, True)
    check(hip, x, None, w, 1e-5, True, False, off=1)
    check(hip, x, r, w, 1e-5, True, False)


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("cols", [100, 4096, 40001])
def test_norms_in_place(hip, t, cols):
    rng = np.random.default_rng(cols)
    x, r, w = rows_of(rng, 6, cols, F[t]), rows_of(rng, 6, cols, F[t]), (1 + rng.standard_normal(cols) * 0.3).astype(F[t])
    check(hip, x, r, w, 1e-5, True, True, in_place="sum in residual")
    check(hip, x, r, w, 1e-5, True, True, in_place="sum in x")
    check(hip, x, r, w, 1e-5, False, False, in_place="y in x")
    check(hip, x, None, w, 1e-5, False, False, in_place="y in x")


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("cols", [60, 3000, 40001])
def test_codes_next_to_a_half(hip, t, cols):
    """Whole numbers whose 127-fold over the largest is a half, or as near to one as numbers of the type come."""
    rng = np.random.default_rng(cols)
    x = rng.integers(-254, 255, (8, cols)).astype(np.float64)
    x[:, cols // 2] = 254                                                # 127 x / 254 = x / 2: every odd one is a half
    x[4:] = np.nextafter(x[4:].astype(F[t]), F[t](0)).astype(np.float64)
    x[4:, cols // 2] = 254
    w = np.ones(cols)
    w[::3] = 0.5
    w[cols // 2] = 1
    check(hip, x.astype(F[t]), None, w.astype(F[t]), 1e-5, True, False)


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("cols", [40, 2000, 40001])
def test_rows_of_nothing_and_of_what_is_not_finite(hip, t, cols):
    rng = np.random.default_rng(cols)
    x, w = rows_of(rng, 8, cols, F[t], wild=False), (1 + rng.standard_normal(cols) * 0.3).astype(F[t])
    top = np.finfo(F[t]).max
    x[0] = 0
    x[1, 3], x[2, cols - 1], x[3, 0] = np.nan, np.inf, -np.inf
    x[4] = top                                                          # the largest: squares beyond fp32 for fp32 rows
    x[5] = np.finfo(F[t]).tiny
    x[6, 1:] = 0
    check(hip, x, None, w, 1e-5, True, True)
    d = hip.DeviceMatrix(8, cols, F[t], data=x)
    y = hip.DeviceMatrix(8, cols, F[t])
    hip.rmsnorm(d, hip.DeviceMatrix(1, cols, F[t], data=w[None]), y)
    hip.sync()
    got = y.download().astype(np.float64)
    with np.errstate(all="ignore"):
        want = ref.rmsnorm(x, None, w, 1e-5, False)[1]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    tol = relative(cols, F[t]) * np.abs(want) + (2.0 ** -11 * np.abs(want) * (1 + 2.0 ** -9) + 2.0 ** -25 if t == "f16" else 2.0 ** -149)
    assert (np.abs(got - want)[fine] <= tol[fine]).all()
    bad = w.copy(); bad[1] = np.inf
    check(hip, rows_of(rng, 3, cols, F[t]), None, bad, 1e-5, True, False)


def test_rows_beyond_4_gib(hip):
    rng = np.random.default_rng(3)
    cols, ld, rows = 1000, 1200000000, 3
    x, w = rng.standard_normal((rows, cols)).astype(np.float16), np.ones((1, cols), np.float16)
    L, at = hip.lib(), lambda d, m, e: ctypes.c_void_p(d.ptr.value + m * ld * e)                 # noqa: E731
    dx, dy = hip.DeviceMatrix(rows, ld, np.float16), hip.DeviceMatrix(rows, ld, np.int8)
    dw, ds = hip.DeviceMatrix(1, cols, np.float16, data=w), hip.DeviceMatrix(1, rows, np.float32)
    for m in range(rows):
        hip.check(L.decx_hip_memcpy2d_async(at(dx, m, 2), 2 * cols, x[m].ctypes.data, 2 * cols, 2 * cols, 1, 0, None))
    hip.sync()
    hip.check(L.decx_hip_rmsnorm_f16(dx.ptr, None, dw.ptr, None, dy.ptr, ds.ptr, rows, cols, ld, 0, 0, ld, 1e-5, None))
    hip.sync()
    want = ref.rmsnorm(x, None, w[0], 1e-5, True)[1]
    for m in range(rows):
        got = np.empty(cols, np.int8)
        hip.check(L.decx_hip_memcpy2d_async(got.ctypes.data, cols, at(dy, m, 1), cols, cols, 1, 1, None))
        hip.sync()
        assert np.array_equal(got, want[m])


def test_a_layer_step_by_step(hip):
    """The operators as a layer uses them: weights laid out once; residual added and normed to 8 bits; the product with 4-bit
    weights; the next residual added in its epilogue.  Each step is held against 64 bits on what the step before gave."""
    rng = np.random.default_rng(11)
    cols, hidden, group = 1000, 1500, 64
    w1, w2 = (rng.standard_normal((hidden, cols)) * 0.03).astype(np.float32), (rng.standard_normal((cols, hidden)) * 0.03).astype(np.float16)
    q1, q2 = hip.Q4Matrix(hidden, cols, group, True), hip.Q4Matrix(cols, hidden, group)
    hip.quantize_q4(hip.DeviceMatrix(hidden, cols, np.float32, data=w1), q1)
    hip.quantize_q4(hip.DeviceMatrix(cols, hidden, np.float16, data=w2), q2)
    v1, v2 = ref.values(*ref.quantize(w1, group, True), group), ref.values(*ref.quantize(w2, group, False), group)
    weight = (1 + rng.standard_normal(cols) * 0.2).astype(np.float16)
    dweight = hip.DeviceMatrix(1, cols, np.float16, data=weight[None])
    for rows in (1, 9, 70):
        x, r = rng.standard_normal((rows, cols)).astype(np.float16), (rng.standard_normal((rows, cols)) * 4).astype(np.float16)
        dx, dr = hip.DeviceMatrix(rows, cols, np.float16, data=x), hip.DeviceMatrix(rows, cols, np.float16, data=r)
        dq, ds = hip.DeviceMatrix(rows, cols, np.int8), hip.DeviceMatrix(1, rows, np.float32)
        dh, do = hip.DeviceMatrix(rows, hidden, np.float16), hip.DeviceMatrix(rows, cols, np.float16)
        hip.rmsnorm(dx, dweight, dq, residual=dr, sum_out=dr, y_scales=ds)
        hip.gemm_q4(dq, q1, dh, x_scales=ds)
        hip.gemm_q4(dh, q2, do, C=dr, alpha=1.0, beta=1.0)
        hip.sync()
        h, codes, _ = ref.rmsnorm(x, r, weight, 1e-5, True)
        assert np.array_equal(dr.download(), h) and np.array_equal(dq.download(), codes)
        xs = ds.download()[0]
        y, tol = ref.product(codes.astype(np.int8), xs, v1, None, 1, 1, group, False)
        got = dh.download()
        assert (np.abs(got.astype(np.float64) - y) <= tol).all()
        y, tol = ref.product(got, None, v2, h, 1.0, 1.0, group, False)
        assert (np.abs(do.download().astype(np.float64) - y) <= tol).all()
