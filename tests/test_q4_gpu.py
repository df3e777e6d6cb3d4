"""Products with 4-bit weights, and the making of such weights, against their definitions in 64 bits."""
import ctypes

import numpy as np
import pytest

from oracle import q4_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from decx_amd import hip as h
    h.init()
    return h


def weights(rng, N, K, group, with_zeros):
    G = -(-K // group)
    code = np.clip(np.rint(rng.standard_normal((N, K)) * 3 + 8), 0, 15).astype(np.int64)
    scale = (np.abs(rng.standard_normal((N, G))) * 0.01 + 0.003).astype(np.float16)
    zero = rng.integers(0, 16, (N, G)) if with_zeros else None
    return code, scale, zero


class Device4:
    """A Q4Matrix filled with given parts; what the padding of the arrays holds is as unkind as it may be."""

    def __init__(self, hip, code, scale, zero, group):
        N, K = code.shape
        self.Q = hip.Q4Matrix(N, K, group, zero is not None)
        parts = ref.pack(code, scale, zero, group, pad_code=15, pad_scale=np.nan, pad_zero=3)
        for dm, host in zip((self.Q.codes, self.Q.scales, self.Q.zeros), parts):
            if host is not None and host.size:
                dm.upload_raw(host.reshape(1, -1))


def run_product(hip, rng, M, N, K, group, with_zeros, i8, f32, c_rows=None, alpha=1.0, beta=1.0, ldx=None, ldy=None, off=0, stream=None, workspace=None,
                in_place=False):
    code, scale, zero = weights(rng, N, K, group, with_zeros)
    d = Device4(hip, code, scale, zero, group)
    out = np.float32 if f32 else np.float16
    if i8:
        x = rng.integers(-128, 128, (M, K)).astype(np.int8)
        xs = (rng.random(M) * 0.05 + 0.001).astype(np.float32)
        dx = hip.DeviceMatrix(M, K, np.int8, ldx or K, x, pad_value=99, offset_elems=off)
        dxs = hip.DeviceMatrix(1, M, np.float32, data=xs[None])
    else:
        x = (rng.standard_normal((M, K)) * (1 + 20 * (rng.random((1, K)) < 0.02))).astype(np.float16)
        xs = dxs = None
        dx = hip.DeviceMatrix(M, K, np.float16, ldx or K, x, pad_value=np.nan, offset_elems=off)
    C = None if c_rows is None else rng.standard_normal((c_rows, N)).astype(out)
    dy = hip.DeviceMatrix(M, N, out, ldy or N, C if in_place else None, pad_value=-777.0, offset_elems=off)
    dc = dy if in_place else None if C is None else hip.DeviceMatrix(c_rows, N, out, N + 3, C, pad_value=np.nan, offset_elems=off)
    print("product", M, N, K, group, with_zeros, i8, f32, c_rows, flush=True)
    hip.gemm_q4(dx, d.Q, dy, dc, alpha, beta, x_scales=dxs, workspace=workspace, stream=stream)
    hip.sync(stream)
    raw = dy.download_raw()
    want, tol = ref.product(x, xs, ref.values(code, scale, zero, group), C, alpha, beta, group, f32)
    got = raw[:, :N].astype(np.float64)
    assert np.isfinite(got).all()
    off_by = np.abs(got - want)
    assert (off_by <= tol).all(), (off_by - tol).max()
    assert (raw[:, N:] == -777.0).all()                       # columns behind the last one stay as they were
    return raw


ODD = [(1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 33, 31), (3, 100, 250), (7, 503, 701), (15, 16, 1000), (16, 48, 384), (17, 47, 383), (33, 130, 515),
       (64, 64, 640), (65, 200, 257), (100, 77, 1029), (129, 250, 130), (200, 515, 259), (257, 300, 1030)]


@pytest.mark.parametrize("M,N,K", ODD)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_products_of_odd_sizes(hip, M, N, K, group):
    for at, (with_zeros, i8, f32) in enumerate([(False, False, False), (True, True, False), (True, False, True), (False, True, True)]):
        run_product(hip, np.random.default_rng([M, N, K, group, at]), M, N, K, group, with_zeros, i8, f32, ldx=K + at, ldy=N + 2 * at)


@pytest.mark.parametrize("M,N,K,group", [(1, 4096, 4096, 128), (1, 1024, 16384, 32), (5, 2048, 11008, 64), (1, 30001, 512, 128), (16, 6000, 2000, 64),
                                         (48, 1024, 4096, 128), (100, 2048, 1024, 32), (256, 1024, 2048, 128), (511, 1030, 1111, 64), (1000, 515, 640, 128)])
@pytest.mark.parametrize("i8", [False, True])
def test_products_of_layers(hip, M, N, K, group, i8):
    rng = np.random.default_rng([M, N, K])
    workspace = hip.DeviceMatrix(1, 4 << 20, np.float32)
    raw = run_product(hip, rng, M, N, K, group, M % 2 == 0, i8, False, c_rows=M if M > 5 else None, alpha=0.5, beta=-1.5, workspace=workspace)
    again = run_product(hip, np.random.default_rng([M, N, K]), M, N, K, group, M % 2 == 0, i8, False, c_rows=M if M > 5 else None, alpha=0.5, beta=-1.5,
                        workspace=workspace)
    assert np.array_equal(raw, again)                         # the same call gives the same bits
    run_product(hip, np.random.default_rng([M, N, K]), M, N, K, group, M % 2 == 0, i8, True, c_rows=1, alpha=2.0, beta=1.0)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 6, 7, 8, 9, 11, 12, 13, 16, 17, 19, 21, 31, 33, 37, 41, 47, 63])
@pytest.mark.parametrize("i8", [False, True])
def test_products_of_few_rows(hip, M, i8):
    """Every number of loads of X, with and without a part of one, by K below a column tile, of whole ones and with a rest; one
    and two row tiles of W a workgroup, and 8 and 16 wavefronts."""
    rng = np.random.default_rng(M)
    for N, K, group in ((40, 100, 32), (70, 256, 128), (4100, 700, 64), (8200, 300, 128), (8200, 90, 64)):
        run_product(hip, rng, M, N, K, group, M % 2 == 0, i8, False, ldx=K + M % 3)


@pytest.mark.parametrize("off", [1, 3, 7])
@pytest.mark.parametrize("M,N,K", [(1, 100, 517), (9, 64, 256), (70, 99, 777), (300, 270, 600)])
def test_products_at_any_alignment(hip, off, M, N, K):
    for i8 in (False, True):
        run_product(hip, np.random.default_rng([off, M]), M, N, K, 64, True, i8, False, c_rows=M, alpha=1.0, beta=1.0, ldx=K + off, ldy=N + off, off=off)


@pytest.mark.parametrize("M,N,K", [(1, 40, 300), (20, 60, 256), (150, 300, 500)])
def test_c_may_be_y(hip, M, N, K):
    for i8 in (False, True):
        run_product(hip, np.random.default_rng([M, N]), M, N, K, 128, False, i8, True, c_rows=M, alpha=0.25, beta=2.0, ldy=N + 5, in_place=True)


def test_empty_products(hip):
    rng = np.random.default_rng(0)
    for M, N in ((3, 20), (40, 40)):
        for i8 in (False, True):
            raw = run_product(hip, rng, M, N, 0, 64, False, i8, False)
            assert (raw == 0).all()
            run_product(hip, rng, M, N, 0, 64, False, i8, False, c_rows=M, alpha=3.0, beta=0.5)
    L, P = hip.lib(), ctypes.c_void_p
    assert L.decx_hip_gemm_q4_f16(None, None, None, None, None, None, 0, 5, 5, 64, 5, 0, 5, 1.0, 1.0, 0, None, 0, None) == 0
    assert L.decx_hip_gemm_q4_f16(None, None, None, None, None, None, 5, 0, 5, 64, 5, 0, 5, 1.0, 1.0, 0, None, 0, None) == 0
    assert L.decx_hip_q4_quantize_f32(None, None, None, None, 0, 5, 5, 64, None) == 0
    assert L.decx_hip_rmsnorm_f16(None, None, None, None, None, None, 0, 5, 5, 0, 0, 5, 1e-5, None) == 0


@pytest.mark.parametrize("M", [1, 30, 200])
def test_what_is_not_a_number_stays_in_its_row_and_column(hip, M):
    rng = np.random.default_rng(M)
    N, K, group = 50, 400, 64
    code, scale, zero = weights(rng, N, K, group, True)
    code[7, :] = 9
    scale[5, 3] = np.nan
    x = rng.standard_normal((M, K)).astype(np.float16)
    x[M - 1, 17] = np.inf
    d = Device4(hip, code, scale, zero, group)
    dx, dy = hip.DeviceMatrix(M, K, np.float16, data=x), hip.DeviceMatrix(M, N, np.float32)
    hip.gemm_q4(dx, d.Q, dy)
    hip.sync()
    got = dy.download()
    with np.errstate(all="ignore"):
        w = ref.values(code, scale, zero, group)
        want = (x[:, None, :].astype(np.float64) * w[None]).sum(2)
    assert np.isnan(got[:, 5]).all()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    fine = np.isfinite(want)
    assert np.allclose(got[fine], want[fine], rtol=1e-4, atol=1e-4)
    assert np.array_equal(np.sign(got[np.isinf(want)]), np.sign(want[np.isinf(want)]))
    # int8 rows: the factor of a row alone
    xi, xs = rng.integers(-128, 128, (M, K)).astype(np.int8), np.ones(M, np.float32)
    xs[M - 1] = np.nan
    di, ds = hip.DeviceMatrix(M, K, np.int8, data=xi), hip.DeviceMatrix(1, M, np.float32, data=xs[None])
    hip.gemm_q4(di, d.Q, dy, x_scales=ds)
    hip.sync()
    got = dy.download()
    assert np.isnan(got[M - 1]).all() and np.isnan(got[:, 5]).all()
    assert np.isfinite(np.delete(got[:M - 1], 5, 1)).all()


def test_a_captured_product_replays_beside_eager_ones_on_other_streams(hip):
    rt = ctypes.CDLL("libamdhip64.so.7")
    vp = ctypes.c_void_p
    rng = np.random.default_rng(5)
    cases = [(1, 2048, 4096, False), (40, 512, 4096, True), (130, 512, 4096, False)]
    stream, other = hip.Stream(), hip.Stream()
    for M, N, K, i8 in cases:
        code, scale, zero = weights(rng, N, K, 128, False)
        d = Device4(hip, code, scale, zero, 128)
        x = rng.integers(-99, 99, (M, K)).astype(np.int8) if i8 else rng.standard_normal((M, K)).astype(np.float16)
        dx = hip.DeviceMatrix(M, K, x.dtype, data=x)
        dxs = hip.DeviceMatrix(1, M, np.float32, data=np.ones((1, M), np.float32)) if i8 else None
        need = max(1, int(hip.lib().decx_hip_gemm_q4_workspace(1 if i8 else 0, M, N, K, 128)))
        ys = [hip.DeviceMatrix(M, N, np.float16) for _ in range(3)]
        ws = [hip.DeviceMatrix(1, need, np.uint8) for _ in range(3)]
        hip.gemm_q4(dx, d.Q, ys[0], x_scales=dxs, workspace=ws[0], stream=stream.handle)
        stream.sync()
        want = ys[0].download()
        graph, run = vp(), vp()
        assert rt.hipStreamBeginCapture(stream.handle, 0) == 0
        hip.gemm_q4(dx, d.Q, ys[1], x_scales=dxs, workspace=ws[1], stream=stream.handle)
        assert rt.hipStreamEndCapture(stream.handle, ctypes.byref(graph)) == 0
        assert rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
        for replay in range(4):
            for y in ys[1:]:
                y.upload_raw(np.full((M, N), -3.0, np.float16))
            print("replay", M, replay, flush=True)
            hip.gemm_q4(dx, d.Q, ys[2], x_scales=dxs, workspace=ws[2], stream=other.handle)
            assert rt.hipGraphLaunch(run, stream.handle) == 0
            assert rt.hipGraphLaunch(run, stream.handle) == 0
            stream.sync(); other.sync()
            assert np.array_equal(ys[1].download(), want) and np.array_equal(ys[2].download(), want)
        assert rt.hipGraphExecDestroy(run) == 0 and rt.hipGraphDestroy(graph) == 0
    stream.destroy(); other.destroy()


def test_codes_beyond_4_gib(hip):
    """Row tiles whose codes begin past 2^32 bytes, rows of X and Y far apart: closed forms, all exact."""
    N, K, M = 70000, 131072, 2
    Q = hip.Q4Matrix(N, K, 128)
    assert Q.codes.nbytes > 1 << 32
    L = hip.lib()
    hip.check(L.decx_hip_memset_async(Q.codes.ptr, 0x99, Q.codes.nbytes, None))        # code 9: one step above the middle
    hip.check(L.decx_hip_memset_async(Q.scales.ptr, 0x3c, Q.scales.nbytes, None))      # 0x3c3c = 1.05859375
    s = float(np.array([0x3c3c], np.uint16).view(np.float16)[0])
    ld = 1500000000
    x = np.ones((M, K), np.float16); x[1] = -2
    dx, dy = hip.DeviceMatrix(M, ld, np.float16), hip.DeviceMatrix(M, ld, np.float32)
    for m in range(M):
        hip.check(L.decx_hip_memcpy2d_async(ctypes.c_void_p(dx.ptr.value + m * ld * 2), 2 * K, x[m].ctypes.data, 2 * K, 2 * K, 1, 0, None))
    hip.sync()
    print("product beyond 4 GiB", flush=True)
    hip.check(L.decx_hip_gemm_q4_f16(dx.ptr, *Q.parts(), None, dy.ptr, M, N, K, 128, ld, 0, ld, 1.0, 1.0, 1, None, 0, None))
    hip.sync()
    got = np.empty((M, N), np.float32)
    for m in range(M):
        hip.check(L.decx_hip_memcpy2d_async(got[m].ctypes.data, 4 * N, ctypes.c_void_p(dy.ptr.value + m * ld * 4), 4 * N, 4 * N, 1, 1, None))
    hip.sync()
    assert np.array_equal(got, np.broadcast_to(np.float32([[s * K], [-2 * s * K]]), (M, N)))


# ---- making them ------------------------------------------------------------------------------------------------------

def fetch(Q):
    c = Q.codes.download_raw().reshape(-1)
    s = Q.scales.download_raw().reshape(-1)
    return ref.unpack(c, s, None if Q.zeros is None else Q.zeros.download_raw().reshape(-1), Q.rows, Q.cols, Q.group)


def hard_rows(rng, N, K, dtype):
    """Rows with everything a group may hold: zeros, one value, only positive, quotients that are halves, tiny, huge."""
    W = (rng.standard_normal((N, K)) * 0.02).astype(np.float64)
    top = 6e4 if dtype == np.float16 else 3e38
    kinds = [lambda r: r * 0, lambda r: np.full_like(r, 0.3), lambda r: np.abs(r), lambda r: -np.abs(r) - 1, lambda r: np.rint(r * 400) / 2 * 0.25,
             lambda r: r * 1e-6, lambda r: r * 2e-8 / 0.02, lambda r: np.clip(r / 0.02 * top / 3, -top, top), lambda r: np.where(np.arange(r.size) % 37 == 0, 5.0, r),
             lambda r: (np.arange(r.size) % 15 - 7.0) / 2]
    for n in range(N):
        if n % 3 == 0:
            W[n] = kinds[n // 3 % len(kinds)](W[n])
    return W.astype(dtype)


@pytest.mark.parametrize("N,K", [(1, 1), (31, 128), (33, 130), (60, 515), (100, 1000)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_quantisation_by_its_definition(hip, N, K, group, dtype):
    """Codes, zero points and scales equal those of the definition in 64 bits, and come back as the values they stand for."""
    rng = np.random.default_rng([N, K, group])
    W = hard_rows(rng, N, K, dtype)
    for with_zeros in (False, True):
        for off in (0, 1):
            dW = hip.DeviceMatrix(N, K, dtype, K + 3 * off, W, pad_value=np.nan, offset_elems=off)
            Q = hip.Q4Matrix(N, K, group, with_zeros)
            hip.quantize_q4(dW, Q)
            hip.sync()
            want = ref.quantize(W, group, with_zeros)
            got = fetch(Q)
            assert np.array_equal(got[1].view(np.uint16), want[1].view(np.uint16))
            if with_zeros:
                assert np.array_equal(got[2], want[2])
            assert np.array_equal(got[0], want[0])
            v = ref.values(*want, group)
            for t in (np.float32, np.float16):
                back = hip.DeviceMatrix(N, K, t, K + 5, offset_elems=off, pad_value=-777.0)
                hip.dequantize_q4(Q, back)
                hip.sync()
                raw = back.download_raw()
                with np.errstate(over="ignore"):
                    assert np.array_equal(raw[:, :K], v.astype(t))
                assert (raw[:, K:] == -777.0).all()


def test_quantisation_of_what_is_not_finite(hip):
    rng = np.random.default_rng(1)
    W = rng.standard_normal((20, 256)).astype(np.float32)
    W[3, 10], W[4, 100], W[5, 200] = np.nan, np.inf, -np.inf
    for with_zeros in (False, True):
        Q = hip.Q4Matrix(20, 256, 64, with_zeros)
        hip.quantize_q4(hip.DeviceMatrix(20, 256, np.float32, data=W), Q)
        hip.sync()
        want, got = ref.quantize(W, 64, with_zeros), fetch(Q)
        bad = np.zeros((20, 4), bool); bad[3, 0] = bad[4, 1] = bad[5, 3] = True
        assert np.array_equal(np.isnan(got[1]), bad)
        assert np.array_equal(got[1][~bad], want[1][~bad]) and np.array_equal(got[0], want[0])


def test_padding_of_a_made_matrix_is_harmless(hip):
    """The arrays are whole tiles; what lies behind the last row and column stands for zero."""
    W = np.ones((3, 5), np.float32)
    Q = hip.Q4Matrix(3, 5, 32, True)
    for a in (Q.codes, Q.scales, Q.zeros):
        a.upload_raw(np.full((1, a.pitch), 255 if a.dtype == np.uint8 else np.nan, a.dtype))
    hip.quantize_q4(hip.DeviceMatrix(3, 5, np.float32, data=W), Q)
    hip.sync()
    whole = ref.unpack(Q.codes.download_raw().reshape(-1), Q.scales.download_raw().reshape(-1), Q.zeros.download_raw().reshape(-1), 16, 128, 32)
    v = ref.values(*whole, 32)
    assert np.isfinite(whole[1]).all()
    inside = np.zeros((16, 128), bool); inside[:3, :5] = True
    assert (v[~inside] == 0).all() and np.allclose(v[inside], 1, rtol=2.0 ** -10)
