"""Every kernel of the products with 4-bit weights on data, each at sizes with a rest in every direction, whatever the planner
would take there; products on ranges of K with their workspace, alone, in place, recorded and replayed.  Against the definition
in 64 bits, with the bound that oracle/q4_reference.py derives."""
import ctypes

import numpy as np
import pytest

from oracle import q4_reference as ref
from test_q4_gpu import Device4, weights
from test_q4_plans import ROWS_16, ROWS_16_NARROW, ROWS_16_WIDE, ROWS_32, ROWS_32_NARROW, ROWS_64, ROWS_64_NARROW, TILES_64x128, TILES_64x256, TILES_128x384

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from decx_amd import hip as h
    h.init()
    return h


class Product:
    """One product: the operands on the device, what the definition gives, and how far a result may be from it."""

    def __init__(self, hip, M, N, K, group, with_zeros, i8, f32=False, c=None, alpha=1.0, beta=1.0, ldx=0, ldc=0, off=0):
        rng = np.random.default_rng([M, N, K, group, with_zeros, i8, f32, off])
        self.hip, self.shape, self.i8, self.group, self.off = hip, (M, N, K), i8, group, off
        code, scale, zero = weights(rng, N, K, group, with_zeros)
        self.q = Device4(hip, code, scale, zero, group).Q
        self.out = np.float32 if f32 else np.float16
        if i8:
            x, xs = rng.integers(-128, 128, (M, K)).astype(np.int8), (rng.random(M) * 0.05 + 0.001).astype(np.float32)
            self.xs = hip.DeviceMatrix(1, M, np.float32, data=xs[None])
        else:
            x, xs = (rng.standard_normal((M, K)) * (1 + 20 * (rng.random((1, K)) < 0.02))).astype(np.float16), None
            self.xs = None
        self.x = hip.DeviceMatrix(M, K, x.dtype, K + ldx, x, pad_value=99 if i8 else np.nan, offset_elems=off)
        self.C = None if c is None else rng.standard_normal((c, N)).astype(self.out)
        self.c = None if c is None else hip.DeviceMatrix(c, N, self.out, N + ldc, self.C, pad_value=np.nan, offset_elems=off)
        self.alpha, self.beta = alpha, beta
        self.want, self.tol = ref.product(x, xs, ref.values(code, scale, zero, group), self.C, alpha, beta, group, f32)

    def result(self, ldy=0):
        return self.hip.DeviceMatrix(self.shape[0], self.shape[1], self.out, self.shape[1] + ldy, pad_value=-777.0, offset_elems=self.off)

    def room(self, splits=0):
        M, N, K = self.shape
        need = splits * M * ((N + 3) // 4 * 4) * 4 if splits else self.hip.lib().decx_hip_gemm_q4_workspace(1 if self.i8 else 0, M, N, K, self.group)
        return self.hip.DeviceMatrix(1, need, np.uint8) if need else None

    def into(self, y, plan=None, workspace=None, stream=None, in_place=False):
        self.hip.gemm_q4(self.x, self.q, y, y if in_place else self.c, self.alpha, self.beta, x_scales=self.xs, workspace=workspace, stream=stream, plan=plan)

    def check(self, y):
        raw = y.download_raw()
        N = self.shape[1]
        off_by = np.abs(raw[:, :N].astype(np.float64) - self.want)
        assert (off_by <= self.tol).all(), (off_by - self.tol).max()
        assert (raw[:, N:] == -777.0).all()                   # columns behind the last one stay as they were
        return raw

    def run(self, kernel, splits=1, ldy=0, in_place=False):
        """On that kernel and that many ranges of K, as even as the planner makes them."""
        kt = -(-self.shape[2] // 128)
        plan = self.hip.Q4Plan(kernel, splits, -(-kt // splits))
        y = self.result(ldy)
        if in_place:
            held = np.full((self.shape[0], y.pitch), -777.0, self.out)
            held[:, :self.shape[1]] = self.C
            y.upload_raw(held)
        print("product", self.shape, self.group, "int8" if self.i8 else "fp16", "kernel", kernel, "ranges", splits, flush=True)
        self.into(y, plan, self.room(splits) if splits > 1 else None, in_place=in_place)
        self.hip.sync()
        return self.check(y)


# block tiles of rows x columns: one row and column more than one or two of them, and fewer
TILED = [(TILES_64x128, 64, 128), (TILES_64x256, 64, 256), (TILES_128x384, 128, 384)]


@pytest.mark.parametrize("kernel,bm,bn", TILED)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("with_zeros", [False, True])
def test_tiled_kernels(hip, kernel, bm, bn, group, i8, with_zeros):
    shapes = [(bm + 1, bn + 1, 300), (2 * bm - 3, bn - 5, 128), (17, 2 * bn + 2, 127), (3 * bm, 16, 515), (40, bn, 1), (bm, 2 * bn, 640)]
    for at, (M, N, K) in enumerate(shapes):
        Product(hip, M, N, K, group, with_zeros, i8, f32=at % 2 == 1, ldx=at % 3, off=at % 2).run(kernel, ldy=at)
    # the epilogue: C at a pitch of its own, one row of it, Y itself; four columns at a time and one by one
    for N, f32 in ((bn + 4, False), (bn + 3, False), (bn + 4, True), (bn + 2, True)):
        Product(hip, bm + 9, N, 200, group, with_zeros, i8, f32, c=bm + 9, alpha=0.5, beta=-1.5, ldc=4 - N % 4).run(kernel)
        Product(hip, bm + 9, N, 200, group, with_zeros, i8, f32, c=1, alpha=2.0).run(kernel)
        Product(hip, bm + 9, N, 200, group, with_zeros, i8, f32, c=bm + 9, beta=2.0).run(kernel, in_place=True)


@pytest.mark.parametrize("kernel,bm,bn", TILED)
@pytest.mark.parametrize("i8", [False, True])
def test_tiled_kernels_on_many_tiles(hip, kernel, bm, bn, i8):
    """Enough block tiles that every XCD's range and the groups of 8 tile rows have a rest."""
    Product(hip, 19 * bm + 5, 3 * bn + 20, 260, 64, i8, i8).run(kernel)


@pytest.mark.parametrize("kernel,M", [(ROWS_16_NARROW, 1), (ROWS_16, 3), (ROWS_16_WIDE, 8), (ROWS_16_NARROW, 13), (ROWS_16, 16), (ROWS_16_WIDE, 5), (ROWS_32_NARROW, 17),
                                      (ROWS_32, 32), (ROWS_64_NARROW, 33), (ROWS_64, 64), (ROWS_64_NARROW, 131), (ROWS_64, 190)])
@pytest.mark.parametrize("i8", [False, True])
def test_kernels_of_few_rows(hip, kernel, M, i8):
    for at, (N, K) in enumerate([(50, 2200), (16, 300), (33, 128), (47, 77)]):
        for group in (32, 64, 128):
            Product(hip, M, N, K, group, at % 2 == 0, i8, c=M if at % 2 else None, ldx=at, off=at % 2).run(kernel, ldy=at)


@pytest.mark.parametrize("kernel,i8", [(ROWS_64_NARROW, False), (ROWS_64_NARROW, True), (ROWS_64, True)])
def test_more_rows_than_a_grid_has_workgroups_for(hip, kernel, i8):
    """The rows of the second launch: X, its factors, C and Y each from their place on."""
    M = 65535 * 64 + 70
    for c in (None, 1, M):
        Product(hip, M, 2, 3, 128, False, i8, c=c, ldx=1).run(kernel, ldy=1)


@pytest.mark.parametrize("kernel,M", [(ROWS_16_NARROW, 3), (ROWS_16, 9), (ROWS_16_WIDE, 13), (ROWS_32_NARROW, 18), (ROWS_32, 31), (ROWS_64_NARROW, 50), (ROWS_64, 70),
                                      (TILES_64x128, 65), (TILES_64x256, 40), (TILES_128x384, 130)])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("splits", [1, 2])
def test_rows_behind_the_last_stay_as_they_were(hip, kernel, M, i8, splits):
    if splits > 1 and kernel < TILES_64x128:
        return
    p = Product(hip, M, 37, 500, 64, True, i8)
    y = hip.DeviceMatrix(M + 3, 37, np.float16, pad_value=-777.0)
    y.upload_raw(np.full((M + 3, 37), -777.0, np.float16))
    y.rows = M
    p.into(y, hip.Q4Plan(kernel, splits, 4 // splits), p.room(splits) if splits > 1 else None)
    hip.sync()
    p.check(y)
    y.rows = M + 3
    assert (y.download_raw()[M:] == -777.0).all()


# ---- ranges of K -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kernel,bm,bn", TILED)
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("splits,K", [(2, 3 * 128 + 1), (3, 5 * 128), (4, 8 * 128 - 50), (8, 2000)])
def test_ranges_of_k(hip, kernel, bm, bn, i8, splits, K):
    """The last range shorter than the others and not, sums of whole quads and with a rest, every form of the epilogue."""
    group, with_zeros = {2: 32, 3: 64, 4: 128, 8: 64}[splits], splits % 4 == 0
    for M, N in ((bm + 2, bn + 4), (bm - 7, bn + 1)):
        plain = Product(hip, M, N, K, group, with_zeros, i8)
        assert np.array_equal(plain.run(kernel, splits), plain.run(kernel, splits))            # the same call gives the same bits
        Product(hip, M, N, K, group, with_zeros, i8, f32=True, c=1, alpha=0.5).run(kernel, splits, ldy=N % 4)
        Product(hip, M, N, K, group, with_zeros, i8, c=M, alpha=0.5, beta=-1.5, ldc=4 - N % 4, off=N % 2).run(kernel, splits)
        Product(hip, M, N, K, group, with_zeros, i8, c=M, beta=2.0).run(kernel, splits, in_place=True)


SPLIT = [(65, 300, 4100, 128, False), (65, 302, 4100, 64, False), (65, 2052, 2100, 128, True), (65, 2050, 2100, 32, True), (256, 2048, 4096, 32, False)]


@pytest.mark.parametrize("M,N,K,group,i8", SPLIT)
def test_products_that_the_planner_splits(hip, M, N, K, group, i8):
    for c in (None, 1, M):
        p = Product(hip, M, N, K, group, c == 1, i8, c=c, alpha=0.5 if c else 1.0)
        ws = p.room()
        need = ws.pitch
        assert need > 0 and hip.plan_q4(i8, M, N, K, group, need).k_splits > 1
        # room for all, none, and too little of it: fewer ranges or none, never an error
        for given in (ws, None, hip.DeviceMatrix(1, need - 1, np.uint8), hip.DeviceMatrix(1, 16, np.uint8)):
            y = p.result(ldy=3)
            print("product", M, N, K, group, i8, "workspace", given.pitch if given else 0, flush=True)
            p.into(y, workspace=given)
            hip.sync()
            p.check(y)
    y = p.result()
    y.upload_raw(p.C)
    p.into(y, workspace=ws, in_place=True)
    hip.sync()
    p.check(y)


def test_recorded_products_on_ranges_replay_beside_eager_ones(hip):
    """Two launches that meet in a workspace: recorded, replayed back to back on one stream (which may share it), and beside
    eager calls on another stream with a workspace of their own."""
    rt = ctypes.CDLL("libamdhip64.so.7")
    vp = ctypes.c_void_p
    stream, other = hip.Stream(), hip.Stream()
    products = [Product(hip, M, N, K, group, True, i8) for M, N, K, group, i8 in SPLIT]
    for p in products:
        ws = [p.room(), p.room()]
        assert ws[0] is not None
        ys = [p.result() for _ in range(3)]
        graph, run = vp(), vp()
        p.into(ys[0], workspace=ws[0], stream=stream.handle)
        stream.sync()
        want = p.check(ys[0])
        assert rt.hipStreamBeginCapture(stream.handle, 0) == 0
        p.into(ys[0], workspace=ws[0], stream=stream.handle)
        p.into(ys[1], workspace=ws[0], stream=stream.handle)
        assert rt.hipStreamEndCapture(stream.handle, ctypes.byref(graph)) == 0
        assert rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
        for replay in range(4):
            for y in ys:
                y.upload_raw(np.full((y.rows, y.pitch), -3.0, y.dtype))
            ws[0].upload_raw(np.full((1, ws[0].pitch), 255, np.uint8))        # (NaNs: sums that were not written show)
            print("replay", p.shape, replay, flush=True)
            p.into(ys[2], workspace=ws[1], stream=other.handle)
            assert rt.hipGraphLaunch(run, stream.handle) == 0
            p.into(ys[2], workspace=ws[1], stream=other.handle)
            assert rt.hipGraphLaunch(run, stream.handle) == 0
            stream.sync(); other.sync()
            assert all(np.array_equal(y.download_raw(), want) for y in ys)
        assert rt.hipGraphExecDestroy(run) == 0 and rt.hipGraphDestroy(graph) == 0
    stream.destroy(); other.destroy()
