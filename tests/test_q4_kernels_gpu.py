"""Every kernel of the products with 4-bit weights on data, each at sizes with a rest in every direction, whatever the planner
would take there.  Against the definition in 64 bits, with the bound that oracle/q4_reference.py derives."""
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
