"""The 4-bit layer without a GPU: sizes, refusals, and the layout that the tests and the kernels share."""
import ctypes

import numpy as np
import pytest

from decx_amd import hip
from oracle import q4_reference as ref

P, BAD, NOT_INIT = ctypes.c_void_p, -1, -2


@pytest.mark.parametrize("N,K", [(0, 5), (5, 0), (1, 1), (16, 128), (17, 129), (5003, 7001)])
def test_sizes(N, K):
    L = hip.lib()
    nt, kt = ref.tiles(N, K)
    assert L.decx_hip_q4_codes_bytes(N, K) == nt * kt * 1024
    for group in (32, 64, 128):
        assert L.decx_hip_q4_scales_count(N, K, group) == nt * kt * 16 * (128 // group)
    assert L.decx_hip_q4_scales_count(N, K, 16) == 0


@pytest.mark.parametrize("group", [32, 64, 128])
def test_the_reference_layout_reads_back(group):
    rng = np.random.default_rng(group)
    for N, K in ((1, 1), (16, 128), (17, 300), (40, 257)):
        G = -(-K // group)
        code, scale, zero = rng.integers(0, 16, (N, K)), rng.random((N, G)).astype(np.float16), rng.integers(0, 16, (N, G))
        got = ref.unpack(*ref.pack(code, scale, zero, group), N, K, group)
        assert all(np.array_equal(a, b) for a, b in zip(got, (code, scale, zero)))
        assert got[0].shape == (N, K)


def gemm_args(**change):
    a = dict(X=P(32), codes=P(32), scales=P(32), zeros=P(32), C=P(64), Y=P(32), M=4, N=20, K=130, group=64, ldx=130, ldc=20, ldy=20,
             alpha=1.0, beta=1.0, f32=0, ws=None, ws_bytes=0, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [dict(X=None), dict(codes=None), dict(scales=None), dict(Y=None), dict(group=16), dict(group=0), dict(group=256),
                                    dict(ldx=129), dict(ldy=19), dict(ldc=19), dict(codes=P(40)), dict(scales=P(34)), dict(zeros=P(33)),
                                    dict(X=P(33)), dict(Y=P(33)), dict(C=P(33)), dict(Y=P(34), f32=1), dict(K=0xffffff80, ldx=0xffffffff),
                                    dict(N=0xfffffff0, K=128, ldy=0xffffffff, ldc=0),
                                    dict(C=P(48), Y=P(48), ldc=0), dict(C=P(48), Y=P(48), ldc=21), dict(N=(1 << 25) + 1, ldy=1 << 26, ldc=0),
                                    dict(M=1 << 31, N=1 << 20, ldy=1 << 20, ldc=0)])
def test_products_refuse(change):
    L = hip.lib()
    assert L.decx_hip_gemm_q4_f16(*gemm_args(**change)) == BAD
    if "X" not in change or change["X"] is None:
        a = gemm_args(**change)
        assert L.decx_hip_gemm_q4_i8(a[0], P(32), *a[1:]) == BAD


def test_what_is_allowed_gets_as_far_as_the_missing_gpu():
    """(in a process that never initialised the library: every call is refused for that alone)"""
    import subprocess
    import sys
    code = ("import sys; sys.path.insert(0, 'tests'); import test_q4_layout as t; L = t.hip.lib(); P = t.P\n"
            "for c in ({}, dict(zeros=None), dict(C=None, ldc=0), dict(ldc=0), dict(K=0, X=None, codes=None, scales=None), dict(M=0, X=None),\n"
            "          dict(group=32, zeros=P(36)), dict(X=P(34)), dict(Y=P(36), f32=1)):\n"
            "    a = t.gemm_args(**c)\n"
            "    assert L.decx_hip_gemm_q4_f16(*a) == -2, c\n"
            "    assert L.decx_hip_gemm_q4_i8(a[0], P(32), *a[1:]) == -2, c\n"
            "a = t.gemm_args(); assert L.decx_hip_gemm_q4_i8(P(33), P(32), *a[1:]) == -2\n"
            "assert L.decx_hip_q4_quantize_f16(P(34), P(32), P(32), None, 3, 5, 5, 64, None) == -2\n"
            "assert L.decx_hip_q4_dequantize_f32(P(32), P(32), None, P(36), 3, 5, 5, 64, None) == -2\n"
            "assert L.decx_hip_gemm_q4_f16(*t.gemm_args(C=P(48), Y=P(48))) == -2\n"
            "assert L.decx_hip_rmsnorm_f16(P(32), None, P(64), None, P(33), P(96), 2, 8, 8, 0, 0, 8, 1e-5, None) == -2\n"
            "assert L.decx_hip_rmsnorm_f32(P(32), P(32), P(64), P(32), P(32), None, 2, 8, 8, 8, 8, 8, 0.0, None) == -2\n"
            "assert L.decx_hip_rmsnorm_f32(P(32), P(128), P(64), P(128), P(32), None, 1, 8, 9, 8, 10, 8, 0.0, None) == -2\n")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120, cwd=hip._PKG + "/..")


def test_x_scales_are_needed():
    a = gemm_args()
    assert hip.lib().decx_hip_gemm_q4_i8(a[0], None, *a[1:]) == BAD
    assert hip.lib().decx_hip_gemm_q4_i8(a[0], P(34), *a[1:]) == BAD


def test_what_a_workspace_is_good_for():
    L = hip.lib()
    for i8 in (0, 1):
        assert L.decx_hip_gemm_q4_workspace(i8, 1, 4096, 4096, 128) == 0 and L.decx_hip_gemm_q4_workspace(i8, 4096, 8192, 8192, 128) == 0
        need = L.decx_hip_gemm_q4_workspace(i8, 128, 8192, 8192, 128)
        assert need and need % (128 * 8192 * 4) == 0 and need // (128 * 8192 * 4) in range(2, 9)      # the sums of that many ranges
        assert L.decx_hip_gemm_q4_workspace(i8, 128, 8192, 8192, 100) == 0 and L.decx_hip_gemm_q4_workspace(i8, 0, 8192, 8192, 128) == 0


@pytest.mark.parametrize("change", [dict(W=None), dict(codes=None), dict(scales=None), dict(ldw=7), dict(group=48), dict(codes=P(24)), dict(zeros=P(33)),
                                    dict(scales=P(34)), dict(W=P(33))])
def test_quantisation_refuses(change):
    L = hip.lib()
    a = dict(W=P(32), codes=P(32), scales=P(32), zeros=P(32), N=3, K=8, ldw=8, group=64, stream=None)
    a.update(change)
    for fn in (L.decx_hip_q4_quantize_f16, L.decx_hip_q4_quantize_f32):
        assert fn(*a.values()) == BAD
    v = list(a.values())
    for fn in (L.decx_hip_q4_dequantize_f16, L.decx_hip_q4_dequantize_f32):
        assert fn(v[1], v[2], v[3], v[0], *v[4:]) == BAD


@pytest.mark.parametrize("change", [dict(x=None), dict(weight=None), dict(y=None), dict(cols=0), dict(ldx=7), dict(ldr=7), dict(lds=7), dict(ldy=7),
                                    dict(eps=-1.0), dict(eps=float("nan")), dict(x=P(33)), dict(residual=P(33)), dict(weight=P(33)), dict(sum=P(33)),
                                    dict(y=P(33), y_scales=None), dict(y_scales=P(34)), dict(rows=0x80000000),
                                    # an output in the place of an input: at another pitch, of another type, or where all rows read
                                    dict(sum=P(32), lds=9), dict(sum=P(64), lds=9), dict(sum=P(96)), dict(y=P(32)), dict(y=P(64)), dict(y=P(128)), dict(y=P(96), y_scales=None),
                                    dict(y=P(32), y_scales=None, ldy=9), dict(y=P(128), y_scales=None, ldy=9), dict(y_scales=P(96)), dict(y_scales=P(160))])
def test_norm_refuses(change):
    L = hip.lib()
    a = dict(x=P(32), residual=P(64), weight=P(96), sum=P(128), y=P(160), y_scales=P(192), rows=3, cols=8, ldx=8, ldr=8, lds=8, ldy=8, eps=1e-5, stream=None)
    a.update(change)
    for fn in (L.decx_hip_rmsnorm_f16, L.decx_hip_rmsnorm_f32):
        assert fn(*a.values()) == BAD
