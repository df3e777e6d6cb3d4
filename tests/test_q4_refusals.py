"""Calls of the 4-bit layer that are refused, and their neighbours that are not (no GPU: refusals come before the library looks
for one, and the others end with "not initialised" in a process of their own)."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from decx_amd import hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, BAD, NOT_INIT = ctypes.c_void_p, -1, -2


def calls_get_as_far_as_the_missing_gpu(code):
    """(in a process that never initialised the library, so that nothing can be launched)"""
    head = "import sys; sys.path.insert(0, 'tests')\nimport test_q4_refusals as t\nL, P = t.hip.lib(), t.P\n"
    subprocess.run([sys.executable, "-c", head + code], check=True, timeout=120, cwd=hip._PKG + "/..")


def quantise(name, N, K, group=64):
    W, parts = (P(1 << 20),), (P(2 << 20), P(3 << 20), None)
    return getattr(hip.lib(), name)(*(W + parts if "_quantize" in name else parts + W), N, K, K, group, None)


QUANTISE = ["decx_hip_q4_%s_%s" % (a, t) for a in ("quantize", "dequantize") for t in ("f16", "f32")]


@pytest.mark.parametrize("name", QUANTISE)
@pytest.mark.parametrize("N,K", [(33, 22369621 * 128), (16 * 31, 2164802 * 128 + 1), (1 << 30, 1), ((1 << 30) - 48, 1)])
def test_more_tiles_than_a_launch_has_threads_for(name, N, K):
    """Four tiles a workgroup of 256: from 2^26 - 3 tiles on the launch would have 2^32 threads."""
    assert -(-N // 16) * -(-K // 128) > (1 << 26) - 4
    assert quantise(name, N, K) == BAD


def test_the_largest_number_of_tiles():
    calls_get_as_far_as_the_missing_gpu("for name in t.QUANTISE: assert t.quantise(name, 960, 1118481 * 128) == t.NOT_INIT\n")


def test_rules_about_operands_in_one_place(tmp_path):
    exe = str(tmp_path / "operand_overlap_test")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", os.path.join(ROOT, "tests", "cpp", "operand_overlap_test.cpp"), "-o", exe],
                   check=True, timeout=300)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "all ok" in run.stdout, run.stdout + run.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("i8", [False, True])
def test_operands_in_one_place_are_refused(i8):
    """Through the entry points (the rules are asked only once the library is initialised); every buffer is large enough for
    whatever the call says it is, and a refused call leaves it as it was."""
    hip.init()
    L = hip.lib()
    M, N, K = 20, 64, 128
    names = ["X", "xs", "codes", "scales", "zeros", "C", "Y", "ws"]
    at = {n: hip.DeviceMatrix(1, 1 << 17, np.uint8, data=np.full((1, 1 << 17), 5, np.uint8)) for n in names + ["W"]}

    def product(**place):
        p = {n: at[place.get(n, n)].ptr for n in names}
        rest = (p["codes"], p["scales"], p["zeros"], p["C"], p["Y"], M, N, K, 64, K, N, N, 1.0, 1.0, 0, p["ws"], 1 << 17, None)
        return L.decx_hip_gemm_q4_i8(p["X"], p["xs"], *rest) if i8 else L.decx_hip_gemm_q4_f16(p["X"], *rest)

    def quantise(there, **place):
        p = {n: at[place.get(n, n)].ptr for n in ("W", "codes", "scales", "zeros")}
        parts = (p["codes"], p["scales"], p["zeros"])
        if there:
            return L.decx_hip_q4_quantize_f16(p["W"], *parts, N, K, K, 64, None)
        return L.decx_hip_q4_dequantize_f16(*parts, p["W"], N, K, K, 64, None)
    for other in ("X", "codes", "scales", "zeros") + (("xs",) if i8 else ()):
        assert product(Y=other) == BAD and product(ws=other) == BAD, other
    assert product(ws="C") == BAD and product(ws="Y") == BAD
    for a, b in (("W", "codes"), ("W", "scales"), ("W", "zeros")):
        assert quantise(True, **{a: b}) == BAD and quantise(False, **{a: b}) == BAD, (a, b)
    for a, b in (("codes", "scales"), ("codes", "zeros"), ("scales", "zeros")):
        assert quantise(True, **{a: b}) == BAD, (a, b)
    hip.sync()
    for n, d in at.items():
        assert (d.download() == 5).all(), n
    assert product() == 0 and product(C="Y") == 0 and quantise(False) == 0 and quantise(True) == 0
    hip.sync()


class Operand:
    """What hip.gemm_q4 and hip.rmsnorm look at of a DeviceMatrix."""

    def __init__(self, rows, cols, dtype, pitch=None):
        self.rows, self.cols, self.dtype, self.pitch, self.ptr = rows, cols, np.dtype(dtype), pitch or cols, P(1 << 20)


F16, F32, I8 = np.float16, np.float32, np.int8


@pytest.mark.parametrize("change", [dict(y_scales=Operand(1, 3, F32)), dict(y_scales=Operand(1, 5, F32)), dict(y_scales=Operand(1, 4, F16)),
                                    dict(y_scales=Operand(4, 1, F32, 2)), dict(weight=Operand(2, 8, F16)), dict(weight=Operand(1, 9, F16)),
                                    dict(weight=Operand(1, 8, F32)), dict(residual=Operand(4, 8, F32)), dict(residual=Operand(3, 8, F16)),
                                    dict(sum_out=Operand(4, 8, F32)), dict(sum_out=Operand(4, 9, F16)), dict(y=Operand(4, 8, F16)), dict(y=Operand(5, 8, I8))])
def test_the_view_of_the_norm_checks_its_operands(change):
    """(a y_scales of too few values would be written behind its end)"""
    a = dict(x=Operand(4, 8, F16), weight=Operand(1, 8, F16), y=Operand(4, 8, I8), residual=Operand(4, 8, F16), sum_out=Operand(4, 8, F16), y_scales=Operand(1, 4, F32))
    with pytest.raises(hip.HipError):                      # as it is it gets as far as the library, which has no device
        hip.rmsnorm(**dict(a, y_scales=Operand(4, 1, F32), x=Operand(4, 8, F16, 7)))
    with pytest.raises(AssertionError):
        hip.rmsnorm(**dict(a, **change))


@pytest.mark.parametrize("x_scales", [None, Operand(1, 3, F32), Operand(4, 1, F32, 3), Operand(1, 4, F16)])
def test_the_view_of_the_product_checks_its_factors(x_scales):
    q = Operand(6, 8, np.uint8)
    q.group, q.parts = 64, lambda: (P(1 << 20), P(1 << 20), None)
    with pytest.raises(AssertionError):
        hip.gemm_q4(Operand(4, 8, I8), q, Operand(4, 6, F16), x_scales=x_scales)
    with pytest.raises(hip.HipError):                      # (a pitch below the columns: refused by the library)
        hip.gemm_q4(Operand(4, 8, I8), q, Operand(4, 6, F16, 5), x_scales=Operand(4, 1, F32))


def test_sizes_are_known_beforehand():
    """What decx_hip_gemm_q4_fits, the workspace's and the scales' sizes say of products and matrices that are refused."""
    L = hip.lib()
    for M, N, K, group in ((1, (1 << 25) + 1, 128, 64), (1 << 31, 1 << 20, 128, 64), (0xffffffff, 0xffffff00, 128, 64), (0xffffffff, 1, 128, 64), (1 << 29, 128, 4096, 64),
                           (4, 20, 0xffffff80, 64), (4, 20, 130, 48), (4, 960, 1118481 * 128 + 1, 64)):
        assert L.decx_hip_gemm_q4_fits(M, N, K, group) == 0 and L.decx_hip_gemm_q4_workspace(0, M, N, K, group) == 0, (M, N, K, group)
    for M, N, K, group in ((1, 1 << 25, 128, 64), (0, 5, 0, 32), ((1 << 29) - 65, 100, 300, 128), (65, 300, 4100, 128)):
        assert L.decx_hip_gemm_q4_fits(M, N, K, group) == 1
    assert L.decx_hip_gemm_q4_workspace(0, 65, 300, 4100, 128) > 0
    assert L.decx_hip_q4_scales_count(960, 1118481 * 128, 32) == ((1 << 26) - 4) * 64 and L.decx_hip_q4_scales_count(960, 1118481 * 128 + 1, 32) == 0
    assert L.decx_hip_q4_scales_count(0xffffff01, 128, 64) == 0
