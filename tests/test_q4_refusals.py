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
