"""Calls of the 4-bit layer that are refused, and their neighbours that are not (no GPU: refusals come before the library looks
for one, and the others end with "not initialised" in a process of their own)."""
import ctypes
import subprocess
import sys

import pytest

from decx_amd import hip

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
