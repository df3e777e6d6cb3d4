"""An allocation that the device has no room for is reported by the call that asked for it, and by no later one."""
import ctypes

import numpy as np
import pytest

from decx_amd import hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["decx_hip_malloc", "decx_hip_host_malloc"])
def test_calls_behind_a_failed_allocation(what):
    hip.init()
    L, p = hip.lib(), ctypes.c_void_p()
    rng = np.random.default_rng(1)
    x, w = rng.standard_normal((3, 64)).astype(np.float16), rng.standard_normal((20, 64)).astype(np.float16)
    dx, dw, row = hip.DeviceMatrix(3, 64, np.float16, data=x), hip.DeviceMatrix(20, 64, np.float16, data=w), hip.DeviceMatrix(1, 64, np.float16, data=np.ones((1, 64)))
    q, y, n, d = hip.Q4Matrix(20, 64, 64), hip.DeviceMatrix(3, 20, np.float16), hip.DeviceMatrix(3, 64, np.float16), hip.DeviceMatrix(3, 3, np.float16)
    calls = [lambda: hip.quantize_q4(dw, q), lambda: hip.gemm_q4(dx, q, y), lambda: hip.dequantize_q4(q, dw), lambda: hip.rmsnorm(dx, row, n),
             lambda: hip.gemm(dx, hip.DeviceMatrix(64, 3, np.float16, data=w[:3].T), d)]
    for call in calls:
        call()
        hip.sync()
        assert getattr(L, what)(ctypes.byref(p), 1 << 50) > 0          # a positive code: HIP's own error
        call()                                                         # (raises where the launch reports another call's error)
        hip.sync()
