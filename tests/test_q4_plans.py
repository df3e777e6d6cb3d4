"""Which kernel the planner gives a product with 4-bit weights (no GPU: the plan is worked out on the host)."""
import ctypes

import pytest

from decx_amd import hip

BAD = -1
ROWS_16_NARROW, ROWS_16, ROWS_16_WIDE, ROWS_32_NARROW, ROWS_32, ROWS_64_NARROW, ROWS_64, TILES_64x128, TILES_64x256, TILES_128x384 = range(10)
LARGE = 256 << 20


def pick(i8, M, N, K, group=128, workspace=0):
    p = hip.plan_q4(i8, M, N, K, group, workspace)
    kt = -(-K // 128)
    assert 1 <= p.k_splits <= 8 and (p.split_tiles == kt if p.k_splits == 1 else p.split_tiles >= 2 and -(-kt // p.split_tiles) == p.k_splits)
    return p.kernel, p.k_splits


@pytest.mark.parametrize("i8", [False, True])
def test_every_kernel_serves_some_product(i8):
    """The shapes of use that the planner separates: a change of it that leaves a kernel without work shows here."""
    assert pick(i8, 1, 4096, 4096) == (ROWS_16_NARROW, 1)
    assert pick(i8, 7, 5003, 7001, 64) == (ROWS_16, 1)
    assert pick(i8, 16, 8192, 8192) == (ROWS_16_WIDE, 1)
    assert pick(i8, 20, 2048, 1024) == (ROWS_32_NARROW, 1)
    assert pick(i8, 32, 8192, 8192) == (ROWS_32, 1)
    assert pick(i8, 60, 4096, 4096) == (ROWS_64_NARROW, 1)
    assert pick(i8, 60, 8192, 4096) == (ROWS_64, 1)
    assert pick(i8, 1000, 4096, 8192, 64) == (TILES_64x128, 1)
    assert pick(i8, 2048, 4096, 4096) == (TILES_64x256, 1)
    assert pick(i8, 4096, 8192, 8192) == (TILES_128x384, 1)
    kernel, splits = pick(i8, 128, 8192, 8192, workspace=LARGE)
    assert kernel == TILES_64x128 and splits > 1


def test_ranges_want_their_room():
    for i8 in (False, True):
        need = hip.lib().decx_hip_gemm_q4_workspace(1 if i8 else 0, 128, 8192, 8192, 128)
        assert pick(i8, 128, 8192, 8192, workspace=need) == pick(i8, 128, 8192, 8192, workspace=LARGE)
        assert pick(i8, 128, 8192, 8192, workspace=need - 1)[1] < pick(i8, 128, 8192, 8192, workspace=need)[1]
        assert pick(i8, 128, 8192, 8192)[1] == 1


def test_what_has_no_plan():
    L, out = hip.lib(), hip.Q4Plan()
    for M, N, K, group in ((0, 5, 5, 64), (5, 0, 5, 64), (5, 5, 5, 48), (5, (1 << 25) + 1, 5, 64), (1 << 31, 1 << 20, 5, 64)):
        assert L.decx_hip_gemm_q4_plan(0, M, N, K, group, 0, ctypes.byref(out)) == BAD
    assert L.decx_hip_gemm_q4_plan(0, 5, 5, 5, 64, 0, None) == BAD


@pytest.mark.parametrize("M,plan", [(17, (0, 1, 4)), (16, (3, 1, 4)), (16, (7, 1, 4)), (33, (3, 1, 4)), (32, (5, 1, 4)), (40, (10, 1, 4)), (40, (-1, 1, 4)), (40, (7, 0, 4)),
                                    (40, (7, 1, 3)), (40, (5, 2, 2)), (40, (7, 4, 1)), (40, (7, 3, 2)), (40, (7, 2, 2))])
def test_plans_that_the_planner_could_not_give_are_refused(M, plan):
    """(the last one for its room alone; checked before the library looks for a GPU)"""
    P, p = ctypes.c_void_p, hip.Q4Plan(*plan)
    rest = (P(32), P(32), None, None, P(32), M, 20, 500, 64, 500, 0, 20, 1.0, 1.0, 0, P(64), 2 * M * 20 * 4 - 1, None)
    for xs in (None, P(32)):
        assert hip.lib().decx_hip_gemm_q4_forced_plan(ctypes.byref(p), P(32), xs, *rest) == BAD
    assert hip.lib().decx_hip_gemm_q4_forced_plan(None, P(32), None, *rest) == BAD


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("M,N,K", [(5000000, 16, 512), (1 << 28, 16, 300), (1 << 28, 32, 1000), (65535 * 64, 16, 512), (65535 * 64 + 1, 16, 512)])
def test_many_rows_and_few_columns_fit_their_grid(i8, M, N, K):
    """64 rows a workgroup in y, of which a grid has at most 65535; fewer than 2^32 threads a launch."""
    p = hip.plan_q4(i8, M, N, K, 128)
    if p.kernel in (ROWS_64_NARROW, ROWS_64):
        assert p.launch_rows == min(M, 65535 * 64)
        assert 512 * -(-N // 16) * -(-p.launch_rows // 64) < 1 << 32
    else:
        assert p.kernel >= TILES_64x128 and p.launch_rows == M
    assert hip.plan_q4(i8, 5000000, 16, 512, 128).kernel == ROWS_64_NARROW          # (so the first of them is one that the rule is there for)
    assert hip.plan_q4(i8, 60, 8192, 4096, 128).launch_rows == 60
