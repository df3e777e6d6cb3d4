"""Register budgets of the 4-bit layer's kernels (CPU only: hipcc's own resource report for gfx950, nothing runs): no spills
anywhere, and the wavefronts per SIMD that each schedule is built on."""
import pytest

from test_kernel_resources import resource_report


@pytest.mark.timeout(600)
def test_products_with_4_bit_weights(tmp_path):
    r = resource_report("gemm_q4.hip", tmp_path)
    rows = {k: v for k, v in r.items() if "gemm_q4_rows_kernel" in k}
    tiles = {k: v for k, v in r.items() if "gemm_q4_tiles_kernel" in k}
    assert len(rows) == 6 * (10 + 13) and len(tiles) == 12 * 3                # 2 types of X, 3 groups, with and without zero points
    for k, (waves, scratch) in r.items():
        assert scratch == 0, k
    for k, (waves, _) in rows.items():
        assert waves >= (4 if "ELi1ELi1ELi16E" in k or "ELi1ELi2ELi16E" in k or "ELi1ELi2ELi8E" in k else 2), k
    for k, (waves, _) in tiles.items():
        assert waves >= (3 if "ELi4ELi2ELi1ELi4E" in k else 2), k             # 64 x 128: three workgroups of 4 wavefronts per CU


@pytest.mark.timeout(600)
def test_quantisation_and_norm(tmp_path):
    for source, kernels in (("q4_pack.hip", 18), ("rmsnorm.hip", 24)):
        r = resource_report(source, tmp_path)
        assert len(r) == kernels, source
        for k, (waves, scratch) in r.items():
            assert scratch == 0 and waves >= 5, (k, waves, scratch)
