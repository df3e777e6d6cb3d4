"""The C++ API of the 4-bit layer at the edges of what its objects may be, through tests/cpp/linear4_edges_test."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "linear4_edges_test")


def run(check):
    assert os.path.exists(EXE), "tests/cpp/linear4_edges_test missing: run `python -m decx_amd.build`"
    done = subprocess.run([EXE, check], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0, done.stdout


@pytest.mark.gpu
def test_the_norm_of_a_sum_may_lie_where_the_sum_does():
    run("dst_is_the_sum")


@pytest.mark.gpu
def test_sizes_that_are_refused_leave_the_outputs_as_they_were():
    run("sizes_that_are_refused")
