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


def test_storage_of_objects_that_are_made_anew(tmp_path):
    """re_construct of the classes behind de::Matrix and its kin (CPU: tests/cpp/object_storage_test.cpp, compiled with them)."""
    host, lib = os.path.join(ROOT, "decx_amd", "host"), os.path.join(ROOT, "decx_amd", "lib")
    exe = str(tmp_path / "object_storage_test")
    subprocess.run(["g++", "-O0", "-std=c++17", "-Wall", "-pthread", "-I" + os.path.join(ROOT, "include"), "-I" + host, os.path.join(ROOT, "tests", "cpp", "object_storage_test.cpp")] +
                   [os.path.join(host, f) for f in ("decx_host.cpp", "decx_vector.cpp")] +
                   ["-o", exe, "-L" + lib, "-ldecx_hip", "-Wl,-rpath," + lib], check=True, timeout=300)
    done = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0, done.stdout


@pytest.mark.gpu
def test_outputs_that_were_given_another_type():
    run("outputs_of_another_type")


@pytest.mark.gpu
def test_inputs_that_were_given_another_type():
    run("inputs_of_another_type")
