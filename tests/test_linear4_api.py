"""The C++ API of the 4-bit layer (include/DECX.h), driven through tests/cpp/linear4_test."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "linear4_test")


def run(mode):
    assert os.path.exists(EXE), "tests/cpp/linear4_test missing: run `python -m decx_amd.build`"
    done = subprocess.run([EXE, mode], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0, done.stdout


def test_calls_are_refused_without_a_gpu():
    run("host")


def test_entry_points_are_exported():
    lib = os.path.join(ROOT, "decx_amd", "lib", "libDECX_BLAS_HIP.so")
    syms = subprocess.run(["nm", "-D", "-C", "--defined-only", lib], stdout=subprocess.PIPE, text=True).stdout
    for needle in ["de::CreateGPUMatrix4Ref()", "de::nn::cuda::Quantize4(de::GPU_Matrix&, de::GPU_Matrix4&, unsigned int, bool)",
                   "de::nn::cuda::Linear4(de::GPU_Matrix&, de::GPU_Matrix4&, de::GPU_Matrix&, unsigned int)",
                   "de::nn::cuda::Linear4(de::GPU_Matrix&, de::GPU_Vector&, de::GPU_Matrix4&, de::GPU_Matrix&, de::GPU_Matrix&, de::Number, de::Number)",
                   "de::nn::cuda::RMSNorm(de::GPU_Matrix&, de::GPU_Matrix&, de::GPU_Vector&, de::GPU_Matrix&, de::GPU_Matrix&, de::GPU_Vector&, float)"]:
        assert needle in syms, needle


@pytest.mark.gpu
def test_a_layer_through_the_objects():
    run("gpu")
