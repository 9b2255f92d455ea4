"""The C++ shims of the paged KV4 cache: a host program is compiled against the header and the CUDA library; its rejection
cases run here without a GPU, its two steps of three requests on the GPU."""
import os
import subprocess

import pytest

from fnfl_v100_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "cpp", "paged_shim_test.cpp")
EXE = os.path.join(ROOT, "tests", "cpp", "paged_shim_test.bin")


@pytest.fixture(scope="module")
def exe():
    build.build()
    cuda, pkg = os.environ.get("CUDA_HOME", "/usr/local/cuda"), os.path.join(ROOT, "fnfl_v100_b200")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(cuda, "include"), SRC, "-o", EXE,
           "-L" + pkg, "-l:libfnb200.so", "-L" + os.path.join(cuda, "lib64"), "-lcudart", "-Wl,-rpath," + pkg,
           "-Wl,-rpath," + os.path.join(cuda, "lib64")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return EXE


def test_shims_compile_and_reject_bad_arguments(exe):
    r = subprocess.run([exe, "--reject"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.gpu
def test_two_steps_of_three_requests(exe):
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
