"""The row collectives' check of operands against each other, on addresses alone."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


def test_operands_may_be_one_array_only_where_the_call_says_so(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not found")
    program, package = str(tmp_path / "row_operands"), os.path.join(ROOT, "roc_shmem_amd")
    build = [HIPCC, "-std=c++17", "-O1", "-DROCSHMEM_NO_MPI", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"),
             "-I", os.path.join(package, "csrc"), os.path.join(ROOT, "tests", "cxx", "row_operands.cpp"), "-o", program,
             "-L", package, "-lrocshmem_mi355x", "-Wl,-rpath," + package]
    made = subprocess.run(build, capture_output=True, text=True, timeout=300)
    assert made.returncode == 0, made.stderr
    ran = subprocess.run([program], capture_output=True, text=True, timeout=60)
    assert ran.stdout == "ok\n" and ran.returncode == 0, ran.stdout + ran.stderr
