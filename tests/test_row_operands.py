"""What the row collectives refuse of operands that do not go together, without a GPU."""
import os
import subprocess

import pytest

import roc_shmem_amd as rs

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


def test_the_parts_of_a_normaliser_go_together():
    good = dict(dtype=rs.FLOAT, team=1, rows=4, vocab=8, logits=128, grad_lse=128, grad_logits=128)
    for change, word in [(dict(), "lse"), (dict(largest=128), "largest"), (dict(log_sum=128), "largest"), (dict(lse=128, log_sum=128), "largest"),
                         (dict(lse=128, largest=128), "log_sum"), (dict(lse=128), "rsm_init"), (dict(largest=128, log_sum=128), "rsm_init"),
                         (dict(lse=128, largest=128, log_sum=128), "rsm_init")]:
        with pytest.raises(rs.RocShmemError, match=word):
            rs.roc_shmem_logprob_to_all_grad(rs.LogprobGradArgs(**good, **change))
