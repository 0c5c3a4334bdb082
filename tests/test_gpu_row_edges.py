"""Row collectives at the edges of their contract."""
import pytest

import roc_shmem_amd as rs
from helpers import runtime
from test_gpu_norm_to_all import Case as NormCase
from test_gpu_norm_to_all import run_backward, run_forward

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])


@BOTH
@pytest.mark.parametrize("rows,cols,rows_per_gate", [(100, 72, 1), (100, 72, 10), (100, 72, 99), (100, 72, 100), (100, 72, 1000),
                                                     (37, 1031, 5), (2100, 1100, 1), (2100, 1100, 700), (2100, 1100, 2101)])
def test_rows_per_gate_means_nothing_without_a_gate(dtype, rows, cols, rows_per_gate):
    """Every row has its gradient and counts in the weights' sums, whether a unit walks one row or several."""
    for replicated in (False, True):
        with runtime(2, heap_size=256 << 20):
            c = NormCase(dtype, rows, cols, 2, gate=0, replicated=replicated, seed=rows_per_gate)
            c.fields["rows_per_gate"] = rows_per_gate
            run_forward(c)
            run_backward(c)


def refused(call, args, word):
    with pytest.raises(rs.RocShmemError, match=word):
        call(args)


@pytest.mark.parametrize("replicated", [False, True])
def test_a_result_takes_no_other_results_place(replicated):
    """Only `normed` may be `source` and only `grad_residual` may be `grad_residual_out`, also where a call
    has neither: rows are read and written by workgroups of their own."""
    with runtime(4):
        c = NormCase(rs.FLOAT, 64, 512, 4, gate=0, pre_w=False, post=False, replicated=replicated)
        source, x, out = c.rows_of(64, 512, 0), c.stream(), c.stream()
        fields = dict(c.fields, source=source, residual=x)
        refused(rs.roc_shmem_norm_to_all, rs.NormArgs(residual_out=source, **fields), "residual_out and source overlap")
        rs.roc_shmem_norm_to_all(rs.NormArgs(residual_out=x, **fields))
        grads = dict(c.fields, grad_residual_out=out)
        wide = c.rows_of(64, 512, 0)
        refused(rs.roc_shmem_norm_to_all_grad, rs.NormGradArgs(grad_source=wide, **{**grads, "grad_residual_out": wide}),
                "grad_source and grad_residual_out overlap")
        rs.roc_shmem_norm_to_all_grad(rs.NormGradArgs(grad_source=wide, grad_residual=out, **grads))
        rs.synchronize()


@pytest.mark.parametrize("replicated", [False, True])
def test_in_place_of_one_operand_is_not_in_place_of_two(replicated):
    """One array may be read as two operands, and a result may replace either where nothing else reads its
    array: the other operand's rows are read by other workgroups, at other places."""
    with runtime(4):
        c = NormCase(rs.FLOAT, 64, 512, 4, gate=0, pre_w=False, post=False, replicated=replicated)
        both, out, h = c.rows_of(64, 512, 0), c.stream(), c.rows_of(64, 512, 0)
        fields = dict(c.fields, source=both, residual=both)
        refused(rs.roc_shmem_norm_to_all, rs.NormArgs(residual_out=both, normed=h, **fields), "residual_out and source overlap")
        refused(rs.roc_shmem_norm_to_all, rs.NormArgs(residual_out=out, normed=both, **fields), "normed and residual overlap")
        rs.roc_shmem_norm_to_all(rs.NormArgs(residual_out=out, normed=h, **fields))
        grads = dict(c.fields, grad_normed=both, grad_residual_out=both, residual_out=out)
        refused(rs.roc_shmem_norm_to_all_grad, rs.NormGradArgs(grad_source=both, grad_residual=c.stream(), **grads),
                "grad_source and grad_residual_out overlap")
        refused(rs.roc_shmem_norm_to_all_grad, rs.NormGradArgs(grad_source=h, grad_residual=both, **grads),
                "grad_residual and grad_normed overlap")
        rs.roc_shmem_norm_to_all_grad(rs.NormGradArgs(grad_source=h, grad_residual=c.stream(), **grads))
        rs.synchronize()
