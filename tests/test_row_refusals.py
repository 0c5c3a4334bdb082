"""Arguments that the row collectives refuse whatever the state of the runtime: every call says why and
returns without touching the GPU, so this runs without one."""
import ctypes as C

import pytest

import roc_shmem_amd as rs
from roc_shmem_amd import _lib

NORM = dict(dtype=rs.FLOAT, team=1, rows=4, cols=8, source=128, residual=128, residual_out=128, normed=128)
GRAD = dict(dtype=rs.FLOAT, team=1, rows=4, cols=8, grad_normed=128, residual_out=128, grad_source=128, grad_residual=128)
LOGPROB = dict(dtype=rs.FLOAT, team=1, rows=4, vocab=8, logits=128, tokens=128, logprob=128)
LOGPROB_GRAD = dict(dtype=rs.FLOAT, team=1, rows=4, vocab=8, logits=128, tokens=128, lse=128, entropy=128, grad_logprob=128, grad_logits=128)

REFUSED = [
    (rs.roc_shmem_norm_to_all, rs.NormArgs, NORM, [
        (dict(dtype=rs.DOUBLE), "dtype"), (dict(dtype=-1), "dtype"), (dict(flags=4), "flags"), (dict(cols=0), "cols"),
        (dict(cols=16385), "cols"), (dict(rows=1 << 22), "rows"), (dict(source_ld=7), "stride"), (dict(normed_ld=7), "stride"),
        (dict(residual_ld=7), "stride"), (dict(source_ld=1 << 60), "stride"), (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=1e-40), "eps"),
        (dict(eps=float("nan")), "eps"), (dict(residual_scale=float("inf")), "finite"), (dict(block_scale=float("nan")), "finite"),
        (dict(weight_offset=float("inf")), "finite"), (dict(post_weight=128), "post_weight"), (dict(source=None), "source"),
        (dict(residual=None), "residual"), (dict(residual_out=None), "residual_out"),
        (dict(normed=None, pre_weight=128), "pre_weight")]),
    (rs.roc_shmem_norm_to_all_grad, rs.NormGradArgs, GRAD, [
        (dict(dtype=rs.SHORT), "dtype"), (dict(cols=20000), "cols"), (dict(eps=0.0), "eps"), (dict(grad_source=None), "grad_source"),
        (dict(grad_normed=None), "neither"), (dict(residual_out=None), "residual_out"), (dict(flags=rs.NORM_POST), "total"),
        (dict(gate=128, grad_gate=128), "total"), (dict(grad_gate=128, total=128), "gate"), (dict(grad_post_weight=128), "RSM_NORM_POST"),
        (dict(grad_normed=None, grad_residual_out=128, grad_pre_weight=128), "grad_pre_weight")]),
    (rs.roc_shmem_norm_grad_work_bytes, rs.NormGradArgs, GRAD, [(dict(dtype=rs.INT), "dtype"), (dict(cols=0), "cols")]),
    (rs.roc_shmem_logprob_to_all, rs.LogprobArgs, LOGPROB, [
        (dict(dtype=rs.LONG), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 30), "vocab"), (dict(rows=1 << 22), "rows"),
        (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
        (dict(scale=3e38), "scale"), (dict(scale=1e-40), "scale"),
        (dict(logits=None), "logits"), (dict(tokens=None), "tokens"), (dict(logprob=None), "no result"), (dict(top_k=3), "top_k"),
        (dict(top_ids=128), "top_k"), (dict(top_k=33, top_ids=128, vocab=100), "top_k"), (dict(top_k=9, top_ids=128), "top_k"),
        (dict(top_k=-1, top_ids=128), "top_k")]),
    (rs.roc_shmem_logprob_work_bytes, rs.LogprobArgs, LOGPROB, [(dict(vocab=0), "vocab"), (dict(top_k=33), "top_k")]),
    (rs.roc_shmem_logprob_to_all_grad, rs.LogprobGradArgs, LOGPROB_GRAD, [
        (dict(dtype=rs.LONGLONG), "dtype"), (dict(vocab=0), "vocab"), (dict(scale=0.0), "scale"), (dict(logits=None), "logits"),
        (dict(lse=None), "lse"), (dict(grad_logits=None), "grad_logits"), (dict(grad_logprob=None), "no gradient"),
        (dict(tokens=None), "tokens"), (dict(grad_entropy=128, entropy=None), "entropy")]),
]


@pytest.mark.parametrize("call,args,good,changes", REFUSED, ids=[c[0].__name__ for c in REFUSED])
def test_refusals_name_the_argument(call, args, good, changes):
    for change, word in changes:
        with pytest.raises(rs.RocShmemError, match=word):
            call(args(**{**good, **change}))


@pytest.mark.parametrize("call,args,good,changes", REFUSED, ids=[c[0].__name__ for c in REFUSED])
def test_good_arguments_get_as_far_as_the_runtime(call, args, good, changes):
    assert not _lib.load().rsm_is_initialized()
    with pytest.raises(rs.RocShmemError, match="rsm_init"):
        call(args(**good))


def test_null_arguments():
    lib = _lib.load()
    n = C.c_size_t(7)
    for name in ("rsm_norm_to_all", "rsm_norm_to_all_grad", "rsm_logprob_to_all", "rsm_logprob_to_all_grad"):
        assert getattr(lib, name)(None, None) != 0 and b"NULL" in lib.rsm_last_error()
    for name, args in (("rsm_norm_grad_work_bytes", rs.NormGradArgs(**GRAD)), ("rsm_logprob_work_bytes", rs.LogprobArgs(**LOGPROB))):
        assert getattr(lib, name)(None, C.byref(n)) != 0 and getattr(lib, name)(args, None) != 0
    assert n.value == 7


def test_argument_structures_know_their_fields():
    with pytest.raises(TypeError):
        rs.NormArgs(sauce=128)
    a = rs.LogprobArgs(rows=3)
    with pytest.raises(AttributeError):
        a.colour = 1
    assert a.scale == 1.0 and a.rows == 3 and a.logits is None

    class Array:
        addr = 4096
    assert rs.NormArgs(source=Array()).source == 4096
