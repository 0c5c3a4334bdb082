"""Row collectives at the edges of their contract."""
import numpy as np
import pytest

import roc_shmem_amd as rs
import row_reference as ref
from helpers import runtime
from row_arrays import Rows
from test_gpu_logprob_to_all import NP
from test_gpu_logprob_to_all import Case as LogprobCase
from test_gpu_norm_to_all import A, run_backward, run_forward
from test_gpu_norm_to_all import Case as NormCase

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


# Columns of an infinity: the first, the last, and those that the last two vectors of a row both hold.
ENDS = [(128, (0, 60, 127)), (131, (0, 125, 127, 128, 130)), (1030, (3, 1021, 1022, 1023, 1026, 1029)), (2051, (7, 2043, 2047, 2048, 2050))]


@BOTH
@pytest.mark.parametrize("cols,at", ENDS)
def test_an_infinity_reaches_as_far_in_every_width(dtype, cols, at):
    """A row with an infinite element has an infinite mean of squares, so r = 0: the rest of its normed row
    is 0 and the element itself inf * 0.  The residual stream holds the infinity and its neighbours."""
    with runtime(2):
        c = NormCase(dtype, len(at), cols, 2, gate=0, post=False, replicated=True)
        x, parts = c.numbers(len(at), cols), [c.numbers(len(at), cols) for _ in range(2)]
        for row, col in enumerate(at):
            x[row, col] = ref.to_type(dtype, [-np.inf if row % 2 else np.inf])[0]
        source, h = c.rows_of(len(at), cols, 0).write_all(parts), c.rows_of(len(at), cols, 0)
        out, res = c.stream(), c.stream(x)
        rs.roc_shmem_norm_to_all(rs.NormArgs(source=source, residual=res, residual_out=out, normed=h, **c.fields))
        rs.synchronize()
        got, stream = ref.from_type(dtype, h.read(1)), ref.from_type(dtype, out.read(1))
        hit = np.arange(cols)[None, :] == np.asarray(at)[:, None]
        assert np.array_equal(np.isnan(got), hit)
        assert not got[~hit].any()
        assert np.array_equal(np.isinf(stream), hit) and not np.isnan(stream).any()


@BOTH
@pytest.mark.parametrize("cols,at", ENDS)
def test_an_infinite_sum_reaches_as_far_in_every_width(dtype, cols, at):
    """The same of the members' sum and the norm behind it: z = s r(s) is 0 but for inf * 0, so the residual
    stream keeps its other elements."""
    with runtime(2):
        c = NormCase(dtype, len(at), cols, 2, gate=0, replicated=True)
        x, parts = c.numbers(len(at), cols), [c.numbers(len(at), cols) for _ in range(2)]
        for row, col in enumerate(at):
            parts[1][row, col] = ref.to_type(dtype, [np.inf])[0]
        source, out = c.rows_of(len(at), cols, 0).write_all(parts), c.stream()
        fields = {k: v for k, v in c.fields.items() if k != "pre_weight"}
        rs.roc_shmem_norm_to_all(rs.NormArgs(source=source, residual=c.stream(x), residual_out=out, **fields))
        rs.synchronize()
        got, hit = ref.from_type(dtype, out.read(0)), np.arange(cols)[None, :] == np.asarray(at)[:, None]
        assert np.array_equal(np.isnan(got), hit)
        want = A * ref.from_type(dtype, x)        # one product, exact, rounded once
        assert (np.abs(got - want)[~hit] <= ref.HALF_STEP[dtype] * np.abs(want)[~hit]).all()


@BOTH
@pytest.mark.parametrize("cols,at", ENDS)
def test_an_infinite_gradient_reaches_as_far_in_every_width(dtype, cols, at):
    """mean(t n) is infinite where t is, so D = -n times it: infinite throughout, and NaN only at the element
    itself where inf - inf meet."""
    with runtime(2):
        c = NormCase(dtype, len(at), cols, 2, gate=0, post=False, pre_w=False, replicated=True)
        x = c.numbers(len(at), cols)
        x[:] = ref.to_type(dtype, np.where(c.rng.random(x.shape) < 0.5, -1.0, 1.0) * (0.5 + c.rng.random(x.shape)))
        parts = [c.numbers(len(at), cols) for _ in range(2)]
        for row, col in enumerate(at):
            parts[0][row, col] = ref.to_type(dtype, [np.inf])[0]
        gn, gs, gr = c.rows_of(len(at), cols, 0).write_all(parts), c.rows_of(len(at), cols, 0), c.stream()
        rs.roc_shmem_norm_to_all_grad(rs.NormGradArgs(grad_normed=gn, residual_out=c.stream(x), grad_source=gs, grad_residual=gr, **c.fields))
        rs.synchronize()
        hit = np.arange(cols)[None, :] == np.asarray(at)[:, None]
        v = ref.from_type(dtype, x)
        sign = -np.sign(v) * np.sign((v * hit).sum(1, keepdims=True))
        for got in (ref.from_type(dtype, gs.read(1)), ref.from_type(dtype, gr.read(0))):
            assert np.array_equal(np.isnan(got), hit)
            assert np.array_equal(got[~hit], (sign * np.inf)[~hit])


def rows_of_large_normalisers(rng, dtype, rows, vocab):
    """Logits of 64 bits, rounded to the type, whose normalisers lose digits or all of them as floats."""
    lowest = -3.3895314e38
    base = rng.standard_normal((rows, vocab)) * 2
    kinds = [np.full((rows, vocab), lowest), np.where(np.arange(vocab) % 7 == 3, lowest / 2, lowest), np.full((rows, vocab), -lowest),
             np.where(rng.random((rows, vocab)) < 0.5, lowest, base), base - 3000, np.full((rows, vocab), -np.inf), base,
             np.round(base) + 1e6 if dtype == rs.FLOAT else np.round(base) * 32 + 4096]
    logits = np.empty((rows, vocab))
    for row in range(rows):
        logits[row] = kinds[row % len(kinds)][row]
    return ref.to_type(dtype, logits)


@BOTH
@pytest.mark.parametrize("rows,vocab,scale", [(8, 3000, 1.0), (8, 40000, 1.0), (9, 40000, 2.5), (300, 3000, 0.75), (264, 9001, 1.0)])
def test_gradients_where_the_normaliser_is_large(dtype, rows, vocab, scale):
    """From largest and log_sum the gradient has the forward pass's probabilities, also in rows that are all
    the type's lowest or highest value, or whose scaled normaliser is no float at all."""
    rng = np.random.default_rng(rows + vocab)
    with runtime(3, heap_size=256 << 20):
        c = LogprobCase(dtype, rows, vocab, 3, logits=ref.from_type(dtype, rows_of_large_normalisers(rng, dtype, rows, vocab)),
                        scale=scale, tokens=rng.integers(-1, vocab, rows))
        out = {n: Rows(1, rows, np.float32) for n in ("logprob", "entropy", "largest", "log_sum")}
        for a in out.values():
            a.remember()
        rs.roc_shmem_logprob_to_all(c.call(out))
        rs.synchronize()
        got = {n: a.read(2)[0] for n, a in out.items()}
        for n, a in out.items():
            for pe in range(3):
                assert np.array_equal(a.read(pe)[0], got[n], equal_nan=True)
                a.check_rest(pe, n, 1)
        x = c.f64()
        m = x.max(1)
        empty = m == -np.inf
        assert np.array_equal(got["largest"], m.astype(np.float32))
        # the formulas on logits whose largest is 0: the same rows with a normaliser of ln l
        below = x - np.where(empty, 0, m)[:, None]
        want = ref.logprob_forward(below, c.tokens, c.scale, 0)
        for n, of in (("log_sum", "lse"), ("entropy", "entropy"), ("logprob", "logprob")):
            ref.check(n, rs.FLOAT, got[n], *want[of])
        g = {n: rng.standard_normal(rows).astype(np.float32) for n in ("grad_logprob", "grad_entropy", "grad_lse")}
        value, error = ref.logprob_backward(below, c.tokens, got["log_sum"], got["entropy"], c.scale, *g.values())
        for in_place in (False, True):
            d = c.array if in_place else Rows(rows, c.width, NP[dtype], c.ld)
            fields = dict(entropy=out["entropy"], largest=out["largest"], log_sum=out["log_sum"], grad_logits=d, grad_ld=d.ld)
            rs.roc_shmem_logprob_to_all_grad(rs.LogprobGradArgs(**fields, **{n: c.numbers(v, np.float32) for n, v in g.items()}, **c.fields))
            rs.synchronize()
            for pe in range(3):
                part = slice(pe * c.shard, min(vocab, (pe + 1) * c.shard))
                ref.check("grad_logits on PE %d" % pe, dtype, d.read(pe)[:, :part.stop - part.start], value[:, part], error[:, part])


def test_largest_and_log_sum_alone_and_where_rows_are_not_numbers():
    logits = np.random.default_rng(3).standard_normal((4, 5000)).astype(np.float32)
    logits[1, 77], logits[2, 4999] = np.nan, np.inf
    with runtime(2):
        c = LogprobCase(rs.FLOAT, 4, 5000, 2, logits=logits)
        m, s = Rows(1, 4, np.float32), Rows(1, 4, np.float32)
        rs.roc_shmem_logprob_to_all(c.call({"largest": m}))
        rs.roc_shmem_logprob_to_all(c.call({"log_sum": s}))
        d = Rows(4, c.width, np.float32, c.ld)
        rs.roc_shmem_logprob_to_all_grad(rs.LogprobGradArgs(largest=m, log_sum=s, grad_lse=c.numbers(np.ones(4), np.float32), grad_logits=d,
                                                            **c.fields))
        rs.synchronize()
        assert np.array_equal(np.isnan(s.read(1)[0]), [False, True, True, False])
        assert np.array_equal(m.read(1)[0][[0, 3]], logits[[0, 3]].max(1))
        got = d.read(0)
        assert np.isnan(got[1:3]).all() and np.isfinite(got[[0, 3]]).all()
