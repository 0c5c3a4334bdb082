"""The row collectives as a program runs them: refusals that need the heap, streams, graphs, and a
training step of a small model whose every operator is one of them or a product of matrices."""
import threading

import numpy as np
import pytest

import roc_shmem_amd as rs
import row_reference as ref
from helpers import runtime
from row_arrays import Rows
from test_gpu_logprob_to_all import Case as LogprobCase
from test_gpu_norm_to_all import Case as NormCase

pytestmark = pytest.mark.gpu


def refused(call, args, word):
    with pytest.raises(rs.RocShmemError, match=word):
        call(args)


def test_operands_that_do_not_fit_or_overlap_are_refused():
    with runtime(4):
        c = NormCase(rs.FLOAT, 64, 512, 4, gate=0)
        source, x = c.rows_of(64, 512, 0), c.stream()
        small, out, h = rs.sym_array(64, np.float32), c.stream(), c.rows_of(64, 512, 0)
        fields = dict(c.fields, source=source, residual=x, residual_out=out, normed=h)
        outside = rs.device_array(nbytes=1 << 20)
        for change, word in [(dict(source=small), "source"), (dict(normed=small), "normed"), (dict(residual=small), "residual"),
                             (dict(residual_out=small), "residual_out"), (dict(total=small), "total"),
                             (dict(post_weight=small), "post_weight"), (dict(gate=small), "gate"),
                             (dict(source_ld=1 << 20), "source"), (dict(normed=outside.addr), "symmetric"),
                             (dict(source=rs.roc_shmem_ptr(source.addr, 1)), "symmetric"), (dict(team=12345), "team"),
                             (dict(normed=x), "overlap|fit"), (dict(residual_out=source), "overlap|fit"), (dict(total=out), "overlap"),
                             (dict(normed=source, source_ld=512 + 3), "overlap|fit"), (dict(normed=source.addr + 16), "overlap|fit"),
                             (dict(source=source.addr + 2), "aligned|fit"), (dict(gate=source.addr + 1), "aligned"),
                             (dict(residual_out=c.weights and fields["pre_weight"].addr), "overlap|fit")]:
            refused(rs.roc_shmem_norm_to_all, rs.NormArgs(**{**fields, **change}), word)
        g = dict(c.fields, grad_normed=h, residual_out=x, total=c.shared(), grad_source=source, grad_residual=out,
                 grad_pre_weight=c.rows_of(1, 512, 0))
        refused(rs.roc_shmem_norm_to_all_grad, rs.NormGradArgs(**g), "work")
        refused(rs.roc_shmem_norm_to_all_grad, rs.NormGradArgs(work=small, **g), "work")
        refused(rs.roc_shmem_norm_to_all_grad, rs.NormGradArgs(work=source, **g), "overlap|fit")
        wide = rs.sym_array(1 << 22, np.uint8)
        refused(rs.roc_shmem_norm_to_all_grad, rs.NormGradArgs(work=wide.addr + 4, **g), "aligned")
        d = LogprobCase(rs.FLOAT, 8, 100000, 4, top_k=3)      # so few rows of so many share a workspace
        o = d.outputs()
        args = d.call(o)
        for change, word in [(dict(work=None), "work"), (dict(pSync=None), "pSync"), (dict(pSync=small), "pSync"),
                             (dict(logits_ld=1 << 22), "logits"), (dict(lse=o["entropy"]), "overlap"),
                             (dict(lse=d.array), "overlap|fit"), (dict(shard=200), "cover"), (dict(logits_ld=24999), "stride"),
                             (dict(team=0), "team"), (dict(tokens=outside.addr), "symmetric"),
                             (dict(tokens=d.token_array.addr + 4), "aligned"), (dict(pSync=wide.addr + 4), "aligned"),
                             (dict(lse=wide.addr + 2), "aligned")]:
            fields = dict(top_k=3, work=args.work, pSync=args.pSync, **{**d.fields, **o})
            refused(rs.roc_shmem_logprob_to_all, rs.LogprobArgs(**{**fields, **change}), word)
        lse = d.numbers(np.zeros(8), np.float32)
        fields = dict(lse=lse, grad_lse=lse, grad_logits=d.array, grad_ld=d.ld, **d.fields)
        rs.roc_shmem_logprob_to_all_grad(rs.LogprobGradArgs(**fields))
        refused(rs.roc_shmem_logprob_to_all_grad, rs.LogprobGradArgs(**{**fields, "grad_ld": d.ld + 1}), "overlap|fit")
        refused(rs.roc_shmem_logprob_to_all_grad, rs.LogprobGradArgs(**{**fields, "grad_ld": 10}), "stride")
        refused(rs.roc_shmem_logprob_to_all_grad, rs.LogprobGradArgs(**{**fields, "grad_lse": lse, "grad_logits": lse}), "overlap|fit")
        rs.synchronize()
        outside.free()


class Model:
    """One block and the head of a model on the members of a team, bfloat16 or float: the block is a
    product with each member's slice of a matrix, the head one with each member's part of the vocabulary."""

    def __init__(self, dtype, rows=24, cols=96, vocab=501, pes=4, seed=0):
        self.c = c = NormCase(dtype, rows, cols, pes, gate=1, replicated=True, seed=seed)
        self.dtype, self.pes, self.rows, self.cols, self.vocab = dtype, pes, rows, cols, vocab
        self.shard = -(-vocab // pes)
        self.np = np.uint16 if dtype == rs.BF16 else np.float32
        rng = c.rng
        self.head = rng.standard_normal((cols, vocab)) / 4
        self.tokens = rng.integers(0, vocab, rows)
        self.tokens[3:4] = -1
        new = lambda r, n, t=None: Rows(r, n, t or self.np)  # noqa: E731
        self.partials = [c.numbers(rows, cols) for _ in range(pes)]
        self.x = c.numbers(rows, cols)
        self.a = {"source": new(rows, cols), "residual": new(rows, cols), "residual_out": new(rows, cols), "normed": new(rows, cols),
                  "total": new(c.share, cols), "logits": new(rows, self.shard), "grad_logits": new(rows, self.shard),
                  "tokens": new(1, rows, np.int64), "grad_normed": new(rows, cols), "grad_source": new(rows, cols),
                  "grad_residual": new(rows, cols), "grad_residual_out": new(rows, cols)}
        for n in ("logprob", "entropy", "lse", "grad_logprob", "grad_entropy"):
            self.a[n] = new(1, rows, np.float32)
        for n in ("grad_pre_weight", "grad_post_weight", "grad_gate"):
            self.a[n] = new(1, cols, np.float32)
        a = self.a
        a["source"].write_all(self.partials)
        a["tokens"].write_all([self.tokens] * pes)
        self.scale_by = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32) * 0.1
        for pe in range(pes):
            a["residual"].write(pe, self.x)
            a["grad_residual_out"].write(pe, np.zeros((rows, cols), self.np))
            a["grad_logprob"].write(pe, self.scale_by[0])
            a["grad_entropy"].write(pe, self.scale_by[1])
        f, t = c.fields, c.team
        take = lambda names: {n: a[n] for n in names.split()}  # noqa: E731
        lp = dict(dtype=dtype, team=t, rows=rows, vocab=vocab, **take("logits tokens"))
        self.norm = rs.NormArgs(**take("source residual residual_out normed total"), **f)
        self.logprob = rs.LogprobArgs(**take("logprob entropy lse"), **lp)
        self.logprob_grad = rs.LogprobGradArgs(**take("lse entropy grad_logprob grad_entropy grad_logits"), **lp)
        self.norm_grad = rs.NormGradArgs(**take("grad_normed grad_residual_out residual_out total grad_source grad_residual "
                                                "grad_pre_weight grad_post_weight grad_gate"), **f)
        self.work = rs.sym_array(max(1, rs.roc_shmem_norm_grad_work_bytes(self.norm_grad)), np.uint8)
        self.lwork = rs.sym_array(max(1, rs.roc_shmem_logprob_work_bytes(self.logprob)), np.uint8)
        self.psync = rs.sym_array(rs.ROC_SHMEM_REDUCE_SYNC_SIZE, np.int64, fill=0)
        self.norm_grad.work, self.logprob.work, self.logprob.pSync = self.work.addr, self.lwork.addr, self.psync.addr

    def f(self, v):
        return ref.from_type(self.dtype, v)

    def head_forward(self):
        """Every member's logits from its own copy of the block's output."""
        for pe in range(self.pes):
            part = self.f(self.a["normed"].read(pe)) @ self.head[:, pe * self.shard:(pe + 1) * self.shard]
            whole = np.zeros((self.rows, self.shard))
            whole[:, :part.shape[1]] = part
            self.a["logits"].write(pe, ref.to_type(self.dtype, whole))

    def head_backward(self):
        """Every member's part of the gradient of the head's input."""
        for pe in range(self.pes):
            w = self.head[:, pe * self.shard:(pe + 1) * self.shard]
            g = self.f(self.a["grad_logits"].read(pe))[:, :w.shape[1]] @ w.T
            self.a["grad_normed"].write(pe, ref.to_type(self.dtype, g))


def loss_of(m, leaves):
    """sum g_logprob * logprob + g_entropy * entropy of the whole model, in 64 bits."""
    formula = {**m.c.formula(), **{k: leaves[k] for k in ("pre", "post", "gate")}}
    h = ref.norm_forward(leaves["partials"], leaves["residual"], **formula)["normed"][0]
    out = ref.logprob_forward(h @ m.head, m.tokens, 1.0, 0)
    return (m.scale_by[0].astype(float) * out["logprob"][0]).sum() + (m.scale_by[1].astype(float) * out["entropy"][0]).sum()


@pytest.mark.parametrize("dtype", [rs.FLOAT, rs.BF16])
def test_a_training_step(dtype):
    """Forward and backward through the four operators; gradients against differences of the whole
    model's loss along random directions."""
    with runtime(4):
        m = Model(dtype)
        rs.roc_shmem_norm_to_all(m.norm)
        rs.synchronize()
        m.head_forward()
        rs.roc_shmem_logprob_to_all(m.logprob)
        rs.roc_shmem_logprob_to_all_grad(m.logprob_grad)
        rs.synchronize()
        m.head_backward()
        rs.roc_shmem_norm_to_all_grad(m.norm_grad)
        rs.synchronize()
        assert not m.psync.read(0).any()
        formula = m.c.formula()
        leaves = {"partials": np.stack([m.f(v) for v in m.partials]), "residual": m.f(m.x), **{k: formula[k] for k in ("pre", "post", "gate")}}
        names = {"partials": "grad_source", "residual": "grad_residual", "pre": "grad_pre_weight", "post": "grad_post_weight", "gate": "grad_gate"}
        rng = np.random.default_rng(4)
        # Every tensor between the operators is rounded to the type: normed, logits, grad_logits,
        # grad_normed, the kept sum and the gradient itself.  A rounding is off by half a step of what
        # it rounds, independently from element to element, and each of the six can move every term of
        # the gradient: 6 half steps of the terms' magnitudes at most, and three such standard
        # deviations for sums of independent ones.
        for leaf, name in names.items():
            got = m.a[name].read(1)
            grad = m.f(got) if name in ("grad_source", "grad_residual") else got.astype(np.float64)
            value = leaves[leaf]
            direction = rng.standard_normal(value.shape)
            grad = grad.reshape(grad.shape if leaf in ("residual", "partials", "gate") else value.shape)
            d1, d2 = ((loss_of(m, {**leaves, leaf: value + s * direction}) - loss_of(m, {**leaves, leaf: value - s * direction})) / (2 * s)
                      for s in (1e-3, 5e-4))
            want = d2 + (d2 - d1) / 3
            terms = grad * direction
            bound = 6 * ref.HALF_STEP[dtype] * np.abs(terms).sum() if dtype == rs.BF16 else 2e-5 * np.abs(terms).sum()
            assert abs(terms.sum() - want) <= bound + 1e-8, (leaf, terms.sum(), want, bound)


def test_recorded_calls_replay_like_eager_ones():
    """The four operators recorded into a graph on a stream of their own; every replay, with new inputs
    and the program's own calls between, gives bit for bit what eager calls give."""
    with runtime(4):
        m = Model(rs.BF16)
        stream = rs.Stream()
        results = ("residual_out", "normed", "total", "logprob", "entropy", "lse", "grad_logits", "grad_source", "grad_residual",
                   "grad_pre_weight", "grad_post_weight", "grad_gate")

        def calls(on):
            rs.roc_shmem_norm_to_all(m.norm, on)
            rs.roc_shmem_logprob_to_all(m.logprob, on)
            rs.roc_shmem_logprob_to_all_grad(m.logprob_grad, on)
            rs.roc_shmem_norm_to_all_grad(m.norm_grad, on)

        with rs.Graph.capture(stream) as graph:
            calls(stream)
        rng = np.random.default_rng(6)
        for replay in range(4):
            for name in ("source", "logits", "grad_normed"):
                a = m.a[name]
                a.write_all([ref.to_type(rs.BF16, rng.standard_normal((a.rows, a.cols))) for _ in range(4)])
            rs.synchronize()
            got = []
            for way in ("replayed", "eager"):
                for n in results:
                    m.a[n].whole.fill(0x33)
                rs.synchronize()
                if way == "replayed":
                    graph.launch()
                else:
                    calls(None)
                stream.synchronize()
                rs.synchronize()
                got.append({n: [m.a[n].whole.read(p).tobytes() for p in range(4)] for n in results})
            assert got[0] == got[1], [n for n in results if got[0][n] != got[1][n]]
            assert not m.psync.read(0).any()
        graph.destroy()
        stream.destroy()


def test_two_streams_and_two_threads():
    """Calls with operands and workspaces of their own, on two streams from two host threads at once."""
    with runtime(4, heap_size=256 << 20):
        models = [Model(rs.FLOAT, rows=r, vocab=20001, seed=s) for s, r in enumerate((3, 40))]
        streams = [rs.Stream(), rs.Stream()]
        rng = np.random.default_rng(1)
        for m in models:
            m.a["logits"].write_all([rng.standard_normal((m.rows, m.shard)).astype(np.float32) for _ in range(4)])

        def go(k):
            for _ in range(50):
                rs.roc_shmem_norm_to_all(models[k].norm, streams[k])
                rs.roc_shmem_logprob_to_all(models[k].logprob, streams[k])

        names = ("normed", "residual_out", "total", "logprob", "entropy", "lse")
        read = lambda m: {n: [m.a[n].whole.read(p).tobytes() for p in range(4)] for n in names}  # noqa: E731
        want = []
        for k, m in enumerate(models):
            go(k)
            streams[k].synchronize()
            want.append(read(m))
            for n in names:
                m.a[n].whole.fill(0x44)
        rs.synchronize()
        threads = [threading.Thread(target=go, args=(k,)) for k in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for s in streams:
            s.synchronize()
        # the fill reached what the calls do not write, too: compare the rows alone
        for m, w in zip(models, want):
            for n in names:
                for p in range(4):
                    a = m.a[n]
                    was = a._matrix(np.frombuffer(w[n][p], a.dtype))
                    rows = a.rows if n != "total" else max(0, min(a.rows, m.rows - p * a.rows))
                    assert np.array_equal(a.read(p)[:rows], was[:rows], equal_nan=True), (n, p)
            assert not m.psync.read(0).any()
        for s in streams:
            s.destroy()
