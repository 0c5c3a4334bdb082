"""logprob_to_all and its gradient against their formulas in 64 bits: vocabularies that the members
share unevenly, masks that leave little or nothing, ties, extreme values, batches of one token and of
many."""
import numpy as np
import pytest

import roc_shmem_amd as rs
import row_reference as ref
from helpers import runtime
from row_arrays import Rows

pytestmark = pytest.mark.gpu

NP = {rs.BF16: np.uint16, rs.FLOAT: np.float32}
FORWARD = ("logprob", "entropy", "lse", "top_ids", "top_logprobs")


class Case:
    def __init__(self, dtype, rows, vocab, n_pes, *, team=(0, 1, None), shard=0, pad=0, shift=0, top_k=0, scale=1.0,
                 seed=0, logits=None, tokens=None):
        self.dtype, self.rows, self.vocab, self.n_pes, self.top_k = dtype, rows, vocab, n_pes, top_k
        self.scale = float(np.float32(scale))      # the number that the call gets
        start, stride, size = team
        self.size = size or n_pes
        self.members = [start + stride * m for m in range(self.size)]
        self.team = rs.roc_shmem_team_world()
        if team != (0, 1, None):
            status, self.team = rs.roc_shmem_team_split_strided(self.team, start, stride, self.size)
            assert status == 0
        self.shard = shard or -(-vocab // self.size)
        self.rng = np.random.default_rng(seed)
        self.logits = ref.to_type(dtype, self.rng.standard_normal((rows, vocab)) * 3 if logits is None else logits)
        self.tokens = np.asarray(self.rng.integers(-1, vocab, rows) if tokens is None else tokens, dtype=np.int64)
        self.width = min(self.shard, vocab)
        self.ld = self.width + pad
        self.array = Rows(rows, self.width, NP[dtype], self.ld, shift)
        self.shift = shift
        # what lies behind a short part of the vocabulary must not count: NaN there
        for m, pe in enumerate(self.members):
            part = self.logits[:, m * self.shard:(m + 1) * self.shard]
            whole = ref.to_type(dtype, np.full((rows, self.width), np.nan))
            whole[:, :part.shape[1]] = part
            self.array.write(pe, whole)
        self.token_array = self.numbers(self.tokens, np.int64)
        self.fields = dict(dtype=dtype, team=self.team, rows=rows, vocab=vocab, shard=shard, logits_ld=self.ld,
                           scale=scale, logits=self.array, tokens=self.token_array)

    def numbers(self, values, np_dtype):
        """[rows] on every PE."""
        return Rows(1, self.rows, np_dtype).write_all([np.asarray(values)] * self.n_pes)

    def f64(self):
        return ref.from_type(self.dtype, self.logits)

    def outputs(self):
        out = {n: Rows(1, self.rows, np.float32) for n in FORWARD[:3]}
        if self.top_k:
            out["top_ids"] = Rows(self.rows, self.top_k, np.int32)
            out["top_logprobs"] = Rows(self.rows, self.top_k, np.float32)
        return out

    def call(self, out):
        args = rs.LogprobArgs(top_k=self.top_k, **{**self.fields, **out})
        n = rs.roc_shmem_logprob_work_bytes(args)
        if n:
            self.work = rs.sym_array(n, np.uint8, fill=0xEE)
            self.psync = rs.sym_array(rs.ROC_SHMEM_REDUCE_SYNC_SIZE, np.int64, fill=0)
            args.work, args.pSync = self.work.addr, self.psync.addr
        return args

    def psync_is_zero(self):
        return not hasattr(self, "psync") or not any(self.psync.read(p).any() for p in range(self.n_pes))

    def check(self, out):
        want = ref.logprob_forward(self.f64(), self.tokens, self.scale, self.top_k)
        for name, array in out.items():
            value, error = want[name]
            for pe in range(self.n_pes):
                array.check_rest(pe, name, array.rows if pe in self.members else 0)
                if pe not in self.members:
                    continue
                got = array.read(pe)
                if name == "top_ids":
                    assert np.array_equal(got, value), "ids on PE %d: %s, want %s" % (pe, got[(got != value).any(1)][:2], value[(got != value).any(1)][:2])
                else:
                    ref.check("%s on PE %d" % (name, pe), rs.FLOAT, got, value.reshape(got.shape), np.reshape(error, got.shape))
        assert self.psync_is_zero()


def run_forward(c, times=1, stream=None):
    out = c.outputs()
    for a in out.values():
        a.remember()
    args = c.call(out)
    for _ in range(times):
        rs.roc_shmem_logprob_to_all(args, stream)
    rs.synchronize()
    c.check(out)
    return out, args


def run_backward(c, *, in_place=False, which=("grad_logprob", "grad_entropy", "grad_lse"), pad=0):
    fwd = ref.logprob_forward(c.f64(), c.tokens, c.scale, 0)
    lse, entropy = (np.asarray(fwd[n][0], dtype=np.float32) for n in ("lse", "entropy"))
    g = {n: c.rng.standard_normal(c.rows).astype(np.float32) for n in which}
    out = c.array if in_place else Rows(c.rows, c.width, NP[c.dtype], c.ld + pad, c.shift)
    out.remember()
    args = rs.LogprobGradArgs(lse=c.numbers(lse, np.float32), entropy=c.numbers(entropy, np.float32), grad_logits=out,
                              grad_ld=out.ld, **{n: c.numbers(v, np.float32) for n, v in g.items()}, **c.fields)
    rs.roc_shmem_logprob_to_all_grad(args)
    rs.synchronize()
    want, error = ref.logprob_backward(c.f64(), c.tokens, lse, entropy, c.scale, g.get("grad_logprob"),
                                       g.get("grad_entropy"), g.get("grad_lse"))
    for pe in range(c.n_pes):
        if pe not in c.members:
            out.check_rest(pe, "grad_logits", 0)
            continue
        m = c.members.index(pe)
        part = want[:, m * c.shard:(m + 1) * c.shard]
        got = out.read(pe)
        ref.check("grad_logits on PE %d" % pe, c.dtype, got[:, :part.shape[1]], part, error[:, m * c.shard:(m + 1) * c.shard])
        # nothing is written behind the part, between the rows or around them
        was = out._matrix(out.before[pe])
        assert got[:, part.shape[1]:].tobytes() == was[:, part.shape[1]:].tobytes()
        out.check_rest(pe, "grad_logits", out.rows)


SHAPES = [
    # rows, vocab, pes, what else
    (1, 1, 1, dict(top_k=1)),
    (1, 5, 8, dict(top_k=5)),                                      # members without any id
    (1, 32000, 8, dict(top_k=20)),
    (1, 131072, 1, dict(top_k=32)),
    (2, 50257, 4, dict(top_k=5, scale=0.7)),
    (17, 3001, 3, dict(top_k=7, pad=3, shift=1)),                  # rows start at odd elements
    (64, 8192, 8, dict(top_k=1)),
    (100, 10000, 8, dict(team=(1, 2, 3), top_k=3, scale=1.7)),     # members 1, 3, 5
    (33, 1000, 4, dict(shard=300, top_k=4)),                       # the last part is shorter
    (33, 1000, 4, dict(shard=600, top_k=4)),                       # two members hold nothing
    (255, 4096, 2, dict(top_k=20)),
    (256, 4096, 2, dict(top_k=20)),
    (700, 777, 5, dict(top_k=32)),
    (700, 16500, 2, dict()),
]


@pytest.mark.parametrize("rows,vocab,pes,more", SHAPES)
@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_forward_over_shapes(dtype, rows, vocab, pes, more):
    with runtime(pes, heap_size=256 << 20):
        run_forward(Case(dtype, rows, vocab, pes, seed=rows + vocab, **more))


@pytest.mark.parametrize("rows,vocab,pes,more", SHAPES)
@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_backward_over_shapes(dtype, rows, vocab, pes, more):
    with runtime(pes, heap_size=256 << 20):
        run_backward(Case(dtype, rows, vocab, pes, seed=rows + vocab, **more))


@pytest.mark.parametrize("rows,vocab", [(3, 5000), (300, 5000), (2, 70001)])   # the last: several workgroups to a row
@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_masks(dtype, rows, vocab):
    """Rows with few logits left, one, none; ties everywhere; rows at the type's lowest value."""
    rng = np.random.default_rng(rows)
    base = rng.standard_normal((rows, vocab)) * 2
    lowest = -3.3895314e38
    kinds = {
        "a third banned": np.where(rng.random((rows, vocab)) < 0.33, -np.inf, base),
        "ten left": np.where(np.arange(vocab) % 500 == 17, base, -np.inf),
        "one left": np.where(np.arange(vocab) == 4321, base, -np.inf),
        "none left": np.full((rows, vocab), -np.inf),
        "all equal": np.full((rows, vocab), 1.5),
        "few values": np.round(base),
        "rising": np.broadcast_to(np.arange(vocab) // 64 * 0.25, (rows, vocab)),
        "falling": np.broadcast_to(-(np.arange(vocab) // 64) * 0.25, (rows, vocab)),
        "masked by the lowest value": np.where(rng.random((rows, vocab)) < 0.5, lowest, base),
        "signed zeros": np.where(np.arange(vocab) % 3 == 0, -0.0, 0.0) * np.ones((rows, 1)),
    }
    with runtime(4, heap_size=256 << 20):
        for name, logits in kinds.items():
            print(name, flush=True)
            c = Case(dtype, rows, vocab, 4, logits=logits, top_k=20, tokens=rng.integers(0, vocab, rows))
            run_forward(c)
            run_backward(c)


@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_several_workgroups_to_a_row_of_several_batches_each(dtype):
    rows, vocab = 255, 80001
    rng = np.random.default_rng(4)
    base = rng.standard_normal((rows, vocab)) * 2
    base[40:80] = np.where(rng.random((40, vocab)) < 0.5, -np.inf, base[40:80])
    base[80:100] = np.round(base[80:100])
    base[100:105] = 1.5
    base[105:110] = np.where(np.arange(vocab) % 5000 == 17, base[105:110], -np.inf)
    base[110] = -np.inf
    base[111] = np.where(np.arange(vocab) == vocab - 1, 0.5, -np.inf)
    with runtime(3, heap_size=128 << 20):
        run_forward(Case(dtype, rows, vocab, 3, logits=base, top_k=20, tokens=rng.integers(0, vocab, rows)), times=2)


@pytest.mark.parametrize("vocab", [9000, 20000])
def test_many_rows_that_are_not_long(vocab):
    """Workgroups of half as many waves, with one batch each or several."""
    rows = 2050
    rng = np.random.default_rng(6)
    base = rng.standard_normal((rows, vocab)) * 2
    base[::7] = np.round(base[::7])
    base[::50] = -1.5
    base[1::50, 30:] = -np.inf
    with runtime(2, heap_size=128 << 20):
        run_forward(Case(rs.BF16, rows, vocab, 2, logits=base, top_k=9, tokens=rng.integers(0, vocab, rows)))


def test_rows_at_the_lowest_value_are_uniform():
    """Logits that are all the type's lowest value are equal like any others; the normaliser itself,
    lowest + ln V, is the lowest value as a float."""
    rows, vocab = 2, 3000
    low = np.finfo(np.float32).min
    with runtime(2):
        c = Case(rs.FLOAT, rows, vocab, 2, logits=np.full((rows, vocab), low, dtype=np.float32), tokens=[5, 2999], top_k=3)
        out = c.outputs()
        rs.roc_shmem_logprob_to_all(c.call(out))
        rs.synchronize()
        assert np.allclose(out["logprob"].read(0), -np.log(vocab), rtol=1e-6, atol=0)
        assert np.allclose(out["entropy"].read(1), np.log(vocab), rtol=1e-6, atol=0)
        assert np.array_equal(out["lse"].read(0), np.full((1, rows), low))
        assert np.array_equal(out["top_ids"].read(0), [[0, 1, 2]] * rows)


@pytest.mark.parametrize("rows,vocab", [(4, 2500), (400, 2500), (4, 50000)])
def test_not_a_number(rows, vocab):
    """A row with a NaN or plus infinity has NaN results, its neighbours have their own; NaN is never an
    alternative."""
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((rows, vocab)).astype(np.float32)
    logits[1, 1234] = np.nan
    logits[2, vocab - 1] = np.inf
    logits[3] = np.nan
    with runtime(2):
        c = Case(rs.FLOAT, rows, vocab, 2, logits=logits, tokens=np.full(rows, 7), top_k=4)
        out = c.outputs()
        rs.roc_shmem_logprob_to_all(c.call(out))
        rs.synchronize()
        for n in FORWARD[:3]:
            got = out[n].read(1)[0]
            assert np.isnan(got[1:4]).all() and np.isfinite(np.delete(got, [1, 2, 3])).all(), n
        ids = out["top_ids"].read(0)
        order = lambda v: np.argsort(-v, kind="stable")[:4]  # noqa: E731
        assert np.array_equal(ids[1], order(np.where(np.isnan(logits[1]), -np.inf, logits[1])))
        assert ids[2][0] == vocab - 1
        assert np.array_equal(ids[3], [-1] * 4) and np.isnan(out["top_logprobs"].read(0)[3]).all()
        lse = out["lse"].read(0)[0]
        g = Rows(rows, c.width, np.float32, c.ld)
        rs.roc_shmem_logprob_to_all_grad(rs.LogprobGradArgs(lse=c.numbers(lse, np.float32), grad_lse=c.numbers(np.ones(rows), np.float32),
                                                            grad_logits=g, **c.fields))
        rs.synchronize()
        got = g.read(0)
        assert np.isnan(got[1:4]).all() and np.isfinite(np.delete(got, [1, 2, 3], 0)).all()


def test_tokens_outside_the_vocabulary_raise_the_status_word():
    for rows in (3, 300):
        rs.roc_shmem_init(2, 64 << 20, 4, 1024)
        try:
            tokens = np.zeros(rows, dtype=np.int64)
            tokens[1], tokens[2] = 1000, -5
            c = Case(rs.FLOAT, rows, 1000, 2, tokens=tokens)
            out = c.outputs()
            rs.roc_shmem_logprob_to_all(c.call(out))
            rs.synchronize()
            assert rs.take_status() == 2
            got = out["logprob"].read(0)[0]
            assert np.isnan(got[1]) and got[2] == 0 and np.isfinite(got[0])
            g = Rows(rows, c.width, np.float32, c.ld)
            ones = c.numbers(np.ones(rows), np.float32)
            rs.roc_shmem_logprob_to_all_grad(rs.LogprobGradArgs(lse=c.numbers(out["lse"].read(0)[0], np.float32), grad_logprob=ones,
                                                                grad_logits=g, **c.fields))
            rs.synchronize()
            assert rs.take_status() == 2
            grads = g.read(0)
            assert not grads[1].any() and not grads[2].any() and grads[0].any()
        finally:
            rs.roc_shmem_finalize()


@pytest.mark.parametrize("vocab", [1000, 20000])     # lines of the gradient numbered through, and workgroups of their own
def test_tokens_outside_the_vocabulary_have_no_gradient(vocab):
    rs.roc_shmem_init(2, 64 << 20, 4, 1024)
    try:
        rows = 40
        c = Case(rs.FLOAT, rows, vocab, 2, tokens=np.arange(rows))
        lse = np.asarray(ref.logprob_forward(c.f64(), c.tokens, c.scale, 0)["lse"][0], dtype=np.float32)
        lse, ones = c.numbers(lse, np.float32), c.numbers(np.ones(rows), np.float32)

        def gradient(tokens):
            g = Rows(rows, c.width, np.float32, c.ld)
            args = rs.LogprobGradArgs(lse=lse, grad_logprob=ones, grad_logits=g, **{**c.fields, "tokens": c.numbers(tokens, np.int64)})
            rs.roc_shmem_logprob_to_all_grad(args)
            rs.synchronize()
            return g.read(0), g.read(1)

        whole = gradient(c.tokens)
        assert rs.take_status() == 0
        for row, token in ((0, vocab), (17, 1 << 40), (39, np.iinfo(np.int64).max), (5, -1), (6, np.iinfo(np.int64).min)):
            tokens = c.tokens.copy()
            tokens[row] = token
            part = gradient(tokens)
            assert rs.take_status() == (2 if token > 0 else 0)
            for got, was in zip(part, whole):
                assert not got[row].any()
                assert np.array_equal(np.delete(got, row, 0), np.delete(was, row, 0))
    finally:
        rs.roc_shmem_finalize()


@pytest.mark.parametrize("rows", [3, 300])
def test_as_many_members_as_there_can_be(rows):
    with runtime(128, heap_size=8 << 20):
        for dtype in (rs.BF16, rs.FLOAT):
            run_forward(Case(dtype, rows, 1000, 128, top_k=20))
            run_backward(Case(dtype, rows, 1000, 128))


def test_as_many_rows_as_there_can_be():
    with runtime(1, heap_size=1 << 30):
        c = Case(rs.BF16, (1 << 22) - 1, 6, 1)
        run_forward(c)
        run_backward(c)


@pytest.mark.parametrize("rows", [3, 300])
def test_a_shard_longer_than_any_vocabulary(rows):
    """The first member holds everything; the others' ids would lie past 2^31."""
    with runtime(4):
        for vocab in (5, 3000):
            run_forward(Case(rs.BF16, rows, vocab, 4, shard=(1 << 30) - 1, top_k=5))
            run_backward(Case(rs.BF16, rows, vocab, 4, shard=(1 << 30) - 1))


def test_each_result_alone():
    with runtime(4):
        for rows in (2, 260):
            for names in (("logprob",), ("entropy",), ("lse",), ("top_ids",), ("top_logprobs",), ("lse", "top_ids")):
                top = 3 if any(n.startswith("top") for n in names) else 0
                c = Case(rs.BF16, rows, 4001, 4, top_k=top)
                if "logprob" not in names:
                    c.fields.pop("tokens")
                out = {n: a for n, a in c.outputs().items() if n in names}
                for a in out.values():
                    a.remember()
                rs.roc_shmem_logprob_to_all(c.call(out))
                rs.synchronize()
                c.check(out)


@pytest.mark.parametrize("which", [("grad_logprob",), ("grad_entropy",), ("grad_lse",), ("grad_logprob", "grad_lse")])
def test_each_gradient_alone(which):
    with runtime(2):
        run_backward(Case(rs.FLOAT, 9, 4001, 2), which=which)
        run_backward(Case(rs.BF16, 9, 4001, 2), which=which, pad=3)


@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_gradient_in_place_of_the_logits(dtype):
    with runtime(3):
        run_backward(Case(dtype, 11, 7000, 3, pad=1), in_place=True)


@pytest.mark.parametrize("rows", [1, 5, 200])
def test_calls_in_a_row_share_their_workspace(rows):
    with runtime(8):
        run_forward(Case(rs.BF16, rows, 40000, 8, top_k=6), times=5)


def test_gradients_against_differences():
    """<G, logprob> + <H, entropy> + <K, lse> along random directions against differences of the formula."""
    rows, vocab, scale = 6, 700, float(np.float32(1.3))
    with runtime(2):
        c = Case(rs.FLOAT, rows, vocab, 2, scale=scale, tokens=[0, 5, 699, -1, 350, 349])
        g = {n: c.rng.standard_normal(rows).astype(np.float32) for n in ("grad_logprob", "grad_entropy", "grad_lse")}
        out = c.outputs()
        rs.roc_shmem_logprob_to_all(c.call(out))
        d = Rows(rows, c.width, np.float32, c.ld)
        rs.roc_shmem_logprob_to_all_grad(rs.LogprobGradArgs(lse=out["lse"], entropy=out["entropy"], grad_logits=d,
                                                            **{n: c.numbers(v, np.float32) for n, v in g.items()}, **c.fields))
        rs.synchronize()
        grad = np.concatenate([d.read(0), d.read(1)], 1).astype(np.float64)
        direction = np.random.default_rng(8).standard_normal((rows, vocab))

        def loss(step):
            w = ref.logprob_forward(c.f64() + step * direction, c.tokens, scale, 0)
            return sum((g["grad_" + n].astype(np.float64) * w[n][0]).sum() for n in ("logprob", "entropy", "lse"))

        d1, d2 = ((loss(s) - loss(-s)) / (2 * s) for s in (1e-3, 5e-4))
        want = d2 + (d2 - d1) / 3
        # forward: a lse off by some 20 roundings of 2^-24 moves every probability by as much
        assert abs((grad * direction).sum() - want) <= 1e-5 * np.abs(grad * direction).sum() + 1e-8


def test_rows_beyond_4_gib():
    """Rows whose bytes lie past 2^32 of the array's start."""
    rows, vocab, ld = 9, 600, 300_000_001       # 8 * ld * 2 bytes = 4.8e9
    rs.roc_shmem_init(1, 16 << 30, 4, 1024)
    try:
        rng = np.random.default_rng(2)
        logits = ref.to_type(rs.BF16, rng.standard_normal((rows, vocab)) * 3)
        a = rs.sym_array((rows - 1) * ld + vocab, np.uint16)
        for r in range(rows):
            a.write(0, logits[r], r * ld)
        tokens = rng.integers(0, vocab, rows)
        t = Rows(1, rows, np.int64).write(0, tokens)
        out = {n: Rows(1, rows, np.float32) for n in FORWARD[:3]}
        work, psync = rs.sym_array(1 << 20, np.uint8), rs.sym_array(rs.ROC_SHMEM_REDUCE_SYNC_SIZE, np.int64, fill=0)
        fields = dict(dtype=rs.BF16, team=rs.roc_shmem_team_world(), rows=rows, vocab=vocab, logits_ld=ld, logits=a, tokens=t)
        args = rs.LogprobArgs(work=work, pSync=psync, **out, **fields)
        assert rs.roc_shmem_logprob_work_bytes(args) <= 1 << 20
        rs.roc_shmem_logprob_to_all(args)
        rs.synchronize()
        want = ref.logprob_forward(ref.from_type(rs.BF16, logits), tokens, 1.0, 0)
        for n, o in out.items():
            ref.check(n, rs.FLOAT, o.read(0)[0], *want[n])
        ones = Rows(1, rows, np.float32).write(0, np.ones(rows, np.float32))
        rs.roc_shmem_logprob_to_all_grad(rs.LogprobGradArgs(lse=out["lse"], grad_logprob=ones, grad_logits=a, grad_ld=ld, **fields))
        rs.synchronize()
        value, error = ref.logprob_backward(ref.from_type(rs.BF16, logits), tokens, out["lse"].read(0)[0], None, 1.0,
                                            np.ones(rows), None, None)
        for r in range(rows):
            ref.check("row %d" % r, rs.BF16, a.read(0, vocab, r * ld), value[r], error[r])
    finally:
        rs.roc_shmem_finalize()
