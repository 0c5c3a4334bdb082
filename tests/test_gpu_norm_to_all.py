"""norm_to_all and its gradient against their formulas in 64 bits, over types, widths, strides, teams,
gates and ways of holding the residual stream; bytes beyond the results and other PEs' slices stay as
they were."""
import numpy as np
import pytest

import roc_shmem_amd as rs
import row_reference as ref
from helpers import runtime
from row_arrays import Rows

pytestmark = pytest.mark.gpu

NP = {rs.BF16: np.uint16, rs.FLOAT: np.float32}
EPS, A, B, O = 1e-5, 0.75, 1.5, 0.5


class Case:
    """One batch: its operands on the PEs and the arguments that name them."""

    def __init__(self, dtype, rows, cols, n_pes, *, team=(0, 1, None), post=True, gate=1, pre_w=True, post_w=True,
                 replicated=False, pad=0, shift=0, seed=0, scale=1.0):
        self.dtype, self.rows, self.cols, self.n_pes = dtype, rows, cols, n_pes
        start, stride, size = team
        self.size = size or n_pes
        self.members = [start + stride * m for m in range(self.size)]
        self.team = rs.roc_shmem_team_world()
        if team != (0, 1, None):
            status, self.team = rs.roc_shmem_team_split_strided(self.team, start, stride, self.size)
            assert status == 0
        self.share = max(1, -(-rows // self.size))
        self.replicated, self.post, self.pad, self.shift = replicated, post, pad, shift
        self.rng = np.random.default_rng(seed)
        self.scale = scale
        self.rpg = 0 if gate in (0, 1) else gate
        self.gates = 0 if gate == 0 or rows == 0 else 1 if gate == 1 else -(-rows // gate)
        self.pre_w, self.post_w = pre_w, post_w and post
        self.keep = []
        self.weights = {}
        if pre_w:
            self.weights["pre_weight"] = self.numbers(1, cols, 0.3)
        if self.post_w:
            self.weights["post_weight"] = self.numbers(1, cols, 0.3)
        if self.gates:
            self.weights["gate"] = self.numbers(self.gates, cols, 0.5)
        flags = (rs.NORM_POST if post else 0) | (rs.NORM_REPLICATED if replicated else 0)
        self.fields = dict(dtype=dtype, flags=flags, team=self.team, rows=rows, cols=cols, rows_per_gate=self.rpg,
                           eps=EPS, residual_scale=A, block_scale=B, weight_offset=O,
                           source_ld=cols + pad, residual_ld=cols + 2 * pad, normed_ld=cols + pad)
        for name, v in self.weights.items():
            self.fields[name] = self.rows_of(len(v), cols, 0).write_all([v] * n_pes)

    def numbers(self, rows, cols, scale=1.0):
        return ref.to_type(self.dtype, self.rng.standard_normal((rows, cols)) * scale * self.scale)

    def rows_of(self, rows, cols, ld, dtype=None):
        a = Rows(rows, cols, dtype or NP[self.dtype], ld or None, self.shift)
        self.keep.append(a)
        return a

    def stream(self, values=None):
        """An array held as the residual stream is, with `values` (all rows) on their owners."""
        held = self.rows if self.replicated else self.share
        a = self.rows_of(held, self.cols, self.cols + 2 * self.pad)
        if values is not None:
            for m, pe in enumerate(self.members):
                if self.replicated:
                    a.write(pe, values)
                else:
                    mine = values[m * self.share:(m + 1) * self.share]
                    full = a.read(pe)
                    full[:len(mine)] = mine
                    a.write(pe, full)
        return a

    def shared(self, values=None):
        """An array of `total`'s shape."""
        keep = self.replicated, self.pad
        self.replicated, self.pad = False, 0
        a = self.stream(values)
        self.replicated, self.pad = keep
        return a

    def formula(self):
        f = lambda name: ref.from_type(self.dtype, self.weights[name]) if name in self.weights else None  # noqa: E731
        one = lambda v: None if v is None else v[0]  # noqa: E731
        return dict(pre=one(f("pre_weight")), post=one(f("post_weight")), gate=f("gate"), has_post=self.post,
                    rows_per_gate=self.rpg, eps=float(np.float32(EPS)), a=A, b=B, o=O)

    def check_everywhere(self, name, array, want, error, dtype=None):
        """The same rows on every member, nothing on other PEs."""
        for pe in range(self.n_pes):
            if pe in self.members:
                ref.check("%s on PE %d" % (name, pe), self.dtype if dtype is None else dtype, array.read(pe), want, error)
            array.check_rest(pe, name, array.rows if pe in self.members else 0)

    def check_stream(self, name, array, want, error, replicated=None):
        if self.replicated if replicated is None else replicated:
            return self.check_everywhere(name, array, want, error)
        for pe in range(self.n_pes):
            rows = 0
            if pe in self.members:
                part = slice(self.members.index(pe) * self.share, (self.members.index(pe) + 1) * self.share)
                rows = len(want[part])
                ref.check("%s on PE %d" % (name, pe), self.dtype, array.read(pe)[:rows], want[part], error[part])
            array.check_rest(pe, name, rows)


def run_forward(c, *, in_place=False, keep=True, normed=True, stream=None):
    partials = [c.numbers(c.rows, c.cols) for _ in range(c.size)]
    x = c.numbers(c.rows, c.cols, 2.0)
    source = c.rows_of(c.rows, c.cols, c.cols + c.pad)
    for m, pe in enumerate(c.members):
        source.write(pe, partials[m])
    residual = c.stream(x)
    out = residual if in_place else c.stream()
    h = source if in_place else c.rows_of(c.rows, c.cols, c.cols + c.pad)
    total = c.shared() if keep else None
    watched = [a for a in (out, h, total) if a is not None]
    for a in watched:
        a.remember()
    fields = dict(c.fields)
    if not normed:
        fields.pop("pre_weight", None)
    args = rs.NormArgs(source=source, residual=residual, residual_out=out, normed=h if normed else None, total=total, **fields)
    rs.roc_shmem_norm_to_all(args, stream)
    rs.synchronize()
    want = ref.norm_forward(np.stack([ref.from_type(c.dtype, v) for v in partials]), ref.from_type(c.dtype, x), **c.formula())
    c.check_stream("residual_out", out, *want["residual_out"])
    if normed:
        c.check_everywhere("normed", h, *want["normed"])
    if keep:
        c.check_stream("total", total, *want["total"], replicated=False)
    return args


def run_backward(c, *, in_place=False, has_normed=True, has_out=True, sums=True, without=()):
    partials = [c.numbers(c.rows, c.cols) for _ in range(c.size)]
    x, total, gout = (c.numbers(c.rows, c.cols, s) for s in (2.0, 1.5, 1.0))
    gn = c.rows_of(c.rows, c.cols, c.cols + c.pad) if has_normed else None
    if has_normed:
        for m, pe in enumerate(c.members):
            gn.write(pe, partials[m])
    needs_total = c.post or c.gates
    arrays = {"grad_normed": gn, "residual_out": c.stream(x) if has_normed else None,
              "total": c.shared(total) if needs_total else None, "grad_residual_out": c.stream(gout) if has_out else None,
              "grad_source": gn if in_place and has_normed else c.rows_of(c.rows, c.cols, c.cols + c.pad)}
    arrays["grad_residual"] = arrays["grad_residual_out"] if in_place and has_out else c.stream()
    if sums:
        if has_normed:
            arrays["grad_pre_weight"] = c.rows_of(1, c.cols, 0, np.float32)
        if c.post:
            arrays["grad_post_weight"] = c.rows_of(1, c.cols, 0, np.float32)
        if c.gates:
            arrays["grad_gate"] = c.rows_of(c.gates, c.cols, 0, np.float32)
    for n in without:
        arrays.pop(n)
    results = [n for n in arrays if n in ("grad_source", "grad_residual", "grad_pre_weight", "grad_post_weight", "grad_gate")]
    for n in results:
        arrays[n].remember()
    fields = dict(c.fields)
    if not has_normed:
        fields.pop("pre_weight", None)
    args = rs.NormGradArgs(**arrays, **fields)
    work = rs.sym_array(max(1, rs.roc_shmem_norm_grad_work_bytes(args)), np.uint8, fill=0xEE)
    args.work = work.addr
    rs.roc_shmem_norm_to_all_grad(args)
    rs.synchronize()
    f = lambda v: ref.from_type(c.dtype, v)  # noqa: E731
    want = ref.norm_backward(np.stack([f(v) for v in partials]) if has_normed else None, f(gout) if has_out else None, f(x),
                             f(total) if needs_total else None, **c.formula())
    for n in results:
        value, error = want[n]
        if n == "grad_residual":
            c.check_stream(n, arrays[n], value, error)
        elif n == "grad_source":
            c.check_everywhere(n, arrays[n], value, error)
        else:
            c.check_everywhere(n, arrays[n], np.atleast_2d(value), np.atleast_2d(error), rs.FLOAT)
    return args


# Widths on either side of each change of lanes and vectors per row, odd ones, and the widest.
WIDTHS = [1, 7, 8, 64, 257, 512, 513, 1000, 1024, 1025, 2048, 2050, 4096, 4100, 5119, 8192, 8200, 16384]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_forward_over_widths(dtype, cols):
    with runtime(4):
        run_forward(Case(dtype, 5, cols, 4, seed=cols))


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_backward_over_widths(dtype, cols):
    with runtime(4):
        run_backward(Case(dtype, 5, cols, 4, seed=cols))


SHAPES = [
    # rows, cols, pes, what else
    (1, 640, 8, dict()),
    (1, 640, 8, dict(replicated=True, gate=0)),
    (3, 300, 1, dict(gate=0, post=False)),
    (7, 300, 8, dict(gate=0)),                                     # fewer rows than members: some own none
    (9, 136, 8, dict()),                                           # the last owner's share is short
    (9, 136, 8, dict(replicated=True, gate=2)),
    (37, 1031, 3, dict(gate=10, pad=5, shift=3)),                  # rows start at odd elements
    (37, 1032, 3, dict(gate=10, pad=8, post=False)),
    (33, 96, 8, dict(team=(1, 2, 3), gate=4)),                     # members 1, 3, 5
    (33, 96, 8, dict(team=(2, 1, 5), replicated=True, pad=1, shift=1)),
    (20, 2056, 5, dict(pre_w=False, post_w=False, gate=0)),
    (20, 2056, 5, dict(pre_w=False, post_w=False, gate=1, post=False)),
    (130, 64, 2, dict(gate=1)),
    (130, 64, 2, dict(gate=130)),
    (700, 72, 16, dict(gate=7, seed=3)),
]


@pytest.mark.parametrize("rows,cols,pes,more", SHAPES)
@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_forward_over_shapes(dtype, rows, cols, pes, more):
    with runtime(pes):
        run_forward(Case(dtype, rows, cols, pes, **more))


@pytest.mark.parametrize("rows,cols,pes,more", SHAPES)
@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_backward_over_shapes(dtype, rows, cols, pes, more):
    with runtime(pes):
        run_backward(Case(dtype, rows, cols, pes, **more))


@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
@pytest.mark.parametrize("replicated", [False, True])
def test_results_in_place_of_operands(dtype, replicated):
    with runtime(4):
        run_forward(Case(dtype, 21, 1500, 4, replicated=replicated), in_place=True)
        run_backward(Case(dtype, 21, 1500, 4, replicated=replicated, gate=5), in_place=True)


@pytest.mark.parametrize("cols", [5, 100, 1500, 2051, 8190])
@pytest.mark.parametrize("dtype", [rs.BF16, rs.FLOAT])
def test_rows_that_end_inside_a_vector_in_place(dtype, cols):
    """Without a norm of the sum a row's new residual stream is stored soonest after its loads."""
    with runtime(3):
        for gate in (0, 4):
            for replicated in (False, True):
                run_forward(Case(dtype, 13, cols, 3, gate=gate, post=False, replicated=replicated), in_place=True)
                run_backward(Case(dtype, 13, cols, 3, gate=gate, post=False, replicated=replicated), in_place=True)


def test_as_many_members_as_there_can_be():
    with runtime(128, heap_size=8 << 20):
        for rows in (1, 130, 300):      # most members own nothing, one row, three
            run_forward(Case(rs.BF16, rows, 72, 128, gate=0))
            run_backward(Case(rs.FLOAT, rows, 72, 128, gate=0))


def test_as_many_rows_as_there_can_be():
    with runtime(1, heap_size=1 << 30):
        run_forward(Case(rs.BF16, (1 << 22) - 1, 8, 1, gate=0))
        run_backward(Case(rs.BF16, (1 << 22) - 1, 8, 1, gate=0, post=False), sums=False)


def test_optional_operands():
    with runtime(4):
        run_forward(Case(rs.BF16, 12, 520, 4), keep=False)
        run_forward(Case(rs.BF16, 12, 520, 4), normed=False)
        run_backward(Case(rs.BF16, 12, 520, 4), has_out=False)
        run_backward(Case(rs.BF16, 12, 520, 4), has_normed=False)
        run_backward(Case(rs.FLOAT, 12, 520, 4, gate=3), sums=False)
        run_backward(Case(rs.FLOAT, 12, 520, 4, gate=0, post=False))
        for without in (("grad_residual",), ("grad_pre_weight",), ("grad_post_weight", "grad_gate"), ("grad_pre_weight", "grad_post_weight")):
            for gate in (1, 3):
                run_backward(Case(rs.BF16, 12, 520, 4, gate=gate), without=without)


def test_rows_beyond_4_gib():
    """Strides that take the last rows past 2^32 bytes of their arrays' start."""
    rows, cols, ld = 9, 600, 300_000_001
    rs.roc_shmem_init(1, 64 << 30, 4, 1024)
    try:
        rng = np.random.default_rng(2)
        numbers = lambda: ref.to_type(rs.BF16, rng.standard_normal((rows, cols)))  # noqa: E731
        y, x = numbers(), numbers()

        def far(values):
            a = rs.sym_array((rows - 1) * ld + cols, np.uint16)
            for r in range(rows if values is not None else 0):
                a.write(0, values[r], r * ld)
            return a

        def near(a):
            return np.stack([a.read(0, cols, r * ld) for r in range(rows)])

        source, stream, total = far(y), far(x), rs.sym_array(rows * cols, np.uint16)
        fields = dict(dtype=rs.BF16, flags=rs.NORM_POST, team=rs.roc_shmem_team_world(), rows=rows, cols=cols, eps=EPS,
                      residual_scale=A, block_scale=B, source_ld=ld, residual_ld=ld, normed_ld=ld)
        formula = dict(pre=None, post=None, gate=None, has_post=True, rows_per_gate=0, eps=float(np.float32(EPS)), a=A, b=B, o=O)
        f = lambda v: ref.from_type(rs.BF16, v)  # noqa: E731
        rs.roc_shmem_norm_to_all(rs.NormArgs(source=source, residual=stream, residual_out=stream, normed=source, total=total, **fields))
        rs.synchronize()
        want = ref.norm_forward(f(y)[None], f(x), **formula)
        ref.check("normed", rs.BF16, near(source), *want["normed"])
        ref.check("residual_out", rs.BF16, near(stream), *want["residual_out"])
        out, kept, dn, dx = near(stream), total.read(0).reshape(rows, cols), numbers(), numbers()
        for r in range(rows):
            source.write(0, dn[r], r * ld)
        grad = far(dx)
        rs.roc_shmem_norm_to_all_grad(rs.NormGradArgs(grad_normed=source, grad_source=source, residual_out=stream, total=total,
                                                      grad_residual_out=grad, grad_residual=grad, **fields))
        rs.synchronize()
        want = ref.norm_backward(f(dn)[None], f(dx), f(out), f(kept), **formula)
        ref.check("grad_source", rs.BF16, near(source), *want["grad_source"])
        ref.check("grad_residual", rs.BF16, near(grad), *want["grad_residual"])
    finally:
        rs.roc_shmem_finalize()


@pytest.mark.parametrize("rows_per_gate", [1, 3, 4097, 5000])
def test_gate_gradients_where_units_hold_many_rows(rows_per_gate):
    # more rows than units: a unit walks several rows, whole gate groups or parts of one
    with runtime(2, heap_size=128 << 20):
        run_backward(Case(rs.FLOAT, 9001, 40, 2, gate=rows_per_gate, seed=rows_per_gate))
        run_backward(Case(rs.BF16, 2100, 1100, 2, gate=rows_per_gate, seed=rows_per_gate))


@pytest.mark.parametrize("gate", [0, 1, 3, 700])
def test_many_rows_of_many_members(gate):
    with runtime(5, heap_size=128 << 20):
        run_backward(Case(rs.BF16, 1501, 1100, 5, gate=gate, seed=gate))


def test_no_rows():
    with runtime(4):
        run_forward(Case(rs.BF16, 0, 100, 4, gate=0))
        c = Case(rs.FLOAT, 0, 100, 4, gate=0)
        gp, gq = c.rows_of(1, 100, 0, np.float32), c.rows_of(1, 100, 0, np.float32)
        gn, gs, x, t = (c.rows_of(1, 100, 0) for _ in range(4))
        for a in (gp, gq, gn, gs, x, t):
            a.remember()
        args = rs.NormGradArgs(grad_normed=gn, residual_out=x, total=t, grad_source=gs, grad_pre_weight=gp, grad_post_weight=gq, **c.fields)
        assert rs.roc_shmem_norm_grad_work_bytes(args) == 0
        rs.roc_shmem_norm_to_all_grad(args)
        rs.synchronize()
        for pe in range(4):      # a sum over no rows
            assert not gp.read(pe).any() and not gq.read(pe).any()
            for a in (gn, gs, x, t):
                a.check_rest(pe, "operand", 0)


def test_rows_of_zeros_and_of_infinities():
    with runtime(2):
        c = Case(rs.FLOAT, 4, 128, 2, gate=0)
        source = c.rows_of(4, 128, c.cols)
        v = c.numbers(4, 128)
        v[0] = 0
        x = c.numbers(4, 128)
        x[0] = 0
        bad = v.copy()
        bad[2, 5], bad[3, 7] = np.inf, np.nan
        source.write(0, bad).write(1, v)
        h, out, res = c.rows_of(4, 128, c.cols), c.stream(), c.stream(x)
        rs.roc_shmem_norm_to_all(rs.NormArgs(source=source, residual=res, residual_out=out, normed=h, **c.fields))
        rs.synchronize()
        got = h.read(1)
        assert not got[0].any()                                  # eps keeps a row of zeros at zero
        assert np.isfinite(got[1]).all()                         # and a row's numbers are its own
        assert np.isnan(got[2]).all() and np.isnan(got[3]).all()


def differences(c, f, leaves, name, direction):
    """Central difference of f along `direction` of one leaf, in 64 bits, extrapolated once."""
    def at(step):
        return f({**leaves, name: leaves[name] + step * direction})
    d1 = (at(1e-3) - at(-1e-3)) / 2e-3
    d2 = (at(5e-4) - at(-5e-4)) / 1e-3
    return d2 + (d2 - d1) / 3


@pytest.mark.parametrize("post,gate", [(True, 4), (True, 0), (False, 1), (False, 0)])
def test_gradients_against_differences(post, gate):
    """The kernels' gradients of <G, normed> + <H, residual_out> along random directions against
    differences of the forward formula."""
    with runtime(3):
        c = Case(rs.FLOAT, 10, 200, 3, post=post, gate=gate, replicated=True)
        f64 = lambda v: np.asarray(v, dtype=np.float64)  # noqa: E731
        partials = np.stack([c.numbers(10, 200) for _ in range(3)])
        x, gout = c.numbers(10, 200, 2.0), c.numbers(10, 200)
        gn = np.stack([c.numbers(10, 200) for _ in range(3)])
        leaves = {"partials": f64(partials), "residual": f64(x)}
        formula = c.formula()
        for k in ("pre", "post", "gate"):
            if formula[k] is not None:
                leaves[k] = formula[k]

        def loss(v):
            w = ref.norm_forward(v["partials"], v["residual"], **{**formula, **{k: v[k] for k in ("pre", "post", "gate") if k in v}})
            return (f64(gn).sum(0) * w["normed"][0]).sum() + (f64(gout) * w["residual_out"][0]).sum()

        source = c.rows_of(10, 200, 0).write_all(partials)
        grads = {n: c.rows_of(r, 200, 0, np.float32) for n, r in (("grad_source", 10), ("grad_residual", 10), ("grad_pre_weight", 1))}
        if post:
            grads["grad_post_weight"] = c.rows_of(1, 200, 0, np.float32)
        if gate:
            grads["grad_gate"] = c.rows_of(c.gates, 200, 0, np.float32)
        out, total = c.stream(), c.shared()
        rs.roc_shmem_norm_to_all(rs.NormArgs(source=source, residual=c.stream(x), residual_out=out, normed=c.rows_of(10, 200, 0),
                                             total=total, **c.fields))
        args = rs.NormGradArgs(grad_normed=c.rows_of(10, 200, 0).write_all(gn), grad_residual_out=c.stream(gout), residual_out=out,
                               total=total, **grads, **c.fields)
        work = rs.sym_array(max(1, rs.roc_shmem_norm_grad_work_bytes(args)), np.uint8)
        args.work = work.addr
        rs.roc_shmem_norm_to_all_grad(args)
        rs.synchronize()
        rng = np.random.default_rng(9)
        names = {"residual": "grad_residual", "pre": "grad_pre_weight", "post": "grad_post_weight", "gate": "grad_gate"}
        for leaf, value in leaves.items():
            direction = rng.standard_normal(value.shape)
            grad = f64(grads["grad_source" if leaf == "partials" else names[leaf]].read(2))
            if leaf in ("pre", "post"):
                grad = grad[0]
            want = differences(c, loss, leaves, leaf, direction)
            # kernels: a few hundred roundings of 2^-24 of the terms' sizes; differences: steps of 1e-3
            # extrapolated leave 1e-12 of the fifth derivative
            assert abs((grad * direction).sum() - want) <= 2e-5 * np.abs(grad * direction).sum() + 1e-8, leaf
