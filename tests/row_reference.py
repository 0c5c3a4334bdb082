"""Row collectives from their formulas in 64 bits, with the error that 32-bit arithmetic and one
rounding may make of each result.

A bound is  half a step of the result's type * |result|  +  2^-24 * K * A:  A adds up the magnitudes of
the terms that the result is made of (so that cancellation is allowed for), and K counts roundings: the
members' sum has P - 1, a sum over a row at most 38 (16 elements of a lane, 6 steps in a wave, 16 waves),
a root or an exponential 2, and no chain multiplies more than a dozen factors.  A row's mean is off by
relatively as much as its terms are, which the ratio of the terms' root mean squares allows for."""
import numpy as np

import oracle
import roc_shmem_amd as rs

U32 = 2.0 ** -24
HALF_STEP = {rs.BF16: 2.0 ** -8, rs.FLOAT: 2.0 ** -24}
TINY = 1e-37      # results below the smallest normal number may be 0


def to_type(dtype, values):
    """float array -> stored elements of `dtype`."""
    v = np.asarray(values, dtype=np.float32)
    return oracle.float_to_bf16(v).reshape(v.shape) if dtype == rs.BF16 else v


def from_type(dtype, stored):
    return (oracle.bf16_to_float(stored).reshape(stored.shape) if dtype == rs.BF16 else stored).astype(np.float64)


def check(name, dtype, got, want, error):
    got = from_type(dtype, got)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), name + ": NaN in other places"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), name + ": infinities"
    fine = np.isfinite(want)
    bound = HALF_STEP[dtype] * np.abs(want) * (1 + U32) + error + TINY
    off = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)) / np.where(fine, bound, 1), 0)
    at = np.unravel_index(np.argmax(off), off.shape) if off.size else None
    assert not off.size or off.max() <= 1, "%s: %.3g times the bound at %s: got %r, want %r" % (name, off.max(), at, got[at], want[at])


def rms(v):
    return np.sqrt(np.mean(v * v, axis=1, keepdims=True))


def gate_of(rows, rows_per_gate, gate):
    """The gate row of every row."""
    return gate[np.arange(rows) // (rows_per_gate or max(rows, 1))]


def norm_forward(partials, residual, pre, post, gate, *, has_post, rows_per_gate, eps, a, b, o):
    """{name: (value, error)} of normed, residual_out and total.  partials: [P, rows, cols]; pre, post,
    gate may be None."""
    rows, cols = residual.shape
    k = len(partials) + 64
    s, s_abs = partials.sum(0), np.abs(partials).sum(0)
    z, z_abs = s, s_abs
    if has_post:
        r = 1 / np.sqrt(np.mean(s * s, axis=1, keepdims=True) + eps)
        w = (o + post) if post is not None else np.ones(cols)
        w_abs = np.abs(o) + np.abs(post) if post is not None else np.ones(cols)
        z = s * r * w
        z_abs = (s_abs + np.abs(s) * rms(s_abs) * r) * r * w_abs
    if gate is not None:
        g = gate_of(rows, rows_per_gate, gate)
        z, z_abs = z * g, z_abs * np.abs(g)
    x = a * residual + b * z
    x_abs = np.abs(a * residual) + np.abs(b) * z_abs
    r = 1 / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + eps)
    w = (o + pre) if pre is not None else np.ones(cols)
    w_abs = np.abs(o) + np.abs(pre) if pre is not None else np.ones(cols)
    h = x * r * w
    h_abs = (x_abs + np.abs(x) * rms(x_abs) * r) * r * w_abs
    return {"normed": (h, k * U32 * h_abs), "residual_out": (x, k * U32 * x_abs), "total": (s, k * U32 * s_abs)}


def norm_backward(grad_normed, grad_out, x, total, pre, post, gate, *, has_post, rows_per_gate, eps, a, b, o):
    """{name: (value, error)} of the gradients; grad_normed [P, rows, cols] or None, grad_out or None."""
    rows, cols = grad_out.shape if grad_out is not None else grad_normed.shape[1:]
    k = (0 if grad_normed is None else len(grad_normed)) + 96
    got = {}
    d = grad_out if grad_out is not None else np.zeros((rows, cols))
    d_abs = np.abs(d)
    if grad_normed is not None:
        dh, dh_abs = grad_normed.sum(0), np.abs(grad_normed).sum(0)
        r = 1 / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + eps)
        n = x * r
        w = (o + pre) if pre is not None else np.ones(cols)
        w_abs = np.abs(o) + np.abs(pre) if pre is not None else np.ones(cols)
        t, t_abs = dh * w, dh_abs * w_abs
        d = d + r * (t - n * np.mean(t * n, axis=1, keepdims=True))
        d_abs = d_abs + r * (t_abs + np.abs(n) * np.mean(t_abs * np.abs(n), axis=1, keepdims=True))
        got["grad_pre_weight"] = (dh * n).sum(0), (k + rows) * U32 * (dh_abs * np.abs(n)).sum(0)
    got["grad_residual"] = a * d, k * U32 * np.abs(a) * d_abs
    f, f_abs = b * d, np.abs(b) * d_abs
    r1, u = 1.0, total
    if has_post:
        r1 = 1 / np.sqrt(np.mean(total * total, axis=1, keepdims=True) + eps)
        u = total * r1
    w = (o + post) if post is not None else np.ones(cols)
    w_abs = np.abs(o) + np.abs(post) if post is not None else np.ones(cols)
    if gate is not None:
        if total is not None:
            z, z_abs = (u * w, np.abs(u) * w_abs) if has_post else (u, np.abs(u))
            each, each_abs = f * z, f_abs * z_abs
            at = np.arange(rows) // (rows_per_gate or max(rows, 1))
            grad, grad_abs = np.zeros(gate.shape), np.zeros(gate.shape)
            np.add.at(grad, at, each)
            np.add.at(grad_abs, at, each_abs)
            got["grad_gate"] = grad, (k + rows) * U32 * grad_abs
        g = gate_of(rows, rows_per_gate, gate)
        f, f_abs = f * g, f_abs * np.abs(g)
    if has_post:
        got["grad_post_weight"] = (f * u).sum(0), (k + rows) * U32 * (f_abs * np.abs(u)).sum(0)
        q, q_abs = f * w, f_abs * w_abs
        f = r1 * (q - u * np.mean(q * u, axis=1, keepdims=True))
        f_abs = r1 * (q_abs + np.abs(u) * np.mean(q_abs * np.abs(u), axis=1, keepdims=True))
    got["grad_source"] = f, k * U32 * f_abs
    return got


def logprob_forward(logits, tokens, scale, top_k):
    """{name: (value, error)} of rows of logits over the whole vocabulary; ids have no error.

    A term exp(y - m) is off by 3 roundings of y - m (difference, product, the scale's own) and 2 of the
    exponential; adding V terms up takes at most V / 64 + 60 roundings (a lane's share and its
    rescalings, then the lanes and workgroups)."""
    rows, vocab = logits.shape
    with np.errstate(all="ignore"):
        y = logits * scale
        m = y.max(1, keepdims=True)
        empty = m == -np.inf
        e = np.exp(y - np.where(empty, 0, m))
        total = e.sum(1, keepdims=True)
        p = np.where(empty, 0, e / np.where(empty, 1, total))
        below = np.where(p > 0, y - m, 0)
        spread = -(p * below).sum(1, keepdims=True)            # E[m - y]
        log_l = np.log(total)
        lse = np.where(empty, -np.inf, m + log_l)
        entropy = np.where(empty, 0, log_l + spread)
        n = vocab / 64 + 60
        of_l = (n + 2 + 3 * spread) * U32                       # relative error of l
        of_w = (n + 4) * spread * U32 + 4 * U32 * (p * below * below).sum(1, keepdims=True) + spread * of_l
        fine = lambda v: np.where(np.isfinite(v), v, 0)  # noqa: E731
        got = {"lse": (lse[:, 0], fine(of_l + 3 * U32 * (np.abs(m) + np.abs(log_l)))[:, 0]),
               "entropy": (entropy[:, 0], fine(of_l + of_w + 3 * U32 * np.abs(log_l))[:, 0])}

        def logprobs(at):
            there = np.take_along_axis(y, at, 1)
            lp = np.where(empty, -np.inf, there - lse)
            return lp, fine(of_l + 3 * U32 * (np.abs(there - m) + np.abs(log_l)))

        if tokens is not None:
            lp, err = logprobs(np.maximum(tokens, 0)[:, None])
            lp = np.where(tokens < 0, 0, lp[:, 0])
            got["logprob"] = lp, np.where(tokens < 0, 0, err[:, 0])
        if top_k:
            ids = np.argsort(-logits, axis=1, kind="stable")[:, :top_k]
            got["top_ids"] = ids.astype(np.int32), 0
            got["top_logprobs"] = logprobs(ids)
    return got


def logprob_backward(logits, tokens, lse, entropy, scale, g_logprob, g_entropy, g_lse):
    """(value, error) of the gradient of the logits, from the lse and entropy given.  exp(lp) is off by 3
    roundings of lp and 2 of its own, the factor behind it by 6; and a probability below the smallest
    normal number, 2^-126, may be taken for 0, which leaves out 2^-126 times that factor."""
    rows, vocab = logits.shape
    col = lambda v: np.zeros((rows, 1)) if v is None else np.asarray(v, dtype=np.float64)[:, None]  # noqa: E731
    with np.errstate(all="ignore"):
        empty = col(lse) == -np.inf
        lp = np.where(empty, -np.inf, logits * scale - col(lse))
        p = np.exp(lp)
        gl = np.where((tokens >= 0)[:, None], col(g_logprob), 0) if tokens is not None else np.zeros((rows, 1))
        ge, gs, h = col(g_entropy), col(g_lse), col(entropy)
        inner = np.where(p == 0, 0, lp)
        d = p * (gs - gl - ge * (inner + h))
        factor = np.abs(gs) + np.abs(gl) + np.abs(ge) * (np.abs(inner) + np.abs(h))
        d_abs = p * factor
        if tokens is not None:
            hit = np.arange(vocab)[None, :] == tokens[:, None]
            d = d + np.where(hit, gl, 0)
            d_abs = d_abs + np.where(hit, np.abs(gl), 0)
        return d * scale, U32 * scale * d_abs * (14 + 3 * np.abs(inner)) + scale * 2.0 ** -126 * factor
