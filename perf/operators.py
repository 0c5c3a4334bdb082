"""What the row operators of a model spread over PEs cost: cases, inputs, plain forms and exact results.

Every PE (member) of a team holds a part of the model.  Four operators close the work that the
members did apart, each on whole rows of a batch:

  norm          the members' partial outputs of a block are summed; the sum goes through the norm
                behind the block, its gate and its scale into the residual stream, and the norm in
                front of the next block gives every member that block's input
  norm_grad     its backward pass: the members' partial gradients of the next block's input are
                summed, and every member gets the gradient of its partial output
  logprob       the vocabulary is split over the members: log probabilities of given tokens,
                entropies, normalisers and the likeliest alternatives of every row, on every member
  logprob_grad  its backward pass: every member's part of the gradient of the logits

Buffers have the member in front.  A row of the residual stream is held by its owner alone, the
member row // share with share = ceil(rows / members), at row % share; where `replicated` says so,
every member holds all of them.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "float": torch.float32}
MOST_PES = 8
HEAP_BYTES = 8 << 30
EPS = 1e-6
OUTPUTS = ("normed", "residual_out", "total", "grad_source", "grad_residual", "grad_post", "grad_pre",
           "grad_gate", "logprob", "entropy", "lse", "top_ids", "top_logprobs", "grad_logits")


# ---- the cases ------------------------------------------------------------------------------

def _norm(name, op, dtype, pes, rows, cols, post, gate, rows_per_gate=0, replicated=False, keep=False):
    """gate: "none", "one" (one row for all) or "rows" (one for every rows_per_gate rows); keep: the
    sum is kept for the backward pass."""
    c = {"op": op, "dtype": dtype, "pes": pes, "rows": rows, "cols": cols, "post": post, "gate": gate,
         "rows_per_gate": rows_per_gate, "replicated": replicated, "keep": keep}
    return dict(c, name=name) if name else c


def _logprob(name, op, dtype, pes, rows, vocab, top, scale=1.0, masked=0.0):
    """masked: the share of logits at minus infinity (a grammar, banned tokens)."""
    c = {"op": op, "dtype": dtype, "pes": pes, "rows": rows, "vocab": vocab, "top": top, "scale": scale,
         "masked": masked}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one request being answered, a token at a time: latency is all that counts
        _norm("norm, one token", "norm", "bf16", 8, 1, 8192, True, "none"),
        # a batch of requests being answered, the residual stream on every PE
        _norm("norm, a decode batch", "norm", "bf16", 4, 48, 5120, False, "one", replicated=True),
        # a long prompt, or a training batch whose sums are kept
        _norm("norm, a training batch", "norm", "bf16", 8, 8192, 4096, True, "one", keep=True),
        # a small model in full precision on a team that is no power of two, gates by sequence
        _norm("norm, odd sizes", "norm", "float", 3, 777, 2887, True, "rows", 100),
        # the backward pass of the training batch
        _norm("norm_grad, a training batch", "norm_grad", "bf16", 8, 8192, 4096, True, "one"),
        # a small model in full precision, gates by sequence, the residual stream on every PE
        _norm("norm_grad, odd sizes", "norm_grad", "float", 2, 301, 1111, True, "rows", 60, replicated=True),
        # one request being answered, with the alternatives that its client asked for
        _logprob("logprob, one token", "logprob", "bf16", 8, 1, 128000, 20, scale=1.25),
        # a batch of requests under grammars; the last PE's part of the vocabulary is shorter
        _logprob("logprob, a decode batch", "logprob", "float", 4, 64, 50257, 5, masked=0.3),
        # a long prompt being scored, with alternatives
        _logprob("logprob, a scored prompt", "logprob", "bf16", 8, 4096, 131072, 8),
        # a training batch: the loss alone
        _logprob("logprob, a training batch", "logprob", "bf16", 8, 4096, 131072, 0),
        # the backward pass of the training batch
        _logprob("logprob_grad, a training batch", "logprob_grad", "bf16", 8, 4096, 131072, 0),
        # reinforcement learning on short answers of a small model, entropy and normaliser in the loss
        _logprob("logprob_grad, odd sizes", "logprob_grad", "float", 2, 333, 32003, 0, scale=0.8, masked=0.1),
    ]


def _log_size(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "norm_grad", "logprob", "logprob_grad"))
    dtype = rng.choice(("bf16", "bf16", "float"))
    pes = rng.choice((1, 2, 3, 4, 5, 8, 8))
    rows = _log_size(rng, 1, 8192)
    if op.startswith("norm"):
        cols = _log_size(rng, 64, 16384)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        gate = rng.choice(("none", "one", "rows"))
        case = _norm(None, op, dtype, pes, rows, cols, rng.random() < 0.6, gate,
                     _log_size(rng, 1, rows) if gate == "rows" else 0, rng.random() < 0.4,
                     op == "norm" and rng.random() < 0.5)
    else:
        vocab = _log_size(rng, 1000, 200000)
        if rng.random() < 0.6:
            vocab = vocab // 128 * 128
        case = _logprob(None, op, dtype, pes, rows, vocab,
                        rng.choice((0, 0, 1, 5, 20)) if op == "logprob" else 0,
                        rng.choice((1.0, 1.0, 0.7, 1.6)), rng.choice((0.0, 0.0, 0.2, 0.8)))
    while work(case)["bytes"] > 5e8:
        case["rows"] //= 2
    if case.get("gate") == "rows":
        case["rows_per_gate"] = min(case["rows_per_gate"], case["rows"])
    return case


def _gates(case):
    if case["gate"] == "none":
        return 0
    return 1 if case["gate"] == "one" else -(-case["rows"] // case["rows_per_gate"])


def work(case):
    pes, rows, size = case["pes"], case["rows"], DTYPES[case["dtype"]].itemsize
    if case["op"].startswith("norm"):
        cols, gates = case["cols"], _gates(case)
        one = rows * cols * size
        held = pes if case["replicated"] else 1
        weights = (1 + case["post"] + gates) * cols * size
        if case["op"] == "norm":
            return {"bytes": one * (2 * pes + 1 + held + case["keep"]) + weights, "flops": rows * cols * (pes + 12)}
        kept = case["post"] or gates > 0
        grads = pes * (1 + case["post"] + gates) * cols * 4
        return {"bytes": one * (2 * pes + 2 + kept + held) + weights + grads, "flops": rows * cols * (pes + 30)}
    one = rows * case["vocab"] * size
    if case["op"] == "logprob":
        return {"bytes": one + rows * 8 + pes * rows * (12 + 8 * case["top"]), "flops": rows * case["vocab"] * 6}
    return {"bytes": 2 * one + rows * 28, "flops": rows * case["vocab"] * 10}


# ---- what a program has in hand before the call -------------------------------------------------

class _Job:
    """The PEs of the process, their symmetric heap as one tensor, and the teams in use."""

    def __init__(self):
        import roc_shmem_amd as rs
        torch.cuda.synchronize()
        rs.roc_shmem_init(MOST_PES, HEAP_BYTES, 4, 1024)
        base, nbytes, self.stride = rs.arena()
        view = type("Arena", (), {"__cuda_array_interface__": {
            "shape": (nbytes,), "typestr": "|u1", "data": (base, False), "version": 2}})
        self.rs, self.base, self.bytes, self.teams = rs, base, torch.as_tensor(view(), device="cuda"), {}

    def team(self, pes):
        if pes == MOST_PES:
            return self.rs.roc_shmem_team_world()
        if pes not in self.teams:
            self.teams[pes] = self.rs.roc_shmem_team_split_strided(self.rs.roc_shmem_team_world(), 0, 1, pes)[1]
        return self.teams[pes]

    def tensor(self, array, shape, dtype):
        """The copies of a symmetric array on the first shape[0] PEs."""
        each = torch.empty(shape[1:], dtype=dtype, device="meta").stride()
        return self.bytes.view(dtype).as_strided(shape, (self.stride // dtype.itemsize,) + each,
                                                 (array.addr - self.base) // dtype.itemsize)


class _Held:
    """The symmetric arrays of one state, given back with it."""

    def __init__(self, job):
        self.job, self.arrays = job, {}

    def buffer(self, name, shape, dtype):
        self.arrays[name] = self.job.rs.sym_array(math.prod(shape[1:]) * dtype.itemsize, "u1")
        return self.job.tensor(self.arrays[name], shape, dtype).zero_()

    def __del__(self):
        for a in self.arrays.values():
            a.free()


class _Plain:
    """The same buffers as tensors of torch's own."""

    def buffer(self, name, shape, dtype):
        return torch.zeros(shape, dtype=dtype, device="cuda")


_job = []


def _held():
    if own:
        if not _job:
            _job.append(_Job())
        return _Held(_job[0])
    return _Plain()


def _share(case):
    return -(-case["rows"] // case["pes"])


def _by_share(case, whole):
    """Rows laid out as the residual stream is held: on every member, or each on its owner."""
    if case["replicated"]:
        return whole.expand(case["pes"], *whole.shape)
    share, cols = _share(case), case["cols"]
    out = torch.zeros(case["pes"] * share, cols, dtype=whole.dtype, device=whole.device)
    out[: case["rows"]] = whole
    return out.view(case["pes"], share, cols)


def _norm_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pes, rows, cols, dtype = case["pes"], case["rows"], case["cols"], DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dtype)

    each = []
    for _ in range(pes):
        each.append(normal(rows, cols, scale=1.5 / math.sqrt(pes)))
    got = {"partials": torch.stack(each), "residual": normal(rows, cols, scale=2.0),
           "pre_weight": normal(cols, scale=0.2)}
    got["post_weight"] = normal(cols, scale=0.2) if case["post"] else None
    got["gate"] = normal(_gates(case), cols, scale=0.3, shift=0.8) if _gates(case) else None
    if case["op"] == "norm_grad":
        got["total"] = normal(rows, cols, scale=1.5) if case["post"] or got["gate"] is not None else None
        got["grad_residual_out"] = normal(rows, cols)
    return got


def _logprob_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    logits = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // vocab)
    for i in range(0, rows, step):
        part = torch.randn((min(step, rows - i), vocab), generator=g, device="cuda").mul_(2.5)
        if case["masked"]:
            banned = torch.rand(part.shape, generator=g, device="cuda") < case["masked"]
            part.masked_fill_(banned, -math.inf)
        logits[i : i + step] = part
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    at = torch.arange(rows, device="cuda")
    logits[at, tokens] = (torch.randn(rows, generator=g, device="cuda") * 2 + 7).to(dtype)  # text is mostly likely
    if rows > 1:
        tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.1, -1, tokens)  # padding
    got = {"logits": logits, "tokens": tokens}
    if case["op"] == "logprob_grad":
        got["lse"] = torch.empty(rows, device="cuda")
        got["entropy"] = torch.empty(rows, device="cuda")
        for i in range(0, rows, step):  # what the forward pass of the training step left
            y = logits[i : i + step].double() * case["scale"]
            lse = torch.logsumexp(y, 1)
            p = torch.exp(y - lse[:, None])
            got["lse"][i : i + step] = lse
            got["entropy"][i : i + step] = lse - torch.nan_to_num(p * y, nan=0.0).sum(1)
        for name in ("grad_logprob", "grad_entropy", "grad_lse"):
            got[name] = torch.randn(rows, generator=g, device="cuda") * (1.0 if name == "grad_logprob" else 0.05)
    return got


def prepare(case, seed):
    held, pes, rows, dtype = _held(), case["pes"], case["rows"], DTYPES[case["dtype"]]
    st = {"case": case, "held": held}

    def take(name, value):
        st[name] = None if value is None else held.buffer(name, value.shape, value.dtype).copy_(value)

    def room(name, *shape, dtype=dtype):
        st[name] = held.buffer(name, (pes,) + shape, dtype)

    everywhere = lambda v: None if v is None else v.expand(pes, *v.shape)  # noqa: E731
    if case["op"].startswith("norm"):
        cols, got = case["cols"], _norm_inputs(case, seed)
        by_share = lambda v: None if v is None else _by_share(case, v)  # noqa: E731
        mine = (rows if case["replicated"] else _share(case), cols)
        for name in ("pre_weight", "post_weight", "gate"):
            take(name, everywhere(got[name]))
        if case["op"] == "norm":
            take("source", got["partials"])
            take("residual", by_share(got["residual"]))
            room("normed", rows, cols)
            room("residual_out", *mine)
            if case["keep"]:
                room("total", _share(case), cols)
        else:
            take("grad_normed", got["partials"])
            take("residual_out", by_share(got["residual"]))
            take("total", None if got["total"] is None else _by_share(dict(case, replicated=False), got["total"]))
            take("grad_residual_out", by_share(got["grad_residual_out"]))
            room("grad_source", rows, cols)
            room("grad_residual", *mine)
            room("grad_pre", cols, dtype=torch.float32)
            if case["post"]:
                room("grad_post", cols, dtype=torch.float32)
            if _gates(case):
                room("grad_gate", _gates(case), cols, dtype=torch.float32)
    else:
        vocab, got = case["vocab"], _logprob_inputs(case, seed)
        shard = -(-vocab // pes)
        st["logits"] = held.buffer("logits", (pes, rows, shard), dtype)
        for m in range(pes):
            part = got["logits"][:, m * shard : (m + 1) * shard]
            st["logits"][m, :, : part.shape[1]] = part
        take("tokens", everywhere(got["tokens"]))
        if case["op"] == "logprob":
            for name in ("logprob", "entropy", "lse"):
                room(name, rows, dtype=torch.float32)
            if case["top"]:
                room("top_ids", rows, case["top"], dtype=torch.int32)
                room("top_logprobs", rows, case["top"], dtype=torch.float32)
        else:
            for name in ("lse", "entropy", "grad_logprob", "grad_entropy", "grad_lse"):
                take(name, everywhere(got[name]))
            room("grad_logits", rows, shard)
    st["written"] = [name for name in _written(case) if name in st]
    if own:
        st["call"] = _call(case, st)
    return st


def _written(case):
    """The names of an operator's outputs, in the order of OUTPUTS."""
    theirs = {"norm": OUTPUTS[:3], "norm_grad": OUTPUTS[3:8], "logprob": OUTPUTS[8:13], "logprob_grad": OUTPUTS[13:]}
    return theirs[case["op"]]


def _call(case, st):
    """The framework's call on a state: the operator and its arguments, kept by a program that makes it again."""
    job, a, dtype = st["held"].job, st["held"].arrays, case["dtype"]
    rs = job.rs
    code = rs.BF16 if dtype == "bf16" else rs.FLOAT
    if case["op"].startswith("norm"):
        flags = (rs.NORM_POST if case["post"] else 0) | (rs.NORM_REPLICATED if case["replicated"] else 0)
        numbers = dict(dtype=code, flags=flags, team=job.team(case["pes"]), rows=case["rows"], cols=case["cols"],
                       rows_per_gate=case["rows_per_gate"], eps=EPS, residual_scale=1.0, block_scale=0.5,
                       weight_offset=1.0, pre_weight=a["pre_weight"], post_weight=a.get("post_weight"),
                       gate=a.get("gate"), residual_out=a["residual_out"], total=a.get("total"))
        if case["op"] == "norm":
            args = rs.NormArgs(source=a["source"], residual=a["residual"], normed=a["normed"], **numbers)
            return rs.roc_shmem_norm_to_all, args
        args = rs.NormGradArgs(grad_normed=a["grad_normed"], grad_residual_out=a["grad_residual_out"],
                               grad_source=a["grad_source"], grad_residual=a["grad_residual"],
                               grad_pre_weight=a["grad_pre"], grad_post_weight=a.get("grad_post"),
                               grad_gate=a.get("grad_gate"), **numbers)
        st["held"].buffer("work", (1, max(1, rs.roc_shmem_norm_grad_work_bytes(args))), torch.uint8)
        args.work = a["work"].addr
        return rs.roc_shmem_norm_to_all_grad, args
    numbers = dict(dtype=code, team=job.team(case["pes"]), rows=case["rows"], vocab=case["vocab"],
                   scale=case["scale"], logits=a["logits"], tokens=a["tokens"], lse=a["lse"], entropy=a["entropy"])
    if case["op"] == "logprob":
        args = rs.LogprobArgs(top_k=case["top"], logprob=a["logprob"], top_ids=a.get("top_ids"),
                              top_logprobs=a.get("top_logprobs"), **numbers)
        st["held"].buffer("work", (1, max(1, rs.roc_shmem_logprob_work_bytes(args))), torch.uint8)
        st["held"].buffer("psync", (1, rs.ROC_SHMEM_REDUCE_SYNC_SIZE), torch.int64)
        args.work, args.pSync = a["work"].addr, a["psync"].addr
        return rs.roc_shmem_logprob_to_all, args
    args = rs.LogprobGradArgs(grad_logprob=a["grad_logprob"], grad_entropy=a["grad_entropy"],
                              grad_lse=a["grad_lse"], grad_logits=a["grad_logits"], **numbers)
    return rs.roc_shmem_logprob_to_all_grad, args


# ---- one pass ---------------------------------------------------------------------------------------

def run(state):
    if own:
        call, args = state["call"]
        call(args, torch.cuda.current_stream().cuda_stream)
    else:
        {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "logprob": _plain_logprob,
         "logprob_grad": _plain_logprob_grad}[state["case"]["op"]](state)
    return {name: state[name] for name in state["written"]}


def _rows_of(case, held):
    """The rows of the residual stream, as one matrix, from the members that hold them."""
    return held[0] if case["replicated"] else held.reshape(-1, case["cols"])[: case["rows"]]


def _leave(case, held, rows):
    """Rows of the residual stream to the members that hold them."""
    if case["replicated"]:
        held.copy_(rows.expand(held.shape))
    else:
        held.view(-1, case["cols"])[: case["rows"]] = rows.to(held.dtype)


def _gate_rows(case, gate):
    """The gate of every row."""
    g = gate[0].float()
    if case["gate"] == "one":
        return g
    return g.repeat_interleave(case["rows_per_gate"], 0)[: case["rows"]]


def _plain_norm(st):
    case = st["case"]
    total = st["source"].float().sum(0)
    z = total
    if case["post"]:
        z = total * torch.rsqrt((total * total).mean(1, keepdim=True) + EPS) * (1.0 + st["post_weight"][0].float())
    if st["gate"] is not None:
        z = z * _gate_rows(case, st["gate"])
    x = _rows_of(case, st["residual"]).float() + 0.5 * z
    h = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * (1.0 + st["pre_weight"][0].float())
    st["normed"].copy_(h.expand(st["normed"].shape))
    _leave(case, st["residual_out"], x)
    if case["keep"]:
        _leave(dict(case, replicated=False), st["total"], total)


def _plain_norm_grad(st):
    case = st["case"]
    dh = st["grad_normed"].float().sum(0)
    x = _rows_of(case, st["residual_out"]).float()
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    n = x * r
    t = dh * (1.0 + st["pre_weight"][0].float())
    dx = _rows_of(case, st["grad_residual_out"]).float() + r * (t - n * (t * n).mean(1, keepdim=True))
    st["grad_pre"].copy_((dh * n).sum(0).expand(st["grad_pre"].shape))
    _leave(case, st["grad_residual"], dx)
    dz = 0.5 * dx
    if st["total"] is not None:
        s = _rows_of(dict(case, replicated=False), st["total"]).float()
    if case["post"]:
        r = torch.rsqrt((s * s).mean(1, keepdim=True) + EPS)
        u = s * r
        w = 1.0 + st["post_weight"][0].float()
    if st["gate"] is not None:
        z = u * w if case["post"] else s
        each = dz * z
        if case["gate"] == "rows":
            short = _gates(case) * case["rows_per_gate"] - case["rows"]
            each = torch.cat([each, each.new_zeros(short, case["cols"])])
        st["grad_gate"].copy_(each.view(_gates(case), -1, case["cols"]).sum(1).expand(st["grad_gate"].shape))
        dz = dz * _gate_rows(case, st["gate"])
    if case["post"]:
        st["grad_post"].copy_((dz * u).sum(0).expand(st["grad_post"].shape))
        q = dz * w
        dz = r * (q - u * (q * u).mean(1, keepdim=True))
    st["grad_source"].copy_(dz.expand(st["grad_source"].shape))


def _whole_rows(case, held):
    """Rows over the whole vocabulary from the members' parts."""
    return held.transpose(0, 1).reshape(case["rows"], -1)[:, : case["vocab"]].float()


def _plain_logprob(st):
    case = st["case"]
    x = _whole_rows(case, st["logits"])
    y = x * case["scale"]
    m = y.max(1, keepdim=True).values
    e = torch.exp(y - m)
    total = e.sum(1)
    lse = m[:, 0] + torch.log(total)
    spread = torch.where(e > 0, e * (y - m), 0.0).sum(1)
    token = st["tokens"][0]
    taken = y.gather(1, token.clamp(min=0)[:, None])[:, 0] - lse
    st["lse"].copy_(lse.expand(st["lse"].shape))
    st["entropy"].copy_((torch.log(total) - spread / total).expand(st["entropy"].shape))
    st["logprob"].copy_(torch.where(token < 0, 0.0, taken).expand(st["logprob"].shape))
    if case["top"]:
        bits = (x + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()  # grows with the value
        key = (order << 20) + ((1 << 20) - 1 - torch.arange(case["vocab"], device=x.device))  # ties: the lowest first
        ids = (1 << 20) - 1 - (torch.topk(key, case["top"], 1).values & ((1 << 20) - 1))
        st["top_ids"].copy_(ids.expand(st["top_ids"].shape))
        st["top_logprobs"].copy_((y.gather(1, ids) - lse[:, None]).expand(st["top_logprobs"].shape))


def _plain_logprob_grad(st):
    case = st["case"]
    y = _whole_rows(case, st["logits"]) * case["scale"]
    lp = y - st["lse"][0][:, None]
    p = torch.exp(lp)
    token = st["tokens"][0]
    of_token = torch.where(token < 0, 0.0, st["grad_logprob"][0])
    d = p * (st["grad_lse"][0] - of_token)[:, None]
    d -= st["grad_entropy"][0][:, None] * torch.where(p > 0, p * (lp + st["entropy"][0][:, None]), 0.0)
    d.scatter_add_(1, token.clamp(min=0)[:, None], of_token[:, None])
    d *= case["scale"]
    pes, rows, shard = st["grad_logits"].shape
    short = pes * shard - case["vocab"]
    d = torch.cat([d, d.new_zeros(rows, short)], 1) if short else d
    st["grad_logits"].copy_(d.view(rows, pes, shard).transpose(0, 1))


# ---- the definitions, in 64 bits ----------------------------------------------------------------------

def _block_end(case, total, residual, post_weight, gate, pre_weight):
    """(normed, residual_out) of rows, from the definition."""
    cols = total.shape[1]

    def rms_norm(v, weight):
        return v / torch.sqrt(torch.linalg.vector_norm(v, dim=1, keepdim=True) ** 2 / cols + EPS) * (weight + 1)

    out = rms_norm(total, post_weight) if case["post"] else total
    if gate is not None:
        at = torch.arange(case["rows"], device=total.device) // (case["rows_per_gate"] or case["rows"])
        out = out * gate[at]
    stream = residual + out / 2
    return rms_norm(stream, pre_weight), stream


def _exact_norm(case, seed):
    v = {k: None if t is None else t.double() for k, t in _norm_inputs(case, seed).items()}
    weights = [v["post_weight"], v["gate"], v["pre_weight"]]
    pes = case["pes"]
    if case["op"] == "norm":
        total = v["partials"].sum(0)
        h, x = _block_end(case, total, v["residual"], *weights)
        got = {"normed": h.expand(pes, *h.shape), "residual_out": _by_share(case, x)}
        if case["keep"]:
            got["total"] = _by_share(dict(case, replicated=False), total)
        return got
    # The gradients by automatic differentiation, in two steps, since what the forward pass kept is
    # given here: from normed to the residual stream, and from there back through the block's end.
    stream = v["residual"].requires_grad_()
    pre = v["pre_weight"].requires_grad_()
    bare = dict(case, post=False, gate="none", rows_per_gate=0)
    h, _ = _block_end(bare, torch.zeros_like(stream), stream, None, None, pre)
    into, grad_pre = torch.autograd.grad(h, (stream, pre), v["partials"].sum(0))
    dx = into + v["grad_residual_out"]
    got = {"grad_residual": _by_share(case, dx), "grad_pre": grad_pre.expand(pes, -1)}
    if v["total"] is None:
        got["grad_source"] = (dx / 2).expand(pes, *dx.shape)
        return got
    leaves = {"grad_source": v["total"], "grad_post": v["post_weight"], "grad_gate": v["gate"]}
    leaves = {k: t.requires_grad_() for k, t in leaves.items() if t is not None}
    _, x = _block_end(case, v["total"], torch.zeros_like(dx), v["post_weight"], v["gate"], pre.detach())
    for name, grad in zip(leaves, torch.autograd.grad(x, list(leaves.values()), dx)):
        got[name] = grad.expand(pes, *grad.shape)
    return got


def _exact_logprob(case, seed):
    v = _logprob_inputs(case, seed)
    pes, rows, vocab = case["pes"], case["rows"], case["vocab"]
    got = {name: [] for name in _written(case)}
    step = max(1, (1 << 25) // vocab)
    for i in range(0, rows, step):
        x = v["logits"][i : i + step].double()
        token = v["tokens"][i : i + step]
        lp = torch.log_softmax(x * case["scale"], 1)
        p = lp.exp()
        at = token.clamp(min=0)[:, None]
        if case["op"] == "logprob":
            got["lse"].append(torch.logsumexp(x * case["scale"], 1))
            got["entropy"].append(torch.special.entr(p).sum(1))
            got["logprob"].append(lp.gather(1, at)[:, 0] * (token >= 0))
            if case["top"]:
                ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : case["top"]]
                got["top_ids"].append(ids.int())
                got["top_logprobs"].append(lp.gather(1, ids))
        else:
            # d logprob = 1[token] - p,  d lse = p,  d entropy = -p (log p + entropy), each times the scale
            g = {k: v[k][i : i + step].double()[:, None] for k in ("grad_logprob", "grad_entropy", "grad_lse")}
            hit = torch.zeros_like(p).scatter_(1, at, 1.0) * (token >= 0)[:, None]
            entropy = torch.special.entr(p).sum(1, keepdim=True)
            d = g["grad_logprob"] * (hit - p * (token >= 0)[:, None]) + g["grad_lse"] * p
            d = (d + g["grad_entropy"] * (torch.special.entr(p) - p * entropy)) * case["scale"]
            got["grad_logits"].append(d)
    got = {k: torch.cat(t) for k, t in got.items() if t}
    if case["op"] == "logprob":
        return {k: t.expand(pes, *t.shape) for k, t in got.items()}
    shard = -(-vocab // pes)
    whole = torch.nn.functional.pad(got["grad_logits"], (0, pes * shard - vocab))
    return {"grad_logits": whole.view(rows, pes, shard).transpose(0, 1)}


def exact(case, seed):
    return _exact_norm(case, seed) if case["op"].startswith("norm") else _exact_logprob(case, seed)
