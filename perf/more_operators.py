"""What stands around a layer of experts in a block of a model, as cases that
can be timed: the norms before and after the block with its gate and its residual
scale, dense matrix products in 16 and 32 bits with bias, activation and residual
(router, shared expert), and the loss that balances the experts with their counts,
each with its gradient.

A case is a dict of plain values:

    name     listed cases only
    op       join | dense | balance
    dtype    f32 | bf16 | f16: the block's numbers; the products' operands; the
             router's logits
    grad     whether the pass goes backward too

    join     rows, width, kind (rms | layer), bias, wide (the residual stream and
             the norms' weights are in 32 bits), block. With `block` one pass
             takes a block's output y into the stream, gated per `gate` (none |
             channel | row | all) by `gate_by` (none | sigmoid | tanh | silu), behind
             a norm of its own with `after`, and normalises the new stream for
             the next block; without, it is the first block's norm alone.
    dense    rows, cols, depth, bias, activation (none | relu | silu | gelu |
             gelu_tanh), residual, wide (residual and result in 32 bits). With
             `grad` also the gradients of the activations, the weights and the bias.
    balance  tokens, experts, topk, score (softmax | sigmoid), sequences (0: all
             tokens are one), padded (tokens behind the last sequence, whose
             logits are all masked), masked (experts that no token may choose),
             z (the weight of the squared log-sum-exp). One pass: loss, counts
             and shares by sequence and expert; with `grad` the logits' gradient.

`run` computes them in elementary torch operations, or, where `own` is true,
with the package's operators.
"""
import math

import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-5
SCALE, CARRY = 0.75, 0.96875       # of a block's output, of the stream that it is added to

#: Most rows of a drawn case, and most multiplications and additions (the largest listed ones'; in 32 bits the matrix
#: units have a sixteenth of the rate).
MOST_ROWS = {"join": 16384, "dense": 8192, "balance": 65536}
MOST_FLOPS = 6 * 8192 * 8192 * 4096


# ---- the cases -----------------------------------------------------------------
def _join(rows, width, kind="rms", bias=False, wide=False, block=True, after=True, gate="none", gate_by="none", dtype="bf16",
          grad=False):
    return {"op": "join", "rows": rows, "width": width, "kind": kind, "bias": bias, "wide": wide, "block": block, "after": after,
            "gate": gate, "gate_by": gate_by, "dtype": dtype, "grad": grad}


def _dense(rows, cols, depth, bias=False, activation="none", residual=False, wide=False, dtype="bf16", grad=False):
    return {"op": "dense", "rows": rows, "cols": cols, "depth": depth, "bias": bias, "activation": activation, "residual": residual,
            "wide": wide, "dtype": dtype, "grad": grad}


def _balance(tokens, experts, topk, score="softmax", sequences=0, padded=0, masked=0, z=0.0, dtype="f32", grad=False):
    return {"op": "balance", "tokens": tokens, "experts": experts, "topk": topk, "score": score, "sequences": sequences,
            "padded": padded, "masked": masked, "z": z, "dtype": dtype, "grad": grad}


def listed():
    cases = {
        # a sequence answers a token at a time, everything between two blocks at once: latency
        "join_1": _join(1, 4096, gate="channel"),
        # a prompt of ordinary length, no size a multiple of anything, gated number by number
        "join_1999_odd": _join(1999, 2501, "layer", bias=True, gate="all", gate_by="sigmoid", dtype="f16"),
        # a training step's tokens, forward and backward, a 16-bit stream
        "join_16384_training": _join(16384, 4096, gate="channel", grad=True),
        # the same of a large layer with its stream in 32 bits, a gate for each token
        "join_8192_wide_training": _join(8192, 8192, wide=True, gate="row", gate_by="tanh", grad=True),
        # one token through one projection: the weights are what is read
        "dense_1": _dense(1, 4096, 4096, bias=True, activation="silu"),
        # a few sequences answering together, no size a multiple of a tile
        "dense_50_odd": _dense(50, 5001, 2500, bias=True, activation="gelu", residual=True, dtype="f16"),
        # the router's logits in 32 bits
        "dense_4096_router": _dense(4096, 256, 4096, dtype="f32"),
        # a prompt of ordinary length, into a stream in 32 bits
        "dense_2048": _dense(2048, 4096, 4096, residual=True, wide=True),
        # a training step of a large layer, forward and all gradients
        "dense_8192_training": _dense(8192, 8192, 4096, bias=True, activation="silu", grad=True),
        # a few sequences' tokens: latency
        "balance_8": _balance(8, 64, 6),
        # a training step's tokens on one rank, balanced in each of its sequences, logits as a bf16 product left them
        "balance_4099_sequences_training": _balance(4099, 64, 6, sequences=9, padded=37, masked=3, z=1e-3, dtype="bf16", grad=True),
        # the largest batch: every rank's tokens
        "balance_65536_training": _balance(65536, 256, 8, score="sigmoid", grad=True),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _between(rng, least, most):
    """A whole number, its logarithm spread evenly; every second one odd or ragged as it falls,
    the others multiples of 16 as layers have them."""
    n = round(math.exp(rng.uniform(math.log(least), math.log(most))))
    if n >= 64 and rng.random() < 0.5:
        n = n // 16 * 16
    return max(least, min(most, n))


def draw(rng):
    op = rng.choice(("join", "join", "dense", "dense", "balance"))
    rows = _between(rng, 1, MOST_ROWS[op])
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    grad = rng.random() < 0.5
    if op == "join":
        gate = rng.choice(("none", "channel", "row", "all"))
        block = rng.random() < 0.75
        return _join(rows, _between(rng, 64, 8192), rng.choice(("rms", "rms", "layer")), rng.random() < 0.3, rng.random() < 0.4, block,
                     rng.random() < 0.6, gate if block else "none", rng.choice(("none", "sigmoid", "tanh", "silu")) if block and gate != "none" else "none",
                     dtype, grad)
    if op == "balance":
        experts = _between(rng, 4, 512)
        masked = rng.randrange(experts // 4 + 1) if rng.random() < 0.3 else 0
        return _balance(rows, experts, rng.randint(1, min(16, experts)), rng.choice(("softmax", "sigmoid")),
                        _between(rng, 1, 64) if rng.random() < 0.5 else 0, rng.randrange(rows // 8 + 1) if rng.random() < 0.5 else 0,
                        masked, rng.choice((0.0, 1e-3)), dtype, grad)
    cols, depth = _between(rng, 64, 8192), _between(rng, 64, 8192)
    most = MOST_FLOPS // ((16 if dtype == "f32" else 1) * (6 if grad else 2) * cols * depth)
    return _dense(max(1, min(rows, most)), cols, depth, rng.random() < 0.5, rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")),
                  rng.random() < 0.5, rng.random() < 0.3, dtype, grad)


# ---- what a program has in hand ------------------------------------------------
def _activations(g, rows, depth, dtype):
    """Normal numbers, some channels much larger than the others, as layers' outputs have them."""
    x = torch.randn(rows, depth, generator=g, device="cuda")
    return (x * (torch.rand(depth, generator=g, device="cuda") * 4 - 2).exp()).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    dtype = DTYPE[case["dtype"]]
    s = {"case": case}
    if case["op"] == "join":
        n, c = case["rows"], case["width"]
        stream = torch.float32 if case["wide"] else dtype
        norm = lambda: {"weight": (1 + 0.1 * rand(c)).to(stream), "bias": (0.1 * rand(c)).to(stream) if case["bias"] else None}  # noqa: E731
        s["stream"] = _activations(g, n, c, stream)
        s["before"] = norm()
        s["after"] = norm() if case["block"] and case["after"] else None
        s["y"] = _activations(g, n, c, dtype) if case["block"] else None
        shape = {"none": None, "channel": (c,), "row": (n, 1), "all": (n, c)}[case["gate"]]
        s["gate"] = rand(*shape).to(dtype) if shape else None
        if case["grad"]:
            s["d_stream"] = rand(n, c).to(stream) if case["block"] else None
            s["d_next"] = rand(n, c).to(dtype)
        return s
    if case["op"] == "dense":
        m, n, k = case["rows"], case["cols"], case["depth"]
        out = torch.float32 if case["wide"] else dtype
        s["x"] = _activations(g, m, k, dtype)
        s["w"] = (rand(n, k) * k ** -0.5).to(dtype)
        s["bias"] = (0.1 * rand(n)).to(dtype) if case["bias"] else None
        s["residual"] = rand(m, n).to(out) if case["residual"] else None
        s["d_out"] = rand(m, n).to(out) if case["grad"] else None
        return s
    t, e, k = case["tokens"], case["experts"], case["topk"]
    logits = rand(t, e) * 1.5 + rand(e) * 0.5
    logits[:, torch.randperm(e, generator=g, device="cuda")[:case["masked"]]] = -math.inf
    logits[t - case["padded"]:] = -math.inf
    s["logits"] = logits.to(dtype)
    found = s["logits"].float().sort(dim=-1, descending=True, stable=True)
    s["experts"] = torch.where(found.values[:, :k] == -math.inf, -1, found.indices[:, :k]).to(torch.int32).contiguous()
    s["offsets"] = None
    if case["sequences"]:       # some of them may be empty
        cuts = torch.randint(0, t - case["padded"] + 1, (case["sequences"] - 1,), generator=g, device="cuda").sort().values
        end = torch.tensor([t - case["padded"]], device="cuda")
        s["offsets"] = torch.cat([end * 0, cuts, end]).to(torch.int32)
    s["d_loss"] = torch.rand((), generator=g, device="cuda") + 0.5 if case["grad"] else None
    return s


# ---- the operators in their plain form -----------------------------------------
def _plain_norm(x, norm, kind):
    """(what is normalised, the reciprocal root of its mean square, the norm of x), in 32 bits."""
    centred = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    q = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xh = centred * q
    y = xh * norm["weight"].float()
    return xh, q, y + norm["bias"].float() if norm["bias"] is not None else y


def _plain_norm_grad(d, xh, q, norm, kind):
    """The gradients of x, of the weight and of the bias."""
    dw = d * norm["weight"].float()
    dx = dw - xh * (dw * xh).mean(-1, keepdim=True)
    if kind == "layer":
        dx = dx - dw.mean(-1, keepdim=True)
    return dx * q, (d * xh).sum(0), d.sum(0) if norm["bias"] is not None else None


def _gated(gate, by):
    """The gate and its slope."""
    if by == "none":
        return gate, torch.ones_like(gate)
    if by == "tanh":
        a = torch.tanh(gate)
        return a, 1 - a * a
    a = 1 / (1 + torch.exp(-gate))
    return (a, a * (1 - a)) if by == "sigmoid" else (gate * a, a * (1 + gate * (1 - a)))


def _typed(v, like):
    return None if v is None else v.to(like.dtype)


def _plain_join(s):
    c = s["case"]
    kind, stream, before, after = c["kind"], s["stream"], s["before"], s["after"]
    dtype = DTYPE[c["dtype"]]
    if not c["block"]:
        xh, q, h = _plain_norm(stream.float(), before, kind)
        out = {"next": h.to(dtype)}
        if c["grad"]:
            dx, dw, db = _plain_norm_grad(s["d_next"].float(), xh, q, before, kind)
            out.update(d_stream=dx.to(stream.dtype), d_before_weight=_typed(dw, stream), d_before_bias=_typed(db, stream))
        return out
    u = y = s["y"].float()
    if after:
        yh, yq, u = _plain_norm(y, after, kind)
    added, gate = u, None
    if s["gate"] is not None:
        gate, slope = _gated(s["gate"].float(), c["gate_by"])
        added = u * gate
    r = (CARRY * stream.float() + SCALE * added).to(stream.dtype)
    rh, rq, h = _plain_norm(r.float(), before, kind)
    out = {"stream": r, "next": h.to(dtype)}
    if c["grad"]:
        dr, dw, db = _plain_norm_grad(s["d_next"].float(), rh, rq, before, kind)
        d = s["d_stream"].float() + dr
        out.update(d_stream=(CARRY * d).to(stream.dtype), d_before_weight=_typed(dw, stream), d_before_bias=_typed(db, stream))
        du = SCALE * d
        if gate is not None:
            dg = du * u
            dg = dg.sum(0) if c["gate"] == "channel" else dg.sum(1, keepdim=True) if c["gate"] == "row" else dg
            out["d_gate"] = (dg * slope).to(dtype)
            du = du * gate
        if after:
            du, dw, db = _plain_norm_grad(du, yh, yq, after, kind)
            out.update(d_after_weight=_typed(dw, stream), d_after_bias=_typed(db, stream))
        out["d_y"] = du.to(dtype)
    return out


def _activated(z, name):
    """The activation and its slope."""
    if name == "relu":
        return torch.where(z > 0, z, 0), (z > 0).float()
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        root = (2 / math.pi) ** 0.5
        t = torch.tanh(root * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * root * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _plain_dense(s):
    c = s["case"]
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if c["bias"]:
        z = z + s["bias"].float()
    a, slope = _activated(z, c["activation"])
    out = s["residual"].float() + a if c["residual"] else a
    result = {"out": out.to(torch.float32 if c["wide"] else dtype)}
    if c["grad"]:
        dz = s["d_out"].float() * slope
        result.update(d_x=(dz @ w).to(dtype), d_w=(dz.t() @ x).to(dtype))
        if c["bias"]:
            result["d_bias"] = dz.sum(0).to(dtype)
    return result


def _sequence_of(s):
    """(tokens,) the sequence of each token, as many as there are for a token that is in none; and where each begins, and the end."""
    t, offsets = s["case"]["tokens"], s["offsets"]
    if offsets is None:
        return torch.zeros(t, dtype=torch.long, device="cuda"), torch.arange(2, device="cuda") * t
    return torch.searchsorted(offsets[1:].long().contiguous(), torch.arange(t, device="cuda"), right=True), offsets.long()


def _sums(v, ends):
    """The sum of each sequence's rows of v, in 64 bits: they are over many tokens."""
    if ends.numel() == 2:
        upto = torch.arange(v.shape[0], device=v.device)[:, None]
        return torch.where((upto >= ends[0]) & (upto < ends[1]), v, 0).sum(0, keepdim=True, dtype=torch.float64)
    upto = torch.cat([torch.zeros(1, v.shape[1], dtype=torch.float64, device=v.device), v.double().cumsum(0)])
    return upto[ends[1:]] - upto[ends[:-1]]


def _plain_balance(s):
    c = s["case"]
    x, e = s["logits"].float(), c["experts"]
    minus = torch.tensor(-math.inf, device=x.device)
    of, ends = _sequence_of(s)
    n = ends.numel() - 1
    there = (x != minus).any(-1) & (of < n)
    top = torch.where(there, x.amax(-1), 0)[:, None]
    power = torch.exp(x - top)
    lse = torch.where(there, top[:, 0] + torch.log(torch.where(there, power.sum(-1), 1)), 0)
    score = 1 / (1 + torch.exp(-x)) if c["score"] == "sigmoid" else power
    p = torch.where(there[:, None], score, 0) / torch.where(there, score.sum(-1), 1)[:, None]
    by_sequence, tokens = _sums(p, ends), _sums(there[:, None], ends)
    chosen = s["experts"].long()
    key = torch.where((chosen >= 0) & (of < n)[:, None], of[:, None] * e + chosen, n * e)
    counts = torch.bincount(key.reshape(-1), minlength=n * e + 1)[:n * e].view(n, e)
    some = tokens.clamp_min(1)
    sequences = (tokens > 0).sum().clamp_min(1)
    shares = by_sequence / some
    often = counts * e / (c["topk"] * some)
    every = tokens.sum().clamp_min(1)
    loss = (often * shares).sum() / sequences + c["z"] * lse.double().square().sum() / every
    out = {"loss": loss.float(), "counts": counts.to(torch.int32), "shares": shares.float()}
    if c["grad"]:
        d = s["d_loss"].double()
        a = torch.cat([d * often / (sequences * some), torch.zeros(1, e, dtype=torch.float64, device=x.device)]).float()[of]
        slope = p if c["score"] == "softmax" else p * (1 / (1 + torch.exp(x)))
        dx = slope * (a - (p * a).sum(-1, keepdim=True))
        if c["z"]:
            dx = dx + (2 * c["z"] * d / every).float() * lse[:, None] * torch.where(there[:, None], power, 0) / torch.where(there, power.sum(-1), 1)[:, None]
        out["d_logits"] = torch.where(there[:, None] & (x != minus), dx, 0).to(s["logits"].dtype)
    return out


# ---- the package's operators ---------------------------------------------------
def _own_join(s):
    from mintccl_amd.norms import Norm, join, join_grad, norm, norm_grad
    c = s["case"]
    dtype = DTYPE[c["dtype"]]
    described = lambda n: None if n is None else Norm(n["weight"], n["bias"], c["kind"], EPS)  # noqa: E731
    before, after = described(s["before"]), described(s["after"])
    if not c["block"]:
        out = {"next": norm(s["stream"], before, dtype=dtype)}
        if c["grad"]:
            d = norm_grad(s["d_next"], s["stream"], before)
            out.update(d_stream=d.x, d_before_weight=d.weight, d_before_bias=d.bias)
        return out
    options = {"after": after, "gate": s["gate"], "gate_by": None if c["gate_by"] == "none" else c["gate_by"], "scale": SCALE,
               "carry": CARRY, "before": before}
    stream, h = join(s["stream"], s["y"], **options)
    out = {"stream": stream, "next": h}
    if c["grad"]:
        d = join_grad(s["d_stream"], s["d_next"], stream, s["y"], **options)
        out.update(d_stream=d.stream, d_before_weight=d.before_weight, d_before_bias=d.before_bias)
        if s["gate"] is not None:
            out["d_gate"] = d.gate
        if after:
            out.update(d_after_weight=d.after_weight, d_after_bias=d.after_bias)
        out["d_y"] = d.y
    return out


def _own_dense(s):
    from mintccl_amd.dense import activation_grad, input_grad, product, weight_grad
    c = s["case"]
    activation = None if c["activation"] == "none" else c["activation"]
    dtype = torch.float32 if c["wide"] else s["x"].dtype
    options = {"bias": s["bias"], "activation": activation, "residual": s["residual"], "dtype": dtype}
    if not c["grad"]:
        return {"out": product(s["x"], s["w"], **options)}
    out, z = product(s["x"], s["w"], keep=True, **options)
    dz, d_bias = activation_grad(s["d_out"], z, activation, bias=c["bias"], dtype=s["x"].dtype)
    result = {"out": out, "d_x": input_grad(dz, s["w"]), "d_w": weight_grad(dz, s["x"])}
    if c["bias"]:
        result["d_bias"] = d_bias
    return result


def _own_balance(s):
    from mintccl_amd.routing import balance, balance_grad
    c = s["case"]
    options = {"score": c["score"], "offsets": s["offsets"], "z": c["z"]}
    found = balance(s["logits"], s["experts"], **options)
    out = {"loss": found.loss, "counts": found.counts, "shares": found.shares}
    if c["grad"]:
        out["d_logits"] = balance_grad(s["d_loss"], s["logits"], s["experts"], found, **options)
    return out


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


# ---- the definition in 64 bits -------------------------------------------------
def _leaf(v):
    return None if v is None else v.detach().double().requires_grad_()


def _gradients(total, leaves):
    """{name: the gradient of `total` by that leaf}, of the leaves that there are."""
    names = [n for n, v in leaves.items() if v is not None]
    return dict(zip(names, torch.autograd.grad(total, [leaves[n] for n in names])))


def _exact_norm(x, weight, bias, kind):
    if kind == "layer":
        y = torch.nn.functional.layer_norm(x, x.shape[-1:], None, None, EPS)
    else:
        y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
    y = y * weight
    return y if bias is None else y + bias


def _exact_join(s):
    c = s["case"]
    none = {"weight": None, "bias": None}
    before, after = s["before"], s["after"] or none
    v = {"d_stream": _leaf(s["stream"]), "d_y": _leaf(s["y"]), "d_gate": _leaf(s["gate"]),
         "d_before_weight": _leaf(before["weight"]), "d_before_bias": _leaf(before["bias"]),
         "d_after_weight": _leaf(after["weight"]), "d_after_bias": _leaf(after["bias"])}
    r, out, total = v["d_stream"], {}, 0.0
    if c["block"]:
        u = v["d_y"]
        if s["after"]:
            u = _exact_norm(u, v["d_after_weight"], v["d_after_bias"], c["kind"])
        if s["gate"] is not None:
            by = {"none": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh, "silu": torch.nn.functional.silu}[c["gate_by"]]
            u = by(v["d_gate"]) * u
        r = CARRY * r + SCALE * u
        out["stream"] = r.detach()
        if c["grad"]:
            total = (r * s["d_stream"].double()).sum()
    h = _exact_norm(r, v["d_before_weight"], v["d_before_bias"], c["kind"])
    out["next"] = h.detach()
    if c["grad"]:
        total = total + (h * s["d_next"].double()).sum()
        found = _gradients(total, v)
        names = ["d_stream", "d_before_weight", "d_before_bias"]
        if c["block"]:
            names += ["d_gate"] * (s["gate"] is not None) + ["d_after_weight", "d_after_bias"] * (s["after"] is not None) + ["d_y"]
        out.update({n: found.get(n) for n in names})
    return out


def _exact_dense(s):
    c = s["case"]
    F = torch.nn.functional
    act = {"none": lambda t: t, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[c["activation"]]
    x, w = s["x"].double(), s["w"].double()
    z = (F.linear(x, w, s["bias"].double()) if c["bias"] else x.mm(w.T)).requires_grad_(c["grad"])
    a = act(z)
    out = {"out": (a + s["residual"].double() if c["residual"] else a).detach()}
    if c["grad"]:
        dz, = torch.autograd.grad(a, z, s["d_out"].double())
        out.update(d_x=dz.mm(w), d_w=dz.T.mm(x))
        if c["bias"]:
            out["d_bias"] = dz.sum(0)
    return out


def _exact_balance(s):
    c = s["case"]
    t, e = c["tokens"], c["experts"]
    ends = [0, t] if s["offsets"] is None else s["offsets"].tolist()
    x = s["logits"].double()
    masked = torch.isneginf(x)
    leaf = torch.where(masked, 0.0, x).requires_grad_(c["grad"])
    shares = torch.zeros(len(ends) - 1, e, dtype=torch.float64, device=x.device)
    terms, square, every = [], 0.0, 0
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        at = (~masked[a:b]).any(1).nonzero()[:, 0] + a
        if not at.numel():
            continue
        power = leaf[at].masked_fill(masked[at], -math.inf)
        if c["score"] == "sigmoid":
            q = torch.sigmoid(leaf[at]) * ~masked[at]
            p = q / q.sum(1, keepdim=True)
        else:
            p = torch.softmax(power, 1)
        mean = p.mean(0)
        chosen = s["experts"][a:b].reshape(-1)
        often = torch.bincount(chosen[chosen >= 0].long(), minlength=e).double()
        terms.append((mean * often).sum() * e / (c["topk"] * at.numel()))
        shares[i] = mean.detach()
        square = square + torch.logsumexp(power, 1).pow(2).sum()
        every += at.numel()
    loss = torch.stack(terms).mean() + c["z"] * square / every if terms else leaf.sum() * 0
    out = {"loss": loss.detach(), "counts": None, "shares": shares}
    if c["grad"]:
        out["d_logits"] = torch.autograd.grad(loss * s["d_loss"].double(), leaf)[0].masked_fill(masked, 0)
    return out


def exact(case, seed):
    with torch.enable_grad():
        return globals()["_exact_" + case["op"]](prepare(case, seed))


# ---- what a pass cannot do without ---------------------------------------------
def work(case):
    c, size, grad = case, SIZE[case["dtype"]], case["grad"]
    if c["op"] == "join":
        n, stream = c["rows"] * c["width"], 4 if c["wide"] else size
        gate = {"none": 0, "channel": c["width"], "row": c["rows"], "all": n}[c["gate"]] * size
        weights = c["width"] * stream * (1 + c["bias"]) * (1 + (c["block"] and c["after"]))
        if not c["block"]:     # the stream read, its norm written; backward both gradients and the stream again
            return {"bytes": n * (stream + size) + weights + (n * (2 * stream + size) + weights if grad else 0), "flops": 0}
        moved = n * (2 * stream + 2 * size) + gate + weights
        # backward: two incoming gradients, the new stream and the block's output (and gate) read, two gradients (and the gate's) written
        return {"bytes": moved + (n * (3 * stream + 3 * size) + 2 * gate + weights if grad else 0), "flops": 0}
    if c["op"] == "dense":
        m, n, k, out = c["rows"], c["cols"], c["depth"], 4 if c["wide"] else size
        moved = (m * k + n * k) * size + m * n * out * (1 + c["residual"])
        if grad:   # what the activation was applied to is kept, and read with the incoming gradient; operands again, gradients written
            kept = m * n * size if c["activation"] != "none" else 0
            moved += 2 * kept + m * n * out + 2 * (m * k + n * k) * size
        return {"bytes": moved, "flops": (6 if grad else 2) * m * n * k}
    n = c["tokens"] * c["experts"] * size
    return {"bytes": n + c["tokens"] * c["topk"] * 4 + max(1, c["sequences"]) * c["experts"] * 8 + (2 * n if grad else 0), "flops": 0}
