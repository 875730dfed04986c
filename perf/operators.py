"""The operators of an expert layer beside the collectives that spread it over
ranks, as cases that can be timed: the router, matrix products in 8-bit floating
point with a scale for each block of 128 (one weight matrix, or one for each
expert), and the combination of the experts' rows, each with its gradient.

A case is a dict of plain values:

    name     listed cases only
    op       route | product | experts | combine
    dtype    f32 | bf16 | f16: the router's logits; the activations
    grad     whether the pass goes backward too

    route    tokens, experts, topk, score (softmax | sigmoid), bias, groups,
             kept, group_top, renormalise, padded (tokens of no sequence, whose
             logits are all masked). One pass: weights, experts and the
             assignment of tokens to experts; with `grad` the logits' gradient.
    product  rows, cols, depth. One pass: the activations are rounded to 8
             bits and multiplied with a weight matrix laid out in 8 bits
             beforehand; with `grad` also the activations' and the weights'
             gradients, from an incoming one that is rounded likewise.
    experts  tokens, experts, topk, cols, depth, padded. The same with a weight
             matrix for each expert: a row of the result for each pair of a
             token and an expert, in the experts' order.
    combine  tokens, topk, depth, padded. One pass: a token's rows from its
             experts are added up with their weights; with `grad` the rows'
             and the weights' gradients.

`run` computes them in elementary torch operations, or, where `own` is true,
with the package's operators.
"""
import math

import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
E4M3 = torch.float8_e4m3fn
BLOCK = 128
LARGEST = 448.0          # of an 8-bit float with four exponent bits
LEAST = 2.0 ** -96       # a block whose numbers are all smaller is scaled as if this were in it

#: Most multiplications and bytes of a drawn case (the largest listed ones').
MOST_FLOPS = 6 * 65536 * 2048 * 4096
MOST_TOKENS = {"route": 65536, "product": 8192, "experts": 16384, "combine": 16384}


# ---- the cases -----------------------------------------------------------------
def _route(tokens, experts, topk, score="softmax", bias=False, groups=1, kept=1, group_top=1, renormalise=True,
           padded=0, dtype="f32", grad=False):
    return {"op": "route", "tokens": tokens, "experts": experts, "topk": topk, "score": score, "bias": bias, "groups": groups,
            "kept": kept, "group_top": group_top, "renormalise": renormalise, "padded": padded, "dtype": dtype, "grad": grad}


def _product(rows, cols, depth, dtype="bf16", grad=False):
    return {"op": "product", "rows": rows, "cols": cols, "depth": depth, "dtype": dtype, "grad": grad}


def _experts(tokens, experts, topk, cols, depth, padded=0, dtype="bf16", grad=False):
    return {"op": "experts", "tokens": tokens, "experts": experts, "topk": topk, "cols": cols, "depth": depth, "padded": padded,
            "dtype": dtype, "grad": grad}


def _combine(tokens, topk, depth, padded=0, dtype="bf16", grad=False):
    return {"op": "combine", "tokens": tokens, "topk": topk, "depth": depth, "padded": padded, "dtype": dtype, "grad": grad}


def listed():
    cases = {
        # one sequence answers a token at a time: latency
        "route_1": _route(1, 128, 8),
        # a training step's tokens on one rank, forward and backward, logits as a bf16 product left them
        "route_4099_training": _route(4099, 64, 6, dtype="bf16", renormalise=False, padded=37, grad=True),
        # the largest batch: every rank's tokens, experts in groups with a bias that balances them
        "route_65536_groups": _route(65536, 256, 8, score="sigmoid", bias=True, groups=8, kept=4, group_top=2),
        # one token through one layer: the weights are what is read
        "product_1": _product(1, 4096, 4096),
        # a few sequences answering together, no size a multiple of the block
        "product_50_odd": _product(50, 5000, 2500, dtype="f16"),
        # a prompt of ordinary length
        "product_2048": _product(2048, 4096, 4096),
        # a training step of a large layer, forward and both gradients
        "product_8192_training": _product(8192, 8192, 4096, grad=True),
        # eight sequences answering a token at a time, most experts with no row or one
        "experts_8": _experts(8, 64, 6, 1024, 2048),
        # a prompt's tokens over narrow experts, an odd number of them, some of no sequence
        "experts_1999": _experts(1999, 64, 6, 1408, 2048, padded=77),
        # a training step's tokens over wide experts
        "experts_16384_training": _experts(16384, 32, 4, 2048, 4096, grad=True),
        # one token's rows
        "combine_8": _combine(8, 6, 2048),
        # the same training step's rows, forward and backward
        "combine_16384_training": _combine(16384, 4, 4096, padded=300, grad=True),
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
    op = rng.choice(("route", "product", "product", "experts", "experts", "combine"))
    tokens = _between(rng, 1, MOST_TOKENS[op])
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    grad = rng.random() < 0.4
    padded = rng.randrange(tokens // 8 + 1) if rng.random() < 0.5 else 0
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * _between(rng, 4, 512 // groups)
        kept = rng.randint(1, groups)
        sigmoid = rng.random() < 0.5
        return _route(tokens, experts, rng.randint(1, min(16, kept * (experts // groups))), "sigmoid" if sigmoid else "softmax",
                      sigmoid and rng.random() < 0.7, groups, kept, rng.choice((1, 2)) if sigmoid and groups > 1 else 1,
                      rng.random() < 0.6, padded, dtype, grad)
    if op == "combine":
        return _combine(tokens, rng.randint(1, 8), _between(rng, 64, 4096), padded, dtype if dtype != "f32" else "bf16", grad)
    cols, depth = _between(rng, 64, 8192 if op == "product" else 2048), _between(rng, 64, 8192 if op == "product" else 4096)
    experts, topk = _between(rng, 2, 64), rng.randint(1, 8)
    topk = min(topk, experts)
    rows = tokens if op == "product" else tokens * topk
    most = MOST_FLOPS // ((6 if grad else 2) * cols * depth)
    tokens = max(1, tokens * min(rows, most) // rows)
    if op == "product":
        return _product(tokens, cols, depth, dtype, grad)
    return _experts(tokens, experts, topk, cols, depth, min(padded, tokens // 8), dtype, grad)


# ---- what a program has in hand ------------------------------------------------
def _activations(g, rows, depth, dtype):
    """Normal numbers, some channels much larger than the others, as layers' outputs have them."""
    x = torch.randn(rows, depth, generator=g, device="cuda")
    return (x * (torch.rand(depth, generator=g, device="cuda") * 4 - 2).exp()).to(dtype)


def _padded_to(x, dim, multiple):
    short = -x.shape[dim] % multiple
    if not short:
        return x
    shape = list(x.shape)
    shape[dim] = short
    return torch.cat([x, x.new_zeros(shape)], dim)


def _rounded(blocks, dims):
    """8-bit numbers and scales of `blocks`, in 32 bits, whose blocks lie along `dims`."""
    most = blocks.abs().amax(dims, keepdim=True).clamp_min(LEAST)
    largest = torch.full_like(most, LARGEST)      # (a number in its place would be divided by as a product)
    return (blocks * (largest / most)).to(E4M3), most / largest


def _weights(w):
    """Squares of 128 x 128 numbers of w (..., N, K) share a scale: 8-bit numbers (..., N, K),
    rows at multiples of 16 bytes, and scales (..., ceil(N / 128), ceil(K / 128))."""
    n, k = w.shape[-2:]
    wide = _padded_to(_padded_to(w, -1, BLOCK), -2, BLOCK)
    tiles = wide.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))
    q, s = _rounded(tiles, (-3, -1))
    q = q.reshape(wide.shape)[..., :n, :k]
    return _aligned(q), s.squeeze(-1).squeeze(-2).contiguous()


def _aligned(q):
    """`q` with its rows at multiples of 16 bytes."""
    *lead, n, k = q.shape
    room = torch.zeros(*lead, n, -(-k // 16) * 16, dtype=torch.uint8, device=q.device)
    room[..., :k] = q.view(torch.uint8)
    return room[..., :k].view(E4M3)


def _assigned(chosen, experts):
    """Where each pair of a token and an expert stands in the experts' order (-1: in no expert),
    the token at each place, and where each expert begins."""
    flat = chosen.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=key.device)
    offsets[1:] = counts.cumsum(0)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=key.device)
    slots = torch.where(flat < 0, -1, place).to(torch.int32).view(chosen.shape)
    at = torch.arange(order.numel(), device=key.device)
    tokens = torch.where(at < offsets[-1], order // chosen.shape[1], -1).to(torch.int32)
    return offsets, tokens, slots


def _choice(g, tokens, experts, topk, padded):
    """`topk` different experts for each token, some experts liked better; the last `padded` tokens have none."""
    liked = torch.randn(experts, generator=g, device="cuda") * 0.5
    noise = -(-torch.rand(tokens, experts, generator=g, device="cuda").clamp_min(1e-9).log()).log()
    chosen = (liked + noise).topk(topk, -1).indices.to(torch.int32)
    chosen[tokens - padded:] = -1
    return chosen


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPE[case["dtype"]]
    s = {"case": case}
    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        logits = torch.randn(t, e, generator=g, device="cuda") * 1.5
        logits[t - case["padded"]:] = -math.inf
        s["logits"] = logits.to(dtype)
        s["bias"] = torch.randn(e, generator=g, device="cuda") * 0.05 if case["bias"] else None
        s["d_weights"] = torch.randn(t, case["topk"], generator=g, device="cuda") if case["grad"] else None
        return s
    if case["op"] == "combine":
        t, k, h = case["tokens"], case["topk"], case["depth"]
        chosen = _choice(g, t, max(2 * k, 8), k, case["padded"])
        s["offsets"], s["order"], s["slots"] = _assigned(chosen, max(2 * k, 8))
        s["rows"] = torch.randn(t * k, h, generator=g, device="cuda").to(dtype)
        s["weights"] = torch.softmax(torch.randn(t, k, generator=g, device="cuda"), -1).masked_fill(chosen < 0, 0)
        s["d_out"] = torch.randn(t, h, generator=g, device="cuda").to(dtype) if case["grad"] else None
        return s
    n, k = case["cols"], case["depth"]
    if case["op"] == "product":
        rows = out_rows = case["rows"]
        w = torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
    else:
        rows, e = case["tokens"], case["experts"]
        out_rows = rows * case["topk"]
        chosen = _choice(g, rows, e, case["topk"], case["padded"])
        s["offsets"], s["order"], s["slots"] = _assigned(chosen, e)
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        w = torch.randn(e, n, k, generator=g, device="cuda") * k ** -0.5
    s["x"] = _activations(g, rows, k, dtype)
    s["wq"], s["ws"] = _weights(w)
    if case["grad"]:     # the weights as the gradient of the activations reads them, laid out once too
        s["tq"], s["ts"] = _aligned(s["wq"].transpose(-1, -2)), s["ws"].transpose(-1, -2).contiguous()
        s["d_out"] = (torch.randn(out_rows, n, generator=g, device="cuda") * 1e-3).to(dtype)
    return s


# ---- the operators in their plain form -----------------------------------------
def _rows8(x):
    """x (..., K) rounded to 8 bits in blocks of 128 along its rows, as the numbers that stand for it."""
    k = x.shape[-1]
    q, s = _rounded(_padded_to(x.float(), -1, BLOCK).unflatten(-1, (-1, BLOCK)), -1)
    return (q.float() * s).flatten(-2)[..., :k]


def _columns8(x):
    """x (..., M, K) rounded to 8 bits in blocks of 128 along its columns."""
    m = x.shape[-2]
    q, s = _rounded(_padded_to(x.float(), -2, BLOCK).unflatten(-2, (-1, BLOCK)), -2)
    return (q.float() * s).flatten(-3, -2)[..., :m, :]


def _squares(q, s):
    """The numbers that 8-bit weights and their scales stand for."""
    n, k = q.shape[-2:]
    return q.float() * s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _plain_route(s):
    c = s["case"]
    x = s["logits"].float()
    t, e = x.shape
    k, g = c["topk"], c["groups"]
    inf = torch.tensor(math.inf, device=x.device)
    there = x != -inf
    if c["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-x))
        key = score
    else:
        top = x.amax(-1, keepdim=True)
        top = torch.where(top == -inf, 0, top)
        score = torch.exp(x - top)
        key = x
    whole = score.sum(-1, keepdim=True)
    key = key + s["bias"] if c["bias"] else key
    key = torch.where(there, key, -inf)
    if g > 1:
        best = key.view(t, g, e // g).sort(-1, descending=True).values[..., :c["group_top"]]
        of_group = torch.where(best == -inf, 0, best).sum(-1).where(best[..., 0] > -inf, -inf)
        keep = torch.zeros(t, g, dtype=torch.bool, device=x.device)
        keep.scatter_(1, of_group.sort(dim=-1, descending=True, stable=True).indices[:, :c["kept"]], True)
        key = torch.where(keep.repeat_interleave(e // g, 1), key, -inf)
    ranked = key.sort(dim=-1, descending=True, stable=True)
    chosen, valid = ranked.indices[:, :k], ranked.values[:, :k] > -inf
    w = torch.where(valid, score.gather(1, chosen), 0)
    total = w.sum(-1, keepdim=True) if c["renormalise"] else whole if c["score"] == "softmax" else torch.ones_like(whole)
    weights = torch.where(total > 0, w / total, 0)
    experts = torch.where(valid, chosen, -1).to(torch.int32)
    out = {"weights": weights, "experts": experts}
    out["offsets"], out["order"], out["slots"] = _assigned(experts, e)
    if c["grad"]:
        d = torch.where(valid, s["d_weights"], 0)
        d_score = torch.zeros_like(x).scatter_(1, chosen, d)
        if c["renormalise"]:       # through the division by the chosen scores' sum
            among = torch.zeros_like(x).scatter_(1, chosen, valid.float()) > 0
            d_score = torch.where(among, d_score - (weights * d).sum(-1, keepdim=True), 0)
            if c["score"] == "sigmoid":
                d_logits = torch.where(total > 0, d_score / total, 0) * score * (1 - score)
            else:
                d_logits = torch.where(total > 0, score / total, 0) * d_score
        elif c["score"] == "sigmoid":
            d_logits = d_score * score * (1 - score)
        else:
            d_logits = torch.where(whole > 0, score / whole, 0) * (d_score - (weights * d).sum(-1, keepdim=True))
        out["d_logits"] = d_logits.to(s["logits"].dtype)
    return out


def _plain_product(s):
    dtype = s["x"].dtype
    w = _squares(s["wq"], s["ws"])
    out = [(_rows8(s["x"]) @ w.t()).to(dtype)]
    if s["case"]["grad"]:
        out.append((_rows8(s["d_out"]) @ w).to(dtype))
        out.append((_columns8(s["d_out"]).t() @ _columns8(s["x"])).to(dtype))
    return out


def _side_by_side(s):
    """(the place of each expert's i-th row (E, M), whether it has one), M a multiple of 128."""
    m = -(-max(s["most"], 1) // BLOCK) * BLOCK
    at = torch.arange(m, device="cuda")
    first, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    there = at < (end - first)[:, None]
    return torch.where(there, first[:, None] + at, 0), there[..., None]


def _plain_experts(s):
    dtype = s["x"].dtype
    place, there = _side_by_side(s)
    w = _squares(s["wq"], s["ws"])
    token = s["order"].long()[place].clamp_min(0)
    x = torch.where(there, s["x"].float()[token], 0)
    wanted = there.squeeze(-1)
    room = lambda width: torch.zeros(s["order"].numel(), width, device="cuda")  # noqa: E731
    y = room(w.shape[1])
    y[place[wanted]] = torch.matmul(_rows8(x), w.transpose(1, 2).contiguous())[wanted]
    out = [y.to(dtype)]
    if s["case"]["grad"]:
        d = torch.where(there, s["d_out"].float()[place], 0)
        dx = room(w.shape[2])
        dx[place[wanted]] = torch.matmul(_rows8(d), w)[wanted]
        out.append(dx.to(dtype))
        out.append(torch.matmul(_columns8(d).transpose(1, 2).contiguous(), _columns8(x)).to(dtype))
    return out


def _plain_combine(s):
    slots = s["slots"].long()
    there = (slots >= 0)[..., None]
    rows = torch.where(there, s["rows"].float()[slots.clamp_min(0)], 0)
    out = [(rows * s["weights"][..., None]).sum(1).to(s["rows"].dtype)]
    if s["case"]["grad"]:
        d = s["d_out"].float()[:, None]
        wanted = there.squeeze(-1)
        d_rows = torch.zeros(s["rows"].shape, device="cuda")
        d_rows[slots[wanted]] = (d * s["weights"][..., None])[wanted]
        out += [d_rows.to(s["rows"].dtype), (rows * d).sum(-1)]
    return out


# ---- the package's operators ---------------------------------------------------
def _own_route(s):
    from mintccl_amd.routing import assign, route, route_grad
    c = s["case"]
    weights, experts = route(s["logits"], c["topk"], score=c["score"], bias=s["bias"], groups=c["groups"], kept=c["kept"],
                             group_top=c["group_top"], renormalise=c["renormalise"])
    plan = assign(experts, c["experts"])
    out = {"weights": weights, "experts": experts, "offsets": plan.offsets, "order": plan.tokens, "slots": plan.slots}
    if c["grad"]:
        out["d_logits"] = route_grad(s["d_weights"], s["logits"], experts, score=c["score"], renormalise=c["renormalise"])
    return out


def _own_product(s):
    from mintccl_amd.block8 import Blocks, product, weight_grad
    dtype = s["x"].dtype
    out = [product(s["x"], Blocks(s["wq"], s["ws"]), dtype=dtype)]
    if s["case"]["grad"]:
        out.append(product(s["d_out"], Blocks(s["tq"], s["ts"]), dtype=dtype))
        out.append(weight_grad(s["d_out"], s["x"], dtype=dtype))
    return out


def _own_experts(s):
    from mintccl_amd.block8 import Blocks, product, weight_grad
    from mintccl_amd.routing import Assignment
    dtype = s["x"].dtype
    plan = Assignment(s["offsets"], s["order"], s["slots"])
    out = [product(s["x"], Blocks(s["wq"], s["ws"]), plan, gather=True, dtype=dtype)]
    if s["case"]["grad"]:
        out.append(product(s["d_out"], Blocks(s["tq"], s["ts"]), plan, dtype=dtype))
        out.append(weight_grad(s["d_out"], s["x"], plan, gather=True, dtype=dtype))
    return out


def _own_combine(s):
    from mintccl_amd.combine import combine, combine_grad
    from mintccl_amd.routing import Assignment
    plan = Assignment(s["offsets"], s["order"], s["slots"])
    out = [combine(s["rows"], plan, s["weights"])]
    if s["case"]["grad"]:
        out += combine_grad(s["d_out"], s["rows"], plan, s["weights"])
    return out


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


# ---- the definition in 64 bits -------------------------------------------------
def _to8(v, dim):
    """Rounds `v` (64 bits) to 8 bits in blocks of 128 along `dim`, from the definition: a block's
    scale is the 32-bit number next to its largest magnitude / 448, a number is what is next to
    the 32-bit product of it and 448 / largest, in steps of an eighth of its power of two, of 2**-9 at least."""
    v = v.movedim(dim, -1)
    n = v.shape[-1]
    full = torch.zeros(*v.shape[:-1], -(-n // 128) * 128, dtype=torch.float64, device=v.device)
    full[..., :n] = v
    full = full.view(*v.shape[:-1], -1, 128)
    most = torch.maximum(full.abs().max(-1, keepdim=True).values, torch.tensor(2.0 ** -96, dtype=torch.float64, device=v.device))
    scaled = (full * (448 / most).float().double()).float().double()
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp_min(2.0 ** -6))) - 3)
    value = (scaled / step).round() * step * (most / 448).float().double()
    return value.flatten(-2)[..., :n].movedim(-1, dim)


def _of_weights(q, s):
    i = torch.arange(q.shape[-2], device=q.device) // 128
    j = torch.arange(q.shape[-1], device=q.device) // 128
    return q.float().double() * s.double()[..., i[:, None], j]


def _exact_route(s):
    c = s["case"]
    x = s["logits"].double()
    t, e = x.shape
    masked = torch.isneginf(x)
    p = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
    rank_by = (p if c["score"] == "sigmoid" else x) + (s["bias"].double() if c["bias"] else 0)
    rank_by = rank_by.masked_fill(masked, -math.inf)
    if c["groups"] > 1:
        split = rank_by.reshape(t, c["groups"], -1)
        tops = split.topk(min(c["group_top"], split.shape[-1]), -1).values
        group = tops.masked_fill(torch.isneginf(tops), 0).sum(-1).masked_fill(torch.isneginf(tops[..., 0]), -math.inf)
        order = torch.sort(-group, dim=-1, stable=True).indices
        drop = torch.ones(t, c["groups"], dtype=torch.bool, device=x.device)
        drop[torch.arange(t, device=x.device)[:, None], order[:, :c["kept"]]] = False
        rank_by = split.masked_fill(drop[..., None], -math.inf).reshape(t, e)
    order = torch.sort(-rank_by, dim=-1, stable=True).indices[:, :c["topk"]]
    valid = ~torch.isneginf(rank_by.gather(1, order))
    picked = torch.zeros_like(x)
    picked.scatter_(1, order, valid.double())
    leaf = torch.where(masked, -80.0, x).requires_grad_(c["grad"])
    soft = torch.sigmoid(leaf) if c["score"] == "sigmoid" else leaf.exp() / (leaf.exp() * ~masked).sum(-1, keepdim=True).clamp_min(1e-300)
    soft = soft * ~masked
    w = soft / (soft * picked).sum(-1, keepdim=True).clamp_min(1e-300) if c["renormalise"] else soft
    weights = torch.where(valid, w.gather(1, order), 0)
    out = {"weights": weights.detach(), "experts": None, "offsets": None, "order": None, "slots": None}
    if c["grad"]:
        out["d_logits"], = torch.autograd.grad((weights * s["d_weights"].double()).sum(), leaf)
    return out


def _exact_product(s):
    w = _of_weights(s["wq"], s["ws"])
    x = s["x"].double()
    out = [_to8(x, 1) @ w.T]
    if s["case"]["grad"]:
        d = s["d_out"].double()
        out += [_to8(d, 1) @ w, _to8(d, 0).T @ _to8(x, 0)]
    return out


def _exact_experts(s):
    ends = s["offsets"].tolist()
    e, n, k = s["wq"].shape
    y = torch.zeros(s["order"].numel(), n, dtype=torch.float64, device="cuda")
    dx = torch.zeros(s["order"].numel(), k, dtype=torch.float64, device="cuda")
    dw = torch.zeros(e, n, k, dtype=torch.float64, device="cuda")
    for i in range(e):
        a, b = ends[i], ends[i + 1]
        if a == b:
            continue
        w = _of_weights(s["wq"][i], s["ws"][i])
        x = s["x"][s["order"][a:b].long()].double()
        y[a:b] = _to8(x, 1) @ w.T
        if s["case"]["grad"]:
            d = s["d_out"][a:b].double()
            dx[a:b] = _to8(d, 1) @ w
            dw[i] = _to8(d, 0).T @ _to8(x, 0)
    return [y, dx, dw] if s["case"]["grad"] else [y]


def _exact_combine(s):
    t, k = s["slots"].shape
    out = torch.zeros(t, s["rows"].shape[1], dtype=torch.float64, device="cuda")
    d_rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda")
    d_weights = torch.zeros(t, k, dtype=torch.float64, device="cuda")
    for j in range(k):
        token = (s["slots"][:, j] >= 0).nonzero()[:, 0]
        at = s["slots"][token, j].long()
        w = s["weights"][token, j, None].double()
        out[token] += w * s["rows"][at].double()
        if s["case"]["grad"]:
            d = s["d_out"][token].double()
            d_rows[at] = w * d
            d_weights[token, j] = (s["rows"][at].double() * d).sum(1)
    return [out, d_rows, d_weights] if s["case"]["grad"] else [out]


def exact(case, seed):
    with torch.enable_grad():
        return globals()["_exact_" + case["op"]](prepare(case, seed))


# ---- what a pass cannot do without ---------------------------------------------
def work(case):
    c, size, grad = case, SIZE[case["dtype"]], case["grad"]
    if c["op"] == "route":
        pairs = c["tokens"] * c["topk"]
        # logits read; weights, experts, places and tokens written; gradient: weights' read, logits' written
        return {"bytes": c["tokens"] * c["experts"] * size * (2 if grad else 1) + pairs * (20 if grad else 16), "flops": 0}
    if c["op"] == "combine":
        t, k, h = c["tokens"], c["topk"], c["depth"]
        rows = (t - c["padded"]) * k
        moved = (rows + t) * h * size + 8 * t * k
        # backward: the incoming gradient and the rows read, the rows' gradient written
        return {"bytes": moved + ((rows + t) * h * size + t * k * (h * size + 4) if grad else 0), "flops": (6 if grad else 2) * rows * h}
    n, k = c["cols"], c["depth"]
    if c["op"] == "product":
        rows, matrices, out_rows = c["rows"], 1, c["rows"]
    else:
        rows, out_rows = c["tokens"], (c["tokens"] - c["padded"]) * c["topk"]
        matrices = min(c["experts"], max(1, out_rows))    # of those, the ones that have rows are read
    moved = rows * k * size + matrices * n * k + out_rows * n * size
    if grad:   # incoming gradient and weights again, both gradients written
        moved += out_rows * n * size + matrices * n * k + out_rows * k * size + size * (1 if c["op"] == "product" else c["experts"]) * n * k
    return {"bytes": moved, "flops": (6 if grad else 2) * out_rows * n * k}
