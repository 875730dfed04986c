"""Definitions of the operators around an expert layer in 64 bits, written in elementary operations that torch can differentiate, with the
magnitudes that their roundings go by."""
from __future__ import annotations

import math

import torch

from tests.expert_oracle import HALF_ULP, TINY

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = 2.0 ** -24                # a rounding in 32 bits, relative
#: A sum over a row in 32 bits: a lane adds at most 32 numbers one behind the other, six steps join a wavefront's lanes and at most 16 wavefronts
#: follow; each addition rounds once.  A normalised number passes through three such sums at most (mean, mean square, and the gradient's), with a
#: root, a quotient and a dozen products: less than 256 roundings, each of the magnitude that `magnitude_of` has.
ROW = 256 * UNIT


def close(got, want, magnitude, dt, units=ROW, more=0.0):
    """Every number of `got`, of type `dt`, is `want`, rounded once, but for roundings in 32 bits (`units` of `magnitude`); `more` is allowed beside."""
    assert got.dtype == dt and got.shape == want.shape
    got, want = got.double().cpu(), want.double().cpu()
    off = (got - want).abs()
    most = HALF_ULP[dt] * (want.abs() + units * magnitude.cpu()) + units * magnitude.double().cpu() + more + TINY[dt]
    bad = ~((off <= most) | (got == want))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, at worst {float((off - most)[bad].max()):.3g} over {float(most[bad].max()):.3g}"


# ---- norms -----------------------------------------------------------------------
def norm64(x, weight, bias, kind, eps):
    x = x.double()
    m = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    q = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    y = (x - m) * q
    if weight is not None:
        y = y * weight.double()
    return y if bias is None else y + bias.double()


def norm_parts(x, kind, eps):
    """xh, q, and the magnitude of xh: what it is made of, without what cancels."""
    x = x.double()
    m = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    q = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    wide = x.abs() + (x.abs().mean(-1, keepdim=True) if kind == "layer" else 0)
    # (the mean square of what is left when the mean is off by a part of the magnitudes is off by that part, twice)
    return (x - m) * q, q, wide * q * (1 + (wide * wide).mean(-1, keepdim=True) * q * q if kind == "layer" else 1)


def gate64(g, by):
    g = g.double()
    if by is None:
        return g, torch.ones_like(g)
    if by == "tanh":
        return torch.tanh(g), 1 - torch.tanh(g) ** 2
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if by == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def ones(t, like):
    return torch.ones_like(like[0].double()) if t is None else t.double()


def norm_grad64(d, x, weight, kind, eps):
    """((d_x, d_weight, d_bias), their magnitudes)."""
    xh, q, wide = norm_parts(x, kind, eps)
    d, w = d.double(), ones(weight, x)
    dw = d * w
    m0 = (dw * xh).mean(-1, keepdim=True)
    m1 = dw.mean(-1, keepdim=True) if kind == "layer" else 0
    size0 = (dw.abs() * wide).mean(-1, keepdim=True)
    size1 = dw.abs().mean(-1, keepdim=True) if kind == "layer" else 0
    return (q * (dw - xh * m0 - m1), (d * xh).sum(0), d.sum(0)), (q * (dw.abs() + wide * size0 + size1), (d.abs() * wide).sum(0), d.abs().sum(0))


def join_grad64(d_stream, d_next, stream, y, *, after, gate, gate_by, scale, carry, before):
    """{name: (gradient, magnitude)}; `after` and `before` (weight, bias, kind, eps) or None, `stream` the new one."""
    found = {}
    d = torch.zeros(stream.shape, dtype=torch.float64) if d_stream is None else d_stream.double()
    size = d.abs()
    if before is not None:
        zero = torch.zeros(stream.shape, dtype=torch.float64) if d_next is None else d_next
        (dx, dw, db), (mx, mw, mb) = norm_grad64(zero, stream, before[0], *before[2:])
        d, size = d + dx, size + mx
        found.update(before_weight=(dw, mw), before_bias=(db, mb))
    found["stream"] = carry * d, abs(carry) * size
    G, mG = scale * d, abs(scale) * size
    u, wide, w, b = y.double(), y.double().abs(), ones(None, y), None
    yh, yw = u, wide
    if after is not None:
        yh, _, yw = norm_parts(y, *after[2:])
        w, b = ones(after[0], y), after[1]
        u, wide = yh * w, yw * w.abs()
        if b is not None:
            u, wide = u + b.double(), wide + b.double().abs()
    du, mdu = G, mG
    if gate is not None:
        a, slope = gate64(gate, gate_by)
        dg, mg = G * u, mG * wide
        if gate.dim() == 1:
            dg, mg = dg.sum(0), mg.sum(0)
        elif gate.shape[1] == 1 and y.shape[1] != 1:
            dg, mg = dg.sum(1, keepdim=True), mg.sum(1, keepdim=True)
        found["gate"] = dg * slope, mg * (slope.abs() + 2.0 ** -4)      # (a slope is a difference of numbers near 1 at most)
        du, mdu = G * a, mG * a.abs()
    if after is not None:
        (dy, dw, db), (my, mw, mb) = norm_grad64(du, y, after[0], *after[2:])
        scale_of = lambda v: v * 1.0  # noqa: E731
        # (du itself has magnitude mdu, not only its own)
        _, (my2, mw2, mb2) = norm_grad64(mdu, y, after[0], *after[2:])
        found.update(y=(dy, scale_of(my2)), after_weight=(dw, mw2), after_bias=(db, mb2))
    else:
        found["y"] = du, mdu
    return found


# ---- dense products -----------------------------------------------------------------
def activated64(z, name):
    z = z.double()
    F = torch.nn.functional
    return {None: lambda t: t, "relu": torch.relu, "silu": F.silu, "sigmoid": torch.sigmoid, "tanh": torch.tanh, "gelu": F.gelu,
            "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[name](z)


def slope64(z, name):
    z = z.detach().cpu().double().requires_grad_()
    return torch.autograd.grad(activated64(z, name).sum(), z)[0]


#: No activation is steeper (gelu at sqrt 2: 1.129), and its own evaluation in 32 bits takes less than 16 roundings of magnitude max(1, |z|).
STEEPEST, EVALUATED = 1.13, 16 * UNIT


def product64(x, w, depth_sum=None):
    """(x @ w.T, the products' magnitudes' sum)."""
    x, w = x.cpu().double(), w.cpu().double()
    return x @ w.t(), x.abs() @ w.abs().t()


def sum_units(depth, dt="f32"):
    """Of a sum of `depth` products in 32 bits, relative to the magnitudes' sum: an instruction adds 32 of them (in 32 bits four) in some order, and
    its sums are added one behind the other, in up to 256 parts; each addition rounds, or cuts off, once."""
    return (40 + -(-depth // (4 if dt == "f32" else 32))) * 2 * UNIT


# ---- the balance loss ------------------------------------------------------------------
def balance64(logits, experts, score, offsets, z):
    """(loss, counts, shares, there), differentiable by `logits` (64 bits)."""
    t, e = logits.shape
    ends = [0, t] if offsets is None else offsets.tolist()
    n = len(ends) - 1
    masked = torch.isneginf(logits)
    x = logits.masked_fill(masked, 0.0)
    terms, square, every = [], logits.new_zeros(()), 0
    counts, shares, there = torch.zeros(n, e, dtype=torch.int32), torch.zeros(n, e, dtype=torch.float64), torch.zeros(n, dtype=torch.int32)
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        chosen = experts[a:b].reshape(-1).long()
        counts[i] = torch.bincount(chosen[(chosen >= 0) & (chosen < e)], minlength=e).int()
        at = (~masked[a:b]).any(1).nonzero()[:, 0] + a
        there[i] = at.numel()
        if not at.numel():
            continue
        if score == "softmax":
            p = torch.softmax(x[at].masked_fill(masked[at], -math.inf), 1)
        else:
            s = torch.sigmoid(x[at]) * ~masked[at]
            p = s / s.sum(1, keepdim=True)
        shares[i] = p.mean(0).detach()
        terms.append((p.mean(0) * counts[i].double()).sum() * e / (experts.shape[1] * at.numel()))
        square = square + torch.logsumexp(x[at].masked_fill(masked[at], -math.inf), 1).pow(2).sum()
        every += at.numel()
    loss = torch.stack(terms).mean() + (z * square / every if z else 0) if terms else x.sum() * 0
    return loss, counts, shares, there
