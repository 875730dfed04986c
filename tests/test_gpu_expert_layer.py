"""The layer of experts over virtual ranks."""
import weakref

import pytest
import torch

from mintccl_amd.block8 import Blocks
from mintccl_amd.combine import combine
from mintccl_amd.common import VirtualComm
from mintccl_amd.experts import ExpertLayer, small_layer
from tests.expert_oracle import HALF_ULP, TINY, randn, rounded8, weight64

pytestmark = pytest.mark.gpu


def small(world, dev, **options):
    s = small_layer(world, dev)
    return ExpertLayer(VirtualComm(world_size=world, device=dev), s["router"], s["up"], s["down"], 4, **options), s


def test_passes_keep_apart_what_their_gradients_need(dev):
    """Two batches forward and then their backward passes: each one's gradients are what they are alone."""
    layer, s = small(2, dev)
    other = {n: [randn(*t.shape, seed=50 + i, dtype=t.dtype, dev=dev) for i, t in enumerate(s[n])] for n in ("tokens", "grads")}

    def gradients(kept, batch):
        d_tokens, found = layer.backward(batch["grads"], kept)
        return [*d_tokens, *(f[n] for f in found for n in ("up", "down", "router"))]

    alone = []
    for batch in (s, other):
        kept = []
        layer.forward(batch["tokens"], kept)
        alone.append(gradients(kept, batch))
    first, second = [], []
    layer.forward(s["tokens"], first)
    layer.forward(other["tokens"], second)
    for got, want in ((gradients(first, s), alone[0]), (gradients(second, other), alone[1])):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="another pass"):
        layer.forward(s["tokens"], first)
    with pytest.raises(ValueError, match="forward pass"):
        layer.backward(s["grads"], [])


def test_a_layer_that_only_answers_keeps_nothing(dev):
    layer, s = small(2, dev)
    kept = []
    want = layer.forward(s["tokens"], kept)
    there = [weakref.ref(t) for t in kept[0] if isinstance(t, torch.Tensor)]
    assert there and all(t() is not None for t in there)
    kept.clear()
    assert all(t() is None for t in there)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(dev)
    got = layer.forward(s["tokens"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated(dev) == before


def test_the_ranks_sums_are_rounded_once(dev):
    """The outputs are the sums of the ranks' parts, rounded to their type at the end alone."""
    for dtype in (torch.bfloat16, torch.float16):
        layer, s = small(8, dev)
        kept = []
        out = torch.cat(layer.forward([t.to(dtype) for t in s["tokens"]], kept))
        parts = [combine(y, plan, weights).double() for _, _, weights, _, plan, _, _, y in kept]
        want, size = sum(parts), sum(p.abs() for p in parts)
        extra = size * 8 * 2.0 ** -24                       # seven additions in 32 bits
        assert out.dtype == dtype
        assert ((out.double() - want).abs() <= extra + (want.abs() + extra) * HALF_ULP[dtype] * 1.001 + TINY[dtype]).all()


def grouped(key, groups, kept, top):
    """`key` with the groups that are not kept masked."""
    split = key.view(key.shape[0], groups, -1)
    order = split.topk(top, -1).values.sum(-1).sort(dim=-1, descending=True, stable=True).indices
    keep = torch.zeros(key.shape[0], groups, dtype=torch.bool, device=key.device).scatter_(1, order[:, :kept], True)
    return split.masked_fill(~keep[..., None], -torch.inf).view(key.shape)


LAYERS = [(1, {}), (4, {"score": "sigmoid", "groups": 4, "kept": 2, "group_top": 2, "scale": 2.5}),
          (8, {"renormalise": False, "scale": 0.5}), (2, {"score": "sigmoid", "renormalise": False, "biased": True}),
          (4, {"groups": 2, "kept": 1, "biased": True})]


@pytest.mark.parametrize("world,options", LAYERS)
def test_a_layers_steps_one_by_one(dev, world, options):
    """Forward and backward against the steps' definitions in 64 bits, with the roundings that they name.

    A number that a step rounds to 16 bits may fall to the other side of a tie here: off by 2^-8 at most.  Where it is rounded to 8
    bits next, one in sixteen of those may fall to the other side again, off by up to 2^-4 (0.58 of it on the average): all in
    all less than 0.004 and 0.009 in 2-norm, together 0.01."""
    options = dict(options)
    bias = randn(16, seed=9, scale=0.05, dev=dev) if options.pop("biased", False) else None
    layer, s = small(world, dev, bias=bias, **options)
    kept, k, dtype = [], 4, torch.bfloat16
    out = torch.cat(layer.forward(s["tokens"], kept))
    d_tokens, found = layer.backward(s["grads"], kept)
    d = torch.cat(s["grads"]).double()
    x = torch.cat(s["tokens"])
    score, renorm, scale = options.get("score", "softmax"), options.get("renormalise", True), options.get("scale", 1.0)
    near = lambda a, b: float((a.double() - b).norm() / b.norm()) < 0.01  # noqa: E731
    as16 = lambda v: v.to(dtype).double()  # noqa: E731

    logits = x.double() @ s["router"].double().t()
    leaf = logits.clone().requires_grad_()
    scores = torch.sigmoid(leaf) if score == "sigmoid" else torch.softmax(leaf, -1)
    key = (scores.detach() if score == "sigmoid" else logits) + (0 if bias is None else bias.double())
    key = grouped(key, options["groups"], options["kept"], options.get("group_top", 1)) if "groups" in options else key
    experts = key.topk(k, -1).indices
    weights = scores.gather(1, experts)
    weights = scale * (weights / weights.sum(-1, keepdim=True) if renorm else weights)
    w = weights.detach()
    rows = torch.zeros(*w.shape, x.shape[1], dtype=torch.float64, device=dev)
    d_x, d_weights = torch.zeros(*x.shape, dtype=torch.float64, device=dev), torch.zeros_like(w)
    for r, (x_r, _, weights_r, experts_r, plan, u_r, h_r, y_r) in enumerate(kept):
        assert torch.equal(x_r, x) and torch.equal(experts_r.long(), experts)
        assert torch.allclose(weights_r.double(), w, rtol=2.0 ** -16, atol=1e-30)
        at = plan.offsets.tolist()
        for i in range(layer.own):
            token, choice = (experts == r * layer.own + i).nonzero(as_tuple=True)
            own = slice(at[i], at[i + 1])
            assert torch.equal(plan.tokens[own].long(), token)
            if not len(token):
                assert (found[r]["up"][i] == 0).all() and (found[r]["down"][i] == 0).all()
                continue
            up, down = (weight64(Blocks(v.q[i], v.scale[i])) for v in (layer.ranks[r]["up"], layer.ranks[r]["down"]))
            u = as16(rounded8(x[token], 1) @ up.t())
            h = as16(torch.nn.functional.silu(u))
            y = as16(rounded8(h, 1) @ down.t())
            assert near(u_r[own], u) and near(h_r[own], h) and near(y_r[own], y)
            rows[token, choice] = y
            d_weights[token, choice] = (d[token] * y).sum(-1)
            d_y = as16(w[token, choice][:, None] * d[token])
            d_h = as16(rounded8(d_y, 1) @ down)
            sig = torch.sigmoid(u)
            d_u = as16(d_h * (sig + u * sig * (1 - sig)))
            assert near(found[r]["down"][i], rounded8(d_y, 0).t() @ rounded8(h, 0))
            assert near(found[r]["up"][i], rounded8(d_u, 0).t() @ rounded8(x[token], 0))
            d_x.index_add_(0, token, as16(rounded8(d_u, 1) @ up))
    assert near(out, (w[..., None] * rows).sum(1))
    d_logits, = torch.autograd.grad((weights * d_weights).sum(), leaf)
    assert near(torch.cat(d_tokens), d_x + d_logits @ s["router"].double())
    for f in found:
        assert near(f["router"], d_logits.t() @ x.double())


def test_a_layer_of_no_tokens(dev):
    layer, s = small(4, dev)
    none = [t[:0] for t in s["tokens"]]
    kept = []
    assert [tuple(t.shape) for t in layer.forward(none, kept)] == [(0, 320)] * 4
    d_tokens, found = layer.backward(none, kept)
    assert [tuple(t.shape) for t in d_tokens] == [(0, 320)] * 4
    assert all((f[n] == 0).all() for f in found for n in ("up", "down", "router"))


def test_tensors_that_require_a_gradient_are_refused(dev):
    """Their results would have no history, and the gradient would end there without a word."""
    from mintccl_amd.block8 import product, quantise, quantise_weight, weight_grad
    from mintccl_amd.combine import combine_grad
    from mintccl_amd.routing import assign, route, route_grad
    x, w = randn(6, 128, seed=1, dev=dev), quantise_weight(randn(64, 128, seed=2, dev=dev))
    weights, chosen = route(x, 2)
    plan = assign(chosen, 128)
    rows = randn(12, 128, seed=3, dev=dev)
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda f: route(f(x), 2), lambda f: route_grad(f(weights), x, chosen), lambda f: quantise(f(x)), lambda f: quantise_weight(f(x)),
             lambda f: product(f(x), w), lambda f: weight_grad(x, f(x)), lambda f: combine(rows, plan, f(weights)),
             lambda f: combine_grad(f(x), rows, plan, weights)]
    for call in calls:
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call(leaf)
        with torch.no_grad():
            got = call(leaf)
        want = call(lambda t: t)
        detached = call(lambda t: leaf(t).detach())
        for a, b, c in zip(*(v if isinstance(v, tuple) else (v,) for v in (got, want, detached))):
            a, b, c = (v.view(torch.uint8) if v.element_size() == 1 else v for v in (a, b, c))
            assert torch.equal(a, b) and torch.equal(a, c) and not a.requires_grad
    # (the choice has no gradient, and so the bias has none)
    assert torch.equal(route(x, 2, bias=leaf(x[0]))[1], route(x, 2, bias=x[0])[1])
    # a layer of parameters has its own backward pass; tokens that want a gradient of torch's get none here
    s = small_layer(2, dev)
    layer = ExpertLayer(VirtualComm(world_size=2, device=dev), *(torch.nn.Parameter(s[n]) for n in ("router", "up", "down")), 4)
    kept = []
    out = layer.forward(s["tokens"], kept)
    assert all(torch.equal(a, b) for a, b in zip(out, small(2, dev)[0].forward(s["tokens"])))
    assert not any(f["up"].requires_grad for f in layer.backward(s["grads"], kept)[1])
    with pytest.raises(RuntimeError, match="requires a gradient"):
        layer.forward([leaf(t) for t in s["tokens"]])


def test_the_operators_one_behind_the_other(dev):
    """As a program calls them that has all experts: from logits to the tokens' sums."""
    from mintccl_amd.block8 import product, quantise_weight
    from mintccl_amd.routing import assign, route
    experts, width, inner, tokens = 16, 256, 192, 50
    x, logits, b = randn(tokens, width, seed=1, dtype=torch.bfloat16, dev=dev), randn(tokens, experts, seed=2, dev=dev), randn(experts, seed=3, scale=0.1, dev=dev)
    up, down = randn(experts, inner, width, seed=4, scale=width ** -0.5, dev=dev), randn(experts, width, inner, seed=5, scale=inner ** -0.5, dev=dev)
    up8, down8 = quantise_weight(up), quantise_weight(down)
    weights, chosen = route(logits, 6, score="sigmoid", bias=b, groups=8, kept=4, renormalise=True)
    plan = assign(chosen, experts)
    act = torch.nn.functional.silu
    y = combine(product(act(product(x, up8, plan, gather=True)), down8, plan), plan, weights)
    want = torch.zeros(tokens, width, dtype=torch.float64, device=dev)
    for e in range(experts):
        token, choice = (chosen == e).nonzero(as_tuple=True)
        u, d = (weight64(Blocks(w.q[e], w.scale[e])) for w in (up8, down8))
        h = act((rounded8(x[token], 1) @ u.t()).bfloat16())
        want.index_add_(0, token, weights[token, choice].double()[:, None] * (rounded8(h, 1) @ d.t()).bfloat16().double())
    assert float((y.double() - want).norm() / want.norm()) < 0.01            # (as the layer's steps above)
