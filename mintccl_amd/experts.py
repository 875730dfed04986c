"""A layer of experts spread over the ranks of a communicator, and the block around it, forward and
backward: the operators and the collectives as they are used together.

Every rank has some of the experts and some of the tokens.  All tokens are
gathered on all ranks (``allgather``); each rank routes them, makes the rows of its
own experts (``route``, ``assign``, ``product``), adds up each token's rows
(``combine``) and hands the sums to the tokens' owners (``reducescatter``).  The way
back is the same the other way round: the gradient of a reduce-scatter is an allgather, that
of an allgather a reduce-scatter.  No token is dropped, and no row is sent that is not used.

The block norms the residual stream for the layer (``norms``), gives every token a
shared expert as well (``dense``), adds both to the stream with the next
block's norm (``join``), and makes the loss that keeps the experts in balance
(``routing.balance``).  Every rank has its own tokens' stream, and the whole of the block's own weights.

    MINTCCL_TEST_MODE=1 python -m mintccl_amd.experts

runs a small block on virtual ranks and compares it and its layer with the plain ones.  No
counterpart in the reference.
"""
from __future__ import annotations

import os

import torch
import torch.nn.functional as F

from . import dense
from .allgather import allgather
from .allreduce import allreduce
from .block8 import product, quantise_weight, transposed, weight_grad
from .combine import combine, combine_grad
from .common import VirtualComm, world_size_env
from .norms import Norm, join, join_grad, norm, norm_grad
from .reducescatter import reducescatter
from .routing import Balance, assign, balance, balance_grad, route, route_grad


class ExpertLayer:
    """``router`` (experts, width) in float32, ``up`` (experts, inner, width) and
    ``down`` (experts, width, inner): a token's output is the sum over its ``k`` experts of
    weight * silu(x @ up.T) @ down.T.  Rank r has the experts r * experts / world and on,
    as 8-bit weights laid out once.  The options are :func:`~mintccl_amd.routing.route`'s."""

    def __init__(self, comm: VirtualComm, router: torch.Tensor, up: torch.Tensor, down: torch.Tensor, k: int, *,
                 bias: torch.Tensor | None = None, **options) -> None:
        if router.shape[0] % comm.world_size:
            raise ValueError("the experts do not divide over the ranks")
        router, up, down = router.detach(), up.detach(), down.detach()           # (their gradients are backward()'s)
        self.comm, self.router, self.k, self.bias, self.options = comm, router, k, bias, options
        self.own = router.shape[0] // comm.world_size
        self.grad_options = {o: options[o] for o in ("score", "renormalise", "scale") if o in options}
        self.ranks = []
        for r in range(comm.world_size):
            mine = slice(r * self.own, (r + 1) * self.own)
            rank = {"up": quantise_weight(up[mine]), "down": quantise_weight(down[mine])}
            rank.update(up_t=transposed(rank["up"]), down_t=transposed(rank["down"]))
            self.ranks.append(rank)

    def _gathered(self, rows: list[torch.Tensor]) -> list[torch.Tensor]:
        """Every rank's rows on every rank: (world * tokens, width)."""
        t, width = rows[0].shape
        buffers = [torch.empty(self.comm.world_size, t * width, dtype=rows[0].dtype, device=rows[0].device) for _ in rows]
        for r, own in enumerate(rows):
            buffers[r][r] = own.reshape(-1)
        self.comm.run(lambda r: allgather(buffers[r], self.comm))
        return [b.view(-1, width) for b in buffers]

    def _summed(self, rows: list[torch.Tensor], dtype: torch.dtype) -> list[torch.Tensor]:
        """Each rank's own rows of the ranks' sum; ``rows`` are used up.  They travel in float32, so that the sum is rounded once, at its
        end (in 16 bits, half the bytes, every rank on the way would round it)."""
        world, (total, width) = self.comm.world_size, rows[0].shape
        self.comm.run(lambda r: reducescatter(rows[r].view(world, total // world * width), self.comm))
        return [rows[r].view(world, total // world, width)[r].to(dtype) for r in range(world)]

    def forward(self, tokens: list[torch.Tensor], kept: list | None = None) -> list[torch.Tensor]:
        """``tokens``: (n, width) of each rank, the same number on all, bfloat16 or float16.  ``kept``, an empty
        list, takes what :meth:`backward` needs of this pass; without it nothing stays behind."""
        if kept:
            raise ValueError("kept holds what another pass needs")
        sums = []
        for r, x in enumerate(self._gathered(tokens)):
            rank = self.ranks[r]
            logits = x.float() @ self.router.t()
            weights, experts = route(logits, self.k, bias=self.bias, **self.options)
            plan = assign(experts, self.own, r * self.own)
            u = product(x, rank["up"], plan, gather=True, dtype=x.dtype)
            h = F.silu(u)
            y = product(h, rank["down"], plan, dtype=x.dtype)
            # (a rank's part is rounded once more, to the type of the rows that it is made from)
            sums.append(combine(y, plan, weights).float())
            if kept is not None:
                kept.append((x, logits, weights, experts, plan, u, h, y))
        return self._summed(sums, tokens[0].dtype)

    def balance(self, kept: list, z: float = 0.0) -> list[Balance]:
        """The loss that keeps the experts in balance, of all ranks' tokens of the pass that has ``kept``: the same on every rank."""
        return [balance(logits, experts, score=self.options.get("score", "softmax"), z=z) for _, logits, _, experts, *_ in kept]

    def backward(self, grads: list[torch.Tensor], kept: list, *, loss_grads: list[torch.Tensor] | None = None,
                 balances: list[Balance] | None = None, z: float = 0.0) -> tuple[list[torch.Tensor], list[dict[str, torch.Tensor]]]:
        """From the outputs' gradients and what the forward pass that they belong to has ``kept``: each rank's tokens' and its weights'
        gradients (``up``, ``down`` of its own experts; ``router``, the same on all ranks).  ``loss_grads`` (the same
        number on every rank) are the gradients of the ``balances`` that :meth:`balance` found with ``z``."""
        if len(kept) != self.comm.world_size:
            raise ValueError("kept must be what a forward pass of this layer has left")
        if (loss_grads is None) != (balances is None):
            raise ValueError("loss_grads and balances come together")
        sums, found = [], []
        for r, d in enumerate(self._gathered(grads)):
            rank, (x, logits, weights, experts, plan, u, h, y) = self.ranks[r], kept[r]
            d_y, d_weights = combine_grad(d, y, plan, weights)
            d_h = product(d_y, rank["down_t"], plan, dtype=x.dtype)
            d_down = weight_grad(d_y, h, plan)
            s = torch.sigmoid(u.float())
            d_u = (d_h.float() * (s + u.float() * s * (1 - s))).to(x.dtype)
            d_up = weight_grad(d_u, x, plan, gather=True)
            # (pairs of other ranks' experts have no gradient here: the ranks' sums are the whole ones)
            d_logits = route_grad(d_weights, logits, experts, **self.grad_options)
            if balances is not None:
                # (a rank adds the loss's gradient at its own tokens, with all tokens' counts)
                own = slice(r * len(grads[r]), (r + 1) * len(grads[r]))
                d_logits[own] = balance_grad(loss_grads[r], logits[own], experts[own], balances[r], score=self.options.get("score", "softmax"), z=z, add=d_logits[own])
            d_x = combine(product(d_u, rank["up_t"], plan, dtype=x.dtype), plan)
            sums.append(d_x.float() + d_logits @ self.router)
            found.append({"up": d_up, "down": d_down, "router": d_logits.t() @ x.float()})
        self.comm.run(lambda r: allreduce(found[r]["router"], self.comm))
        return self._summed(sums, grads[0].dtype), found


class ExpertBlock:
    """A layer of experts with what stands around it.  Of a rank's residual ``stream`` (n, width) in float32:

        x = before(stream)
        y = layer(x) + silu(x @ up.T) @ down.T
        stream + gate * y, and after(that)

    ``up`` (inner, width) and ``down`` (width, inner) are a shared expert's weights, bfloat16 or float16 (the rows' type); ``gate`` (width,)
    scales the channels, ``before`` and ``after`` are the norms of this block's and of the next one's rows, with weights and biases or without.
    The layer's sum is rounded to the rows' type when the ranks hand it out, and y once more when the shared expert's is added (a result in 32 bits would
    need the next block's rows in 32 bits too), and the rows' gradient likewise on the way back.  ``z`` is :func:`~mintccl_amd.routing.balance`'s."""

    def __init__(self, layer: ExpertLayer, before: Norm, up: torch.Tensor, down: torch.Tensor, after: Norm, gate: torch.Tensor, z: float = 0.0) -> None:
        bare = lambda n: n._replace(**{v: t.detach() for v, t in (("weight", n.weight), ("bias", n.bias)) if t is not None})  # noqa: E731
        self.layer, self.comm, self.z = layer, layer.comm, z
        self.before, self.after, self.up, self.down, self.gate = bare(before), bare(after), up.detach(), down.detach(), gate.detach()

    def forward(self, streams: list[torch.Tensor], kept: list | None = None) -> tuple[list[torch.Tensor], list[torch.Tensor], list[Balance]]:
        """The new streams, the next block's rows and the balance losses of the ranks' streams (the same number of rows on all).  ``kept``,
        an empty list, takes what :meth:`backward` needs."""
        if kept:
            raise ValueError("kept holds what another pass needs")
        rows = [norm(s, self.before, dtype=self.up.dtype) for s in streams]
        of_layer: list = []
        routed = self.layer.forward(rows, of_layer)
        balances = self.layer.balance(of_layer, self.z)
        new, behind, of_block = [], [], []
        for stream, x, y in zip(streams, rows, routed):
            h, u = dense.product(x, self.up, activation="silu", keep=True)
            y = dense.product(h, self.down, residual=y, out=y)
            stream_out, x_out = join(stream, y, gate=self.gate, before=self.after)
            new.append(stream_out)
            behind.append(x_out)
            of_block.append((stream, x, u, h, y, stream_out))
        if kept is not None:
            kept.extend((of_layer, of_block, balances))
        return new, behind, balances

    def backward(self, d_streams: list[torch.Tensor], d_behind: list[torch.Tensor], d_losses: list[torch.Tensor],
                 kept: list) -> tuple[list[torch.Tensor], list[dict[str, torch.Tensor]]]:
        """From the gradients of :meth:`forward`'s three results (a loss's is a number in float32, the same on every rank): the streams' and the
        weights' (``before`` and ``before_bias``, ``after`` and ``after_bias`` where the norms have them, ``gate``, ``shared_up`` and ``shared_down``
        the same on all ranks, and the layer's)."""
        if len(kept) != 3 or len(kept[1]) != self.comm.world_size:
            raise ValueError("kept must be what a forward pass of this block has left")
        of_layer, of_block, balances = kept
        joined = [join_grad(d, d_x, new, y, gate=self.gate, before=self.after)
                  for d, d_x, (_, _, _, _, y, new) in zip(d_streams, d_behind, of_block)]
        d_rows, found = self.layer.backward([j.y for j in joined], of_layer, loss_grads=d_losses, balances=balances, z=self.z)
        d_in = []
        for j, d_x, f, (stream, x, u, h, _, _) in zip(joined, d_rows, found, of_block):
            d_u, _ = dense.activation_grad(dense.input_grad(j.y, self.down), u, "silu", bias=False)
            shared = dense.input_grad(d_u, self.up, dtype=torch.float32)
            n = norm_grad((d_x.float() + shared).to(x.dtype), stream, self.before)
            d_in.append(j.stream + n.x)
            own = {"before": n.weight, "before_bias": n.bias, "after": j.before_weight, "after_bias": j.before_bias, "gate": j.gate,
                   "shared_up": dense.weight_grad(d_u, x, dtype=torch.float32), "shared_down": dense.weight_grad(j.y, h, dtype=torch.float32)}
            f.update({name: t.float() for name, t in own.items() if t is not None})
        for name in own:
            if name in found[0]:
                self.comm.run(lambda r: allreduce(found[r][name], self.comm))  # noqa: B023
        return d_in, found


def plain_layer(x, router, up, down, k, bias=None, score="softmax", renormalise=True):
    """The layer on all tokens at once, in elementary operations of the inputs' type: what it is compared with."""
    logits = x @ router.t()
    key = logits if score == "softmax" else torch.sigmoid(logits)
    chosen = (key if bias is None else key + bias).sort(dim=-1, descending=True, stable=True).indices[:, :k]
    scores = torch.softmax(logits, -1) if score == "softmax" else torch.sigmoid(logits)
    weights = scores.gather(1, chosen)
    if renormalise:
        weights = weights / weights.sum(-1, keepdim=True)
    rows = torch.stack([F.silu(x @ u.t()) @ d.t() for u, d in zip(up, down)], 1)       # (tokens, experts, width)
    return (rows.gather(1, chosen[..., None].expand(-1, -1, rows.shape[2])) * weights[..., None]).sum(1)


def small_layer(world: int, device, tokens: int = 96, width: int = 320, inner: int = 200, experts: int = 16, seed: int = 1):
    """Weights, tokens and gradients of a small layer."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    experts = experts // world * world or world
    return {"router": (rand(experts, width) * width ** -0.5).to(device), "up": (rand(experts, inner, width) * width ** -0.5).to(device),
            "down": (rand(experts, width, inner) * inner ** -0.5).to(device),
            "tokens": [rand(tokens, width).to(torch.bfloat16).to(device) for _ in range(world)],
            "grads": [rand(tokens, width).to(torch.bfloat16).to(device) for _ in range(world)]}


def plain_block(stream, before, after, gate, router, up, down, shared_up, shared_down, k, z, dtype, bias=None, score="softmax", renormalise=True,
                kind="rms", before_bias=0.0, after_bias=0.0):
    """The block on all tokens at once, in elementary operations of the inputs' type: the new stream, the next block's rows and the loss.  What decides
    the choice of experts is rounded as the block rounds it, with the gradient of what is not."""
    def normed(x, weight, bias):
        x = x - x.mean(-1, keepdim=True) if kind == "layer" else x
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight + bias
    x = normed(stream, before, before_bias)
    x = x + (x.to(dtype).to(x.dtype) - x).detach()
    y = plain_layer(x, router, up, down, k, bias, score, renormalise) + F.silu(x @ shared_up.t()) @ shared_down.t()
    new = stream + gate * y
    logits = x @ router.t()
    shares = torch.softmax(logits, -1) if score == "softmax" else torch.sigmoid(logits)
    key = logits if score == "softmax" else shares
    chosen = (key if bias is None else key + bias).sort(dim=-1, descending=True, stable=True).indices[:, :k]
    often = torch.bincount(chosen.reshape(-1), minlength=len(router)) * (len(router) / chosen.numel())
    loss = (often * (shares / shares.sum(-1, keepdim=True)).mean(0)).sum() + z * torch.logsumexp(logits, -1).square().mean()
    return new, normed(new, after, after_bias), loss


def block_distances(world: int, device, kind: str = "rms", weights: bool = True, biases: bool = False, **options) -> dict[str, float]:
    """How far a small block's results and gradients are from the plain one's in 64 bits (2-norms; the loss's own distance).  Its norms are of
    a ``kind``, with ``weights`` and ``biases`` or without."""
    s, z = small_layer(world, device), 0.01
    g = torch.Generator().manual_seed(2)
    width, inner = s["up"].shape[2], 184
    rand = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    own = {"before": 1 + 0.2 * rand(width), "after": 1 + 0.2 * rand(width), "gate": 1 + 0.2 * rand(width),
           "shared_up": rand(inner, width) * width ** -0.5, "shared_down": rand(width, inner) * inner ** -0.5}
    own = {n: t.to(torch.bfloat16 if n.startswith("shared") else torch.float32).to(device) for n, t in own.items()}
    streams = [(t.float() * 3).contiguous() for t in s["tokens"]]
    d_streams = [rand(*t.shape).to(device) for t in streams]
    if biases:
        own.update({f"{n}_bias": (0.2 * rand(width)).to(device) for n in ("before", "after")})
    norms = [Norm(own[n] if weights else None, own.get(f"{n}_bias"), kind) for n in ("before", "after")]
    d_loss = torch.tensor(40.0, device=device)                                       # (so that it weighs about as much as the rest)
    layer = ExpertLayer(VirtualComm(world_size=world, device=device), s["router"], s["up"], s["down"], 4, **options)
    block = ExpertBlock(layer, norms[0], own["shared_up"], own["shared_down"], norms[1], own["gate"], z)
    kept: list = []
    new, behind, balances = block.forward(streams, kept)
    d_in, found = block.backward(d_streams, s["grads"], [d_loss] * world, kept)
    layer.comm.check()
    leaf = {n: t.double().requires_grad_() for n, t in {**own, **{n: s[n] for n in ("router", "up", "down")}}.items()}
    x = torch.cat(streams).double().requires_grad_()
    if not weights:
        leaf.update(before=1.0, after=1.0)
        own = {n: t for n, t in own.items() if n not in ("before", "after")}
    want = plain_block(x, **leaf, k=4, z=z, dtype=torch.bfloat16, kind=kind, **options)
    ((want[0] * torch.cat(d_streams)).sum() + (want[1] * torch.cat(s["grads"]).double()).sum() + want[2] * d_loss).backward()
    off = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    return {"stream": off(torch.cat(new), want[0].detach()), "rows": off(torch.cat(behind), want[1].detach()),
            "loss": max(off(b.loss, want[2].detach()) for b in balances), "streams' gradient": off(torch.cat(d_in), x.grad),
            **{n: off(torch.cat([f[n] for f in found]), leaf[n].grad) for n in ("up", "down")},
            **{f"{n} of rank {r}": off(f[n], leaf[n].grad) for r, f in enumerate(found) for n in ("router", *own)}}


def distances(world: int, device, **options) -> dict[str, float]:
    """How far a small layer's outputs and gradients are from the plain one's in 64 bits (2-norms)."""
    s = small_layer(world, device)
    layer = ExpertLayer(VirtualComm(world_size=world, device=device), s["router"], s["up"], s["down"], 4, **options)
    kept: list = []
    out = layer.forward(s["tokens"], kept)
    d_tokens, found = layer.backward(s["grads"], kept)
    layer.comm.check()
    leaf = {n: s[n].double().requires_grad_() for n in ("router", "up", "down")}
    x = torch.cat(s["tokens"]).double().requires_grad_()
    want = plain_layer(x, leaf["router"], leaf["up"], leaf["down"], 4, **options)
    want.backward(torch.cat(s["grads"]).double())
    off = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    return {"output": off(torch.cat(out), want.detach()), "tokens": off(torch.cat(d_tokens), x.grad),
            "up": off(torch.cat([f["up"] for f in found]), leaf["up"].grad),
            "down": off(torch.cat([f["down"] for f in found]), leaf["down"].grad),
            **{f"router of rank {r}": off(f["router"], leaf["router"].grad) for r, f in enumerate(found)}}


#: What 8 bits leave: a rounding is off by a sixteenth at most, 2.6 % of a number on the average; a path has two to six
#: of them one behind the other, and their errors are independent.
FAR = 0.12


def main() -> int:
    if not os.getenv("MINTCCL_TEST_MODE", ""):
        print("set MINTCCL_TEST_MODE=1 to run the self-test")
        return 0
    worst = distances(world_size_env(), torch.device("cuda:0"))
    worst.update({f"block's {n}": d for n, d in block_distances(world_size_env(), torch.device("cuda:0")).items()})
    for name, d in worst.items():
        print(f"# {name}: {d:.4f} off in 2-norm")
    return 0 if max(worst.values()) < FAR else 1


if __name__ == "__main__":
    import sys
    sys.exit(main())
