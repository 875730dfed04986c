"""A layer of experts spread over the ranks of a communicator, forward and
backward: the expert layer's operators and the collectives as they are used
together.

Every rank has some of the experts and some of the tokens.  All tokens are
gathered on all ranks (``allgather``); each rank routes them, makes the rows of its
own experts (``route``, ``assign``, ``product``), adds up each token's rows
(``combine``) and hands the sums to the tokens' owners (``reducescatter``).  The way
back is the same the other way round: the gradient of a reduce-scatter is an allgather, that
of an allgather a reduce-scatter.  No token is dropped, and no row is sent that is not used.

    MINTCCL_TEST_MODE=1 python -m mintccl_amd.experts

runs a small layer on virtual ranks and compares it with the plain one.  No
counterpart in the reference.
"""
from __future__ import annotations

import os

import torch
import torch.nn.functional as F

from .allgather import allgather
from .allreduce import allreduce
from .block8 import product, quantise_weight, transposed, weight_grad
from .combine import combine, combine_grad
from .common import VirtualComm, world_size_env
from .reducescatter import reducescatter
from .routing import assign, route, route_grad


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

    def backward(self, grads: list[torch.Tensor], kept: list) -> tuple[list[torch.Tensor], list[dict[str, torch.Tensor]]]:
        """From the outputs' gradients and what the forward pass that they belong to has ``kept``: each rank's tokens' and its weights'
        gradients (``up``, ``down`` of its own experts; ``router``, the same on all ranks)."""
        if len(kept) != self.comm.world_size:
            raise ValueError("kept must be what a forward pass of this layer has left")
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
            d_x = combine(product(d_u, rank["up_t"], plan, dtype=x.dtype), plan)
            sums.append(d_x.float() + d_logits @ self.router)
            found.append({"up": d_up, "down": d_down, "router": d_logits.t() @ x.float()})
        self.comm.run(lambda r: allreduce(found[r]["router"], self.comm))
        return self._summed(sums, grads[0].dtype), found


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
    for name, d in worst.items():
        print(f"# {name}: {d:.4f} off in 2-norm")
    return 0 if max(worst.values()) < FAR else 1


if __name__ == "__main__":
    import sys
    sys.exit(main())
