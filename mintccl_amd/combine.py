"""The combination of the experts' rows: a token's rows, added up with its weights,
and the gradients of both (calls of their own, as in :mod:`~mintccl_amd.routing`).  No counterpart in the reference."""
from __future__ import annotations

import torch

from . import _lib
from .routing import Assignment


def combine(rows: torch.Tensor, plan: Assignment, weights: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """(tokens, width): the sum of each token's ``rows`` (places, width) times its
    ``weights`` (tokens, k) in float32 (1 where there are none), in 32 bits,
    rounded once to the rows' type.  A pair without a place adds nothing.  Without
    weights this is also the gradient of a gathered product's input from
    the gradient of its rows."""
    return _lib.experts().combine(rows, plan.slots, weights, out)


def combine_grad(grad: torch.Tensor, rows: torch.Tensor, plan: Assignment,
                 weights: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The gradients of the rows, in their type (zeros behind the last expert's places,
    where no row is a token's), and of the weights in float32 (``None`` without weights) from the result's."""
    return _lib.experts().combine_grad(grad, rows, plan.offsets, plan.slots, weights)
