"""Routing of tokens to experts, its gradient, the assignment of the chosen
pairs to places in the experts' order, and the loss that keeps the experts in balance.

What stands in front of the experts of a layer that is spread over ranks: from
a token's logits, the experts it goes to and their weights (``route``), and
where each pair of a token and an expert stands when the pairs are sorted by
expert (``assign``), which is what :mod:`~mintccl_amd.block8`'s products by
expert and :mod:`~mintccl_amd.combine` go by.  Nothing is recorded for automatic
differentiation: gradients are calls of their own, and a tensor that requires one is
refused unless it is detached or gradients are off, as is one with a tangent of
forward-mode differentiation.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

SCORES = {"softmax": 0, "sigmoid": 1}


class Assignment(NamedTuple):
    """Pairs of a token and an expert in the experts' order."""
    offsets: torch.Tensor    #: (experts + 1) int32: where each expert's places begin, and their end
    tokens: torch.Tensor     #: (tokens * k) int32: the token at each place; -1 behind the end
    slots: torch.Tensor      #: (tokens, k) int32: the place of each pair; -1 where it is no expert's


class Balance(NamedTuple):
    """How a batch's tokens are spread over the experts."""
    loss: torch.Tensor       #: () float32
    counts: torch.Tensor     #: (sequences, experts) int32: the choices of each expert
    shares: torch.Tensor     #: (sequences, experts) float32: each expert's share of a token's scores, on the average
    there: torch.Tensor      #: (sequences,) int32: tokens that have an expert left


def _score(name: str) -> int:
    if name not in SCORES:
        raise ValueError(f"score must be one of {', '.join(SCORES)}: got {name!r}")
    return SCORES[name]


def route(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          kept: int = 1, group_top: int = 1, renormalise: bool = True,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights (tokens, k) in float32 and experts (tokens, k) in int32.

    ``logits`` (tokens, experts) in float32, bfloat16 or float16, rows any
    distance apart; at most 1024 experts, ``k`` at most 64.  A token's scores s
    are the softmax or the sigmoid of its logits x.  The choice goes by x +
    ``bias`` (softmax) or s + ``bias`` (sigmoid; the bias balances the experts and
    is in no weight): of ``groups`` groups of consecutive experts the ``kept``
    ones whose ``group_top`` (1 or 2) largest have the largest sum, and of these
    the k largest, the lowest expert first among equals.  The weights are
    ``scale`` times the chosen ones' s, divided by the sum of these where
    ``renormalise`` is true.

    A logit of -inf masks its expert: where fewer than k are left, the expert is
    -1 and the weight 0.  A NaN ranks above every number, and shows in the
    weights."""
    return _lib.experts().route(logits, k, _score(score), bias, groups, kept, group_top, renormalise, scale)


def route_grad(grad: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, *, score: str = "softmax",
               renormalise: bool = True, scale: float = 1.0) -> torch.Tensor:
    """The logits' gradient, in their type, from the weights' ``grad`` (tokens, k)
    in float32, for the ``experts`` that :func:`route` chose with these options.
    (The choice, and so the bias, has none.)"""
    return _lib.experts().route_grad(grad, logits, experts, _score(score), renormalise, scale)


def assign(experts: torch.Tensor, count: int, first: int = 0) -> Assignment:
    """The pairs of ``experts`` (tokens, k) sorted by expert, those of an expert in
    their own order.  Only the experts ``first .. first + count - 1`` take part:
    the ones that a rank has; the other pairs have no place."""
    return Assignment(*_lib.experts().assign(experts, count, first))


def balance(logits: torch.Tensor, experts: torch.Tensor, *, score: str = "softmax", offsets: torch.Tensor | None = None,
            z: float = 0.0) -> Balance:
    """The loss that keeps experts in balance, and the counts and shares that it is made of.

    ``logits`` (tokens, experts) as for :func:`route`, ``experts`` (tokens, k) int32 what was chosen by them (-1: none).  A
    token's shares p are the softmax of its logits, or their sigmoids divided by the sum of these.  For a sequence of n tokens that
    have an expert left (a logit above -inf), an expert counted c times has the load f = experts * c / (k * n) and the mean
    share P; the loss is the sum of f * P over the experts, its mean over the sequences that have such a token, plus ``z`` times the
    mean over all these tokens of the squared log of their logits' exponentials' sum.  It is 1 where all is even.
    ``offsets`` (sequences + 1) int32, at most 65535 sequences, says where each begins, and the end; tokens outside count nowhere, and
    without it all tokens are one sequence.

    The counts are whole numbers, and their sum over ranks is that of all ranks' tokens: put into the place of a rank's own
    (with ``there``'s), :func:`balance_grad` takes the load of all of them."""
    return Balance(*_lib.experts().balance(logits, experts, _score(score), offsets, z))


def balance_grad(grad: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, found: Balance, *, score: str = "softmax",
                 offsets: torch.Tensor | None = None, z: float = 0.0, add: torch.Tensor | None = None) -> torch.Tensor:
    """The logits' gradient, in their type, from the loss's ``grad`` (one float32 on the device), for what
    :func:`balance` ``found`` with these options; the choice, and so the counts, have none.  ``add``, the logits'
    gradient from elsewhere (:func:`route_grad`), is added before the sum is rounded."""
    return _lib.experts().balance_grad(grad, logits, experts, _score(score), offsets, z, found.counts, found.there, add)
