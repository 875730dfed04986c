"""Norms before and after a block of a model, with the residual stream, a gate and
a residual scale, and their gradients.

What stands around a layer of experts (or any other block): the stream that
passes it by is normalised in front of it (:func:`norm`), and its output is taken
into the stream, behind a norm of its own and a gate where it has them, while the new
stream is normalised for the next block (:func:`join`: both in one pass).
Statistics and sums are in 32 bits.  Gradients are calls of their own, as in
:mod:`~mintccl_amd.routing`.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .common import DTYPE_CODE

KINDS = {"rms": 1, "layer": 2}
GATES = {None: 0, "silu": 2, "sigmoid": 3, "tanh": 4}


class Norm(NamedTuple):
    """A norm of rows: ``(x - m) * q * weight + bias``.  ``rms``: m = 0 and q = 1 / sqrt(mean x**2 + eps); ``layer``: m = mean x
    and q = 1 / sqrt(mean (x - m)**2 + eps)."""
    weight: torch.Tensor | None          #: (width,) in float32, bfloat16 or float16; none: ones
    bias: torch.Tensor | None = None     #: (width,) of the weight's type; none: zeros
    kind: str = "rms"
    eps: float = 1e-6


class NormGrad(NamedTuple):
    x: torch.Tensor                      #: of x's type
    weight: torch.Tensor | None          #: of the weight's
    bias: torch.Tensor | None


class JoinGrad(NamedTuple):
    """Of each its own shape and type; ``None`` for what :func:`join` did not have."""
    stream: torch.Tensor
    y: torch.Tensor
    gate: torch.Tensor | None
    after_weight: torch.Tensor | None
    after_bias: torch.Tensor | None
    before_weight: torch.Tensor | None
    before_bias: torch.Tensor | None


_NONE = (0, None, None, 0.0)


def _norm(n: Norm | None) -> tuple:
    if n is None:
        return _NONE
    if n.kind not in KINDS:
        raise ValueError(f"kind must be one of {', '.join(KINDS)}: got {n.kind!r}")
    return KINDS[n.kind], n.weight, n.bias, n.eps


def _gate(name: str | None) -> int:
    if name not in GATES:
        raise ValueError(f"gate_by must be None or one of {', '.join(g for g in GATES if g)}: got {name!r}")
    return GATES[name]


def _code(dtype: torch.dtype | None) -> int | None:
    if dtype is not None and dtype not in DTYPE_CODE:
        raise TypeError("norms come in float16, bfloat16 or float32")
    return None if dtype is None else DTYPE_CODE[dtype]


def norm(x: torch.Tensor, of: Norm, *, dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The norm of the rows of ``x`` (rows, width), in float32, bfloat16 or float16 and any distance apart: of ``dtype``, which is x's, or
    anything if x is in float32, or into ``out`` (which may be x itself)."""
    if of is None:
        raise TypeError("of must be a Norm")
    if out is not None and dtype is None:
        dtype = out.dtype
    return _lib.experts().join(x, None, None, 0, 1.0, 1.0, *_NONE, *_norm(of), _code(dtype), out)[1]


def norm_grad(grad: torch.Tensor, x: torch.Tensor, of: Norm) -> NormGrad:
    """The gradients of ``norm(x, of)`` from its result's ``grad``."""
    if of is None:
        raise TypeError("of must be a Norm")
    d = _lib.experts().join_grad(None, grad, x, None, None, 0, 1.0, 1.0, *_NONE, *_norm(of))
    return NormGrad(d[0], d[5], d[6])


def join(stream: torch.Tensor, y: torch.Tensor, *, after: Norm | None = None, gate: torch.Tensor | None = None,
         gate_by: str | None = None, scale: float = 1.0, carry: float = 1.0, before: Norm | None = None,
         out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The stream behind a block, ``carry * stream + scale * a(gate) * u`` with u the block's output ``y``
    or ``after`` of it, and its norm ``before`` the next block, of y's type (``None`` without).

    ``stream`` and ``y`` are (rows, width), rows any distance apart; the stream is of
    y's type or in float32.  ``gate`` has a number for each channel (width,), each row (rows, 1) or
    each number (rows, width), and ``gate_by`` is what is applied to it first: sigmoid, tanh, silu or nothing.  The new
    stream may go to ``out``, also to ``stream`` itself; it is rounded once, and the norm is of
    the stream as it is stored."""
    return _lib.experts().join(stream, y, gate, _gate(gate_by), scale, carry, *_norm(after), *_norm(before), None, out)


def join_grad(grad: torch.Tensor | None, grad_before: torch.Tensor | None, stream: torch.Tensor, y: torch.Tensor, *,
              after: Norm | None = None, gate: torch.Tensor | None = None, gate_by: str | None = None, scale: float = 1.0,
              carry: float = 1.0, before: Norm | None = None) -> JoinGrad:
    """The gradients of :func:`join` with these options from those of its two results (either may be ``None``: zeros);
    ``stream`` is the NEW one, as it came back."""
    if y is None:
        raise TypeError("y must be a device tensor")
    return JoinGrad(*_lib.experts().join_grad(grad, grad_before, stream, y, gate, _gate(gate_by), scale, carry, *_norm(after),
                                              *_norm(before)))
