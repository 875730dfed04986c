"""Dense matrix products in 16 and 32 bits with bias, activation and residual, and
their gradients.

What an expert layer has beside its experts (the router, an expert that all tokens
share) and what stands around it.  Sums are in 32 bits.  Gradients are calls of
their own, as in :mod:`~mintccl_amd.routing`: with z what the activation was applied to,

    out, z = product(x, w, bias=b, activation="silu", residual=r, keep=True)
    d_z, d_b = activation_grad(d_out, z, "silu")
    d_x, d_w = input_grad(d_z, w), weight_grad(d_z, x)

(the residual's is that of the result).  No counterpart in the reference.
"""
from __future__ import annotations

import torch

from . import _lib
from .common import DTYPE_CODE

#: ``gelu`` by the normal distribution, ``gelu_tanh`` its approximation by a hyperbolic tangent
ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "sigmoid": 3, "tanh": 4, "gelu": 5, "gelu_tanh": 6}


def _activation(name: str | None) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be None or one of {', '.join(a for a in ACTIVATIONS if a)}: got {name!r}")
    return ACTIVATIONS[name]


def _code(dtype: torch.dtype | None) -> int | None:
    if dtype is not None and dtype not in DTYPE_CODE:
        raise TypeError("products come in float16, bfloat16 or float32")
    return None if dtype is None else DTYPE_CODE[dtype]


def product(x: torch.Tensor, weight: torch.Tensor, *, bias: torch.Tensor | None = None, activation: str | None = None,
            residual: torch.Tensor | None = None, keep: bool = False, dtype: torch.dtype | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``residual + activation(x @ weight.T + bias)``, rounded once: of ``dtype`` (x's type if none is named, or
    float32) or into ``out``.

    ``x`` (rows, depth) and ``weight`` (cols, depth) are of one type: float32, bfloat16 or float16, rows any
    distance apart; ``bias`` (cols,) of that type, ``residual`` (rows, cols) of the result's (it may be ``out`` itself).
    With ``keep`` what the activation is applied to comes back too, in x's type: what the gradients need."""
    return _lib.experts().dense_product(x, weight, bias, _activation(activation), residual, keep, _code(dtype), out)


def activation_grad(grad: torch.Tensor, z: torch.Tensor | None, activation: str | None = None, *, bias: bool = True,
                    dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The gradient in front of the activation, of z's type, and with ``bias`` the bias's, its sum over rows before it is
    rounded, from the result's ``grad`` (of z's type or float32).  Without an activation ``z`` may be ``None`` and
    ``dtype`` names the operands' type (grad's if none is named); grad itself comes back where that is its own."""
    return _lib.experts().activation_grad(grad, z, _activation(activation), bias, _code(dtype))


def input_grad(grad: torch.Tensor, weight: torch.Tensor, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``grad @ weight``: x's gradient, of ``dtype`` (grad's type if none is named, or float32)."""
    return _lib.experts().dense_input_grad(grad, weight, _code(dtype))


def weight_grad(grad: torch.Tensor, x: torch.Tensor, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``grad.T @ x``: the weight's gradient, of ``dtype`` (grad's type if none is named, or float32)."""
    return _lib.experts().dense_weight_grad(grad, x, _code(dtype))
