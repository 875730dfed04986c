"""Definitions of the expert layer's products in 64 bits, on the device that the operands are on, and how far sums
may be from them."""
from __future__ import annotations

import torch

#: Half the relative distance of neighbouring numbers of a type: what one rounding does; and what a number below its normal range may be off.
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
#: Results in bf16 come from instructions that cut each of eight products off at 2^-13 of the largest one's power of two: seven of
#: them lose less than that each, and the largest one is at most the eight magnitudes' sum.
CUT = 7 * 2.0 ** -13


def randn(*shape, seed, dtype=torch.float32, scale=1.0, dev="cpu"):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev)


def rounded8(x: torch.Tensor, dim: int) -> torch.Tensor:
    """The numbers, in 64 bits, that ``x`` stands for when it is rounded to 8 bits in blocks of 128 along ``dim``: a block's scale and the
    numbers' factor are quotients in 32 bits."""
    x = x.float().movedim(dim, -1)
    n = x.shape[-1]
    full = torch.zeros(*x.shape[:-1], -(-n // 128) * 128, device=x.device)
    full[..., :n] = x
    full = full.unflatten(-1, (-1, 128))
    most = full.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -96)
    largest = torch.full_like(most, 448.0)
    q = (full * (largest / most)).to(torch.float8_e4m3fn).float().double()
    return (q * (most / largest).double()).flatten(-2)[..., :n].movedim(-1, dim)


def weight64(w) -> torch.Tensor:
    """What 8-bit weights and their squares' scales stand for."""
    q, s = w.q.float().double(), w.scale.double()
    return q * s.repeat_interleave(128, -2)[..., :q.shape[-2], :].repeat_interleave(128, -1)[..., :q.shape[-1]]


def off_by(got, x, w, blocks=None):
    """How far ``got`` is from x w^T beyond what it may be; nothing where that is zero or less.

    A result in bf16 may lose ``CUT`` of its magnitudes' sum.  Else products are exact, and of the sums' additions (128 of a
    block's, one for each block) every one rounds by 2^-24 of the partial sum, which is at most the magnitudes' sum: independent of each other,
    so they add up in quadrature, of which four times is allowed; four more for the scales' products and the block's.  Then one
    rounding to the result's type."""
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    blocks = -(-x.shape[1] // 128) if blocks is None else blocks
    extra = size * (4 * (128 + blocks) ** 0.5 + 4) * 2.0 ** -24
    if got.dtype == torch.bfloat16:
        extra = extra + size * CUT
    allowed = extra + (want.abs() + extra) * HALF_ULP[got.dtype] * 1.001 + TINY[got.dtype]
    over = (got.double() - want).abs() - allowed
    beyond = (want.abs() + allowed > torch.finfo(got.dtype).max) & (got.double() == want.sign() * torch.inf)     # (of a 16-bit float's range)
    over = torch.where(beyond, 0.0, over)
    return float(over.nan_to_num(nan=float("inf")).max()) if over.numel() else 0.0


def unlike(rows: int, depth: int, seed: int = 0):
    """x (rows, depth) and w(cols) of whole numbers that are 8-bit numbers as they are, whose products are as unlike as they can be and whose
    sums are whole numbers: in a block of 128 the first product of each eight is 2^16 or -2^16 in turn, the seven others are small ones that
    lie just below 2^-13 of it.  (16 numbers of a block are for its scale.)  Returns x and a function of ``cols``."""
    at = torch.arange(depth)
    lead, first = at % 8 == 0, at % 128 < 16
    sign = torch.where(at // 8 % 2 == 0, 1.0, -1.0)
    small = torch.tensor([1.75, 1.5, 1.25, 1.0])
    x = torch.where(lead, 256.0, 0.0) + torch.where(lead, 0.0, 1.0) * small[(torch.arange(rows) + seed) % 4][:, None]
    x = torch.where(first, torch.where(at % 128 == 0, 448.0, 0.0), x)          # 448: the block's scale is 1

    def weights(cols: int):
        few = torch.tensor([4.0, -4.0, 2.0])[(torch.arange(cols) + seed) % 3][:, None]
        w = torch.where(lead, 256.0 * sign, few.expand(cols, depth))
        return torch.where(first, torch.where(at % 128 == 1, 448.0, 0.0), w)
    return x, weights
