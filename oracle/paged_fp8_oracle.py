"""A paged cache of 8-bit floats, and heads' norms, in 64 bits on the CPU."""

from __future__ import annotations

import torch
from torch import Tensor

from .paged_oracle import rotate, spans

BLOCK = 32


def block_scales(x: Tensor) -> Tensor:
    """``[..., D / 32]``: the least of 2^-117 .. 2^119 by which each block's largest
    finite magnitude is at most 448."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    mantissa, exponent = torch.frexp(top / 448)  # top / 448 = mantissa 2^exponent, mantissa in [1/2, 1)
    power = torch.where(top == 0, -117, exponent - (mantissa == 0.5).int()).clamp(-117, 119)
    return torch.ldexp(torch.ones_like(top), power)


def rounded_to_e4m3(y: Tensor) -> Tensor:
    """The nearest E4M3 number, ties to even; NaN where ``y`` is not finite."""
    y = y.double()
    mag = y.abs().clamp(max=448)
    _, exponent = torch.frexp(mag)  # 2^(exponent - 1) <= mag
    step = torch.ldexp(torch.ones_like(mag), (exponent - 1).clamp(min=-6) - 3)
    out = torch.copysign(torch.round(mag / step) * step, y)
    return torch.where(torch.isfinite(y), out, torch.nan)


def quantised(x: Tensor, scales: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Codes' values and scales."""
    scales = block_scales(x) if scales is None else scales
    codes = rounded_to_e4m3(x.double() / scales.repeat_interleave(BLOCK, -1))
    return codes, scales


def values(codes: Tensor, scales: Tensor) -> Tensor:
    """What codes (float8_e4m3fn) and scales (float8_e8m0fnu) stand for."""
    return codes.to(torch.float32).double() * scales.to(torch.float32).double().repeat_interleave(BLOCK, -1)


def normed(x: Tensor, weight: Tensor | None, eps: float) -> Tensor:
    x = x.double()
    return x if weight is None else x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()


def placed(x: Tensor, seq_lens, cu_seqlens, weight=None, eps=1e-6, cos=None, sin=None, interleaved=False):
    """Heads ``[N, H, D]`` after norm and rotation, and each token's (sequence,
    position) or None."""
    out, at = normed(x, weight, eps), spans(seq_lens, cu_seqlens, x.shape[0])
    for t, where in enumerate(at):
        if where is None:
            out[t] = 0
        elif cos is not None:
            out[t] = rotate(out[t], where[1], cos, sin, interleaved)
    return out, at
