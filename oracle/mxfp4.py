"""Microscaled 4-bit floating point in 64 bits on the CPU, from its definition:
32 values of a row share 2^(floor(log2(largest |value|)) - 2), each is the
nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code) times it."""
from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(x: torch.Tensor):
    """(codes uint8 [..., R, C], one a value; scales uint8 [..., R, ceil(C / 32)])."""
    x = x.detach().cpu().double()
    C = x.shape[-1]
    blocks = torch.nn.functional.pad(x, (0, -C % 32)).unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    power = torch.frexp(top).exponent.long() - 3
    power = torch.where(top == 0, -127, power.clamp(min=-127))
    finite = torch.isfinite(top)
    scales = torch.where(finite, power + 127, 255).to(torch.uint8)
    v = (blocks / torch.exp2(power.double())[..., None]).abs()
    distance = (v[..., None] - GRID).abs()
    # among two that are equally near the even code: those come first in this order
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[distance[..., order].argmin(-1)] + 8 * torch.signbit(blocks)
    return code.flatten(-2)[..., :C].to(torch.uint8), scales


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What (codes, scales) stand for."""
    v = GRID[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    return v * s.repeat_interleave(32, -1)[..., :codes.shape[-1]]


def quantized(x: torch.Tensor) -> torch.Tensor:
    return values(*quantize(x))


def linear(x, w, dy):
    """(y, dx, dw) of the linear layer whose three products quantise their operands
    along the dimension they sum over."""
    y = quantized(x) @ quantized(w).T
    dx = quantized(dy) @ quantized(w.T).T
    dw = quantized(dy.T) @ quantized(x.T).T
    return y, dx, dw
