"""64-bit formulas of the rotary operators, shared by their tests."""

from __future__ import annotations

import math

import torch

U32 = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}  # half a step below the normal range


def frequencies(dims, theta, scale, scaling, original):
    """[(axis, radians per position)] and the factor of both tables."""
    out, factor = [], 1.0
    for axis, d in enumerate(dims):
        for i in range(d // 2):
            base, s = theta[axis], scale[axis]
            if scaling == "ntk" and d > 2:
                base = base * s ** (d / (d - 2))
            f = base ** (-2.0 * i / d)
            if scaling == "linear":
                f /= s
            if scaling == "yarn":
                keep = min(1.0, max(0.0, (original * f / (2 * math.pi) - 1) / 31))
                f = keep * f + (1 - keep) * f / s
            out.append((axis, f))
    if scaling == "yarn":
        factor = 1 + 0.1 * math.log(max(scale))
    return out, factor


def tables(positions, dims, theta, scale, scaling, original=None):
    """cos and sin in float64, [..., pairs]."""
    pairs, factor = frequencies(dims, theta, scale, scaling, original)
    angle = torch.stack([positions[..., axis].double() * f for axis, f in pairs], -1)
    return angle.cos() * factor, angle.sin() * factor, factor


def turn(x, cos, sin, interleaved):
    """x (any dtype) turned in float64, and the size of the summands of each value."""
    part = 2 * cos.shape[-1]
    i = torch.arange(part // 2, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + part // 2)
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    x = x.detach().double()
    y, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    size[..., lo], size[..., hi] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def turn_bound(ref, size, dtype):
    """Two fp32 roundings of the summands, one of the result to its type."""
    return 2 * U32 * size + HALF[dtype] * (ref.abs() + 2 * U32 * size) + TINY[dtype]
