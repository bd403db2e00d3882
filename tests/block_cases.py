"""Inputs and error bounds shared by the tests of the block's operators.

Bounds. u = 2^-24 is half a step of float32, 2^-8 of bfloat16, both relative. A float32 sum of
n terms in any order is off by at most (depth) u sum |terms|, depth the longest chain of
additions: at most 32 in a lane and 9 across lanes and waves in the norms, taken as 44 with
the products' own roundings.
"""

from __future__ import annotations

import torch

U32 = 2.0**-24
U16 = 2.0**-8
BF = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def bf(g, *shape, scale=1.0, device="cuda"):
    return (torch.randn(*shape, generator=g) * scale).to(device, BF)


def within(actual, ref, bound, name):
    """|actual - ref| <= bound everywhere (ref, bound float64 of actual's device)."""
    a = actual.detach().double()
    assert a.shape == ref.shape, f"{name}: {tuple(a.shape)} != {tuple(ref.shape)}"
    if a.numel() == 0:
        return
    over = ((a - ref).abs() - bound).flatten()
    worst = int(over.argmax())
    assert torch.isfinite(a).all(), f"{name}: not finite"
    assert over[worst] <= 0, (
        f"{name}: {a.flatten()[worst].item():.9g} against {ref.flatten()[worst].item():.9g}, "
        f"bound {bound.expand_as(ref).flatten()[worst].item():.3g}"
    )


def norm_bounds(p):
    """Condition of each row: how much larger the summands are than what is left of them. The
    mean is off by 44 u size, so r - mean by 47 u size, rstd by a relative 40 u + 94 u cond."""
    cond = p["size"].amax(-1, keepdim=True) * p["rstd"]
    xh = U32 * (47 * cond + p["xh"].abs() * (44 + 94 * cond))
    return cond, xh
