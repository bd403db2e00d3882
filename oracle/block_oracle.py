"""64-bit restatement of the block's operators (kernels.adaln, kernels.int8, kernels.ckpt8).

Plain torch in float64 on the device of its inputs; gradients come from autograd of these
functions. The two quantisers are restated in the number formats they are defined in.
"""

from __future__ import annotations

import math

import torch

GROUP = 32


def norm_parts(x, y, gate, scale, shift, weight, eps, branch_scale=1.0):
    """r, h and the intermediate values of residual_adaln; y None: adaln. gate, scale, shift
    are [B or 1, D]; everything in float64."""
    n = y
    if weight is not None:
        n = y * (y.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * weight
    branch = 0 if y is None else branch_scale * gate[:, None] * n
    r = x + branch
    centred = r - r.mean(-1, keepdim=True)
    rstd = (centred.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xh = centred * rstd
    h = xh * (1 + scale[:, None]) + shift[:, None]
    size = x.abs() if y is None else x.abs() + branch.abs()
    return {"r": r, "h": h, "n": n, "xh": xh, "rstd": rstd, "size": size}


def residual_adaln(x, y, gate, scale, shift, weight=None, eps=1e-6, branch_scale=1.0):
    p = norm_parts(x, y, gate, scale, shift, weight, eps, branch_scale)
    return p["r"], p["h"]


def int8_rows(y32):
    """Codes (int8) and scales (float32 [rows]) of float32 rows: the scale rounded to float32, the
    code 127 y / max in float64 (127 y exact, and a tie's quotient too) to an integer. On the
    CPU: torch's GPU division by a constant multiplies by a rounded reciprocal."""
    dev, y32 = y32.device, y32.cpu()
    amax = y32.abs().amax(-1)
    m = amax.clamp_min(1e-12)
    s = m / 127
    bad = ~torch.isfinite(y32).all(-1)
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    q = torch.round(127 * y32.double() / m.double().unsqueeze(-1))
    return torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q).to(dev, torch.int8), s.reshape(-1).to(dev)


def gelu(x):
    return x * normal_cdf(x)


def normal_cdf(x):
    return 0.5 * torch.special.erfc(-x / math.sqrt(2.0))


def gelu_slope(x):
    return normal_cdf(x) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def checkpoint(x):
    """Codes [rows, 32 G] (int8), exponent bytes [rows, G] (uint8) and kept values [rows, K]
    (float64) of bfloat16 rows."""
    rows, K = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -K % GROUP)).unflatten(1, (-1, GROUP))
    amax = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    top = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))[1]  # 2^(top - 1) <= amax < 2^top
    e = torch.where(amax == 0, torch.full_like(top, 1), (top - 7 + 127).clamp_min(1))
    step = ((e.long() - 127 + 1023) << 52).view(torch.float64)  # 2^(e - 127), by its bits
    codes = torch.round(torch.where(bad[..., None], torch.zeros_like(v), v) / step[..., None]).clamp(-127, 127)
    kept = torch.where(bad[..., None], torch.full_like(v, math.nan), codes * step[..., None])
    exps = torch.where(bad, torch.full_like(e, 255), e)
    return codes.flatten(1).to(torch.int8), exps.to(torch.uint8), kept.flatten(1)[:, :K]
