"""gelu8's float32 arithmetic: before the one rounding to bf16 it is within 2e-6 of GELU and its
slope (relative, where the exponential's argument is small), so that the results are those of the
64-bit formula rounded once but for values within that of a tie.

The fit is off by 8e-7; the exponential's argument x^2 / 2 log2(e) by two roundings of 2^-24 of
itself, the reciprocal and the exponential by 2^-22 each, the other steps by at most 6 roundings:
(2 + x^2) 2^-23 + 10 * 2^-24 in all beside the fit.
"""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import BF
from oracle import block_oracle as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="session")
def ckpt8(pkg):
    return importlib.import_module("anima_flat_amd.kernels.ckpt8")


def _half_step(v):
    """Half of bf16's step at v: 2^-9 of the power of two above."""
    return torch.exp2((torch.frexp(v)[1].double() - 9).clamp(min=-134))


def _error(x):
    return 8e-7 + (2 + x * x) * 2.0**-23 + 10 * 2.0**-24


def test_forward(ckpt8):
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    x = x[torch.isfinite(x) & (x.float() > -12.5)].float()
    x = torch.cat([x, torch.zeros(-len(x) % 8)]).to(BF).view(1, 1, -1).cuda()
    y = ckpt8.gelu8(x).double()
    want = ref.gelu(x.double())
    bound = _half_step(want) + _error(x.double().clamp(-13, 13)) * want.abs() + 2.0**-133
    over = ((y - want).abs() > bound).sum().item()
    assert over == 0, over


def test_backward(ckpt8):
    """dy = 1: the slope, rounded once. Its error is relative to Phi and to x phi, its two terms."""
    x = torch.linspace(-8, 8, 1 << 16).to(BF).view(1, -1, 64).cuda().requires_grad_(True)
    (dx,) = torch.autograd.grad(ckpt8.gelu8(x), [x], torch.ones_like(x))
    kept = ref.checkpoint(x.detach()[0])[2][None]
    want = ref.gelu_slope(kept)
    terms = ref.normal_cdf(-kept.abs()) + (kept.abs() * torch.exp(-0.5 * kept * kept)) * 0.3989422804014327
    bound = _half_step(want) + _error(kept) * terms + 2.0**-23 * want.abs()
    over = ((dx.double() - want).abs() > bound).sum().item()
    assert over == 0, over
