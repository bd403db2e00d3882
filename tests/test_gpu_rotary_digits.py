"""Digits of the rotary tables: the error that the kernel's own arithmetic has, no library's.

The angle's rest r in quarter turns, |r| <= 1/2, is rounded to fp32 once: 2^-26, 2.4e-8 of an
angle. The polynomials as coded, their coefficients rounded to fp32, are off by 2.2e-8 (sine; 3.4e-8
of it) and 0.6e-8 (cosine) in exact arithmetic. In fp32, with u = 2^-24 half a step of 1, the
sine rounds y = r r (a share of 0.08 u reaches the value), the last two sums (r u = 0.5 u and
r y u / 2 = 0.06 u) and the product (0.5 u): 1.14 u; the cosine y (0.31 u) and the last three
sums (0.5 u, 0.25 u and 0.01 u): 1.07 u. Together 1.15e-7 and 0.88e-7.
"""

from __future__ import annotations

import importlib
import math

import pytest
import torch

from block_cases import within

pytestmark = pytest.mark.gpu

U = 2.0**-24
SIN = 2.0**-26 * math.pi / 2 + 2.2e-8 + 1.14 * U
COS = 2.0**-26 * math.pi / 2 * math.sin(math.pi / 4) + 0.6e-8 + 1.07 * U


@pytest.fixture(scope="module")
def rot(pkg):
    return importlib.import_module("anima_flat_amd.kernels.rotary")


@pytest.mark.parametrize("turns", [0, 1, 2, 3, -1, 40, -100])
def test_every_rest_of_a_quarter(rot, turns):
    """One pair of frequency 1: the positions are the angles. The product with 2 / pi in 64 bits
    is off by 3 2^-53 of up to 160 radians."""
    angle = (turns + torch.linspace(-0.5, 0.5, 1 << 20, dtype=torch.float64, device="cuda")) * (math.pi / 2)
    cos, sin = rot.rotary_tables(angle, 2)
    # (Angles on a border between quarters fall to either side: sine and cosine change places.)
    sure = torch.where(angle.cos().abs() < angle.sin().abs(), COS, SIN), torch.where(angle.cos().abs() < angle.sin().abs(), SIN, COS)
    border = ((angle.cos().abs() - angle.sin().abs()).abs() < 1e-9)[..., None]
    most = max(SIN, COS)
    within(sin[:, 0], angle.sin(), torch.where(border[:, 0], most, sure[0]) + 1e-13, "sin")
    within(cos[:, 0], angle.cos(), torch.where(border[:, 0], most, sure[1]) + 1e-13, "cos")
