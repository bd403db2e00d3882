"""Copies of groups whose largest magnitude is in bf16's last power of two, 2^127 and above."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import BF, U16, U32, bf, gen, within
from oracle import block_oracle as ref

pytestmark = pytest.mark.gpu

TOP = [2.0**127, -(2.0**127) * 1.9921875, 1.5 * 2.0**127]  # the first and last of it, one between


@pytest.fixture(scope="session")
def ckpt8(pkg):
    return importlib.import_module("anima_flat_amd.kernels.ckpt8")


def _rows(rows, K, seed):
    """Ordinary rows, every third with one to three of TOP among small and large neighbours."""
    g = gen(seed)
    x = torch.randn(rows, K, generator=g)
    x[1::3] *= torch.exp2(torch.randint(100, 124, (1, K), generator=g).float())
    for i, v in enumerate(TOP):
        x[i::3, (5 * i + 3) % K] = v
    return x.to(BF)[None].cuda()


@pytest.mark.parametrize("rows,K", [(5, 8), (37, 72), (300, 256)])
def test_gelu8(ckpt8, rows, K):
    """dx = dy or 0 far from the origin and dy / 2 where a group's step leaves nothing: exact."""
    x = _rows(rows, K, rows).requires_grad_(True)
    dy = bf(gen(K), 1, rows, K)
    (dx,) = torch.autograd.grad(ckpt8.gelu8(x), [x], dy)
    kept = ref.checkpoint(x.detach()[0])[2][None]
    assert torch.isfinite(kept).all() and (kept.abs() > 2.0**126).any()
    far = (kept == 0) | (kept.abs() > 2.0**90)
    slope = torch.where(kept == 0, 0.5, (kept > 0).double())
    assert torch.equal(dx.double()[far], (dy.double() * slope)[far])
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("rows,K,R", [(5, 8, 8), (37, 72, 16), (300, 256, 40), (900, 264, 64)])
def test_lora_down8(ckpt8, rows, K, R):
    """dA against the formula, of gradients small enough for its sums: 2^-20 times 2^128."""
    g = gen(R)
    x = _rows(rows, K, R)
    a = bf(g, R, K).requires_grad_(True)
    dt = bf(g, 1, rows, R, scale=2.0**-20)
    (da,) = torch.autograd.grad(ckpt8.lora_down8(x, a), [a], dt)
    kept, dtd = ref.checkpoint(x[0])[2], dt.double()[0]
    want = dtd.t() @ kept
    within(da, want, U16 * want.abs() + (rows + 8) * U32 * (dtd.abs().t() @ kept.abs()), "da")
