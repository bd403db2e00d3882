"""The backward operators take only copies of the shape that their own forward makes."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import bf, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,K", [(16, 96), (32, 256), (48, 72)])
def test_the_other_operators_copy(pkg, rows, K):
    """gelu8's exponents are [rows, groups], lora_down8's [groups, rows]: as many bytes where the
    rows are a multiple of 16, in another order."""
    importlib.import_module("anima_flat_amd.kernels.ckpt8")
    ops = torch.ops.anima_flat_amd
    g = gen(rows)
    x, a, dt = bf(g, 1, rows, K), bf(g, 16, K), bf(g, 1, rows, 16)
    _, codes, exps = ops.gelu8(x, True)
    _, lcodes, lexps = ops.lora_down8(x, a, True)
    assert exps.numel() == lexps.numel() and codes.shape == lcodes.shape
    with pytest.raises(ValueError, match="those of the forward"):
        ops.gelu8_bwd(x, lcodes, lexps)
    with pytest.raises(ValueError, match="those of the forward"):
        ops.lora_down8_bwd(dt, a, codes, exps, True, True)
    for wrong in (codes.t(), codes.view(-1)[None], codes[None]):
        with pytest.raises(ValueError, match="those of the forward"):
            ops.gelu8_bwd(x, wrong.contiguous(), exps)
    assert ops.gelu8_bwd(x, codes, exps).shape == x.shape
    assert ops.lora_down8_bwd(dt, a, lcodes, lexps, True, True)[1].shape == a.shape
