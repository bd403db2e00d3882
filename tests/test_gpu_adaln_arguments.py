"""adaln_bwd's native kernel refuses what its Python function refuses."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import bf, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("change,says", [
    ({"stats": lambda t: t["stats"].t().contiguous()}, "those of the forward"),
    ({"stats": lambda t: t["stats"].flatten()}, "those of the forward"),
    ({"stats": lambda t: t["stats"].view(2, -1, 4)}, "those of the forward"),
    ({"y": lambda t: None}, "belong together"),
    ({"y": lambda t: None, "weight": lambda t: None}, "belong together"),
])
def test_refused(pkg, change, says):
    importlib.import_module("anima_flat_amd.kernels.adaln")
    ops = torch.ops.anima_flat_amd
    g = gen(1)
    x, y, dr, dh = (bf(g, 2, 10, 64) for _ in range(4))
    m, w = bf(g, 2, 64), bf(g, 64).float()
    stats = ops.residual_adaln(x, y, m, m, m, w, 1e-6, 1.0, True)[2]
    t = dict(dr=dr, dh=dh, x=x, y=y, gate=m, scale=m, weight=w, stats=stats, shift_rows=2, branch_scale=1.0, mods=True)
    assert ops.adaln_bwd(**t)[0].shape == x.shape
    with pytest.raises(ValueError, match=says):
        ops.adaln_bwd(**(t | {k: f(t) for k, f in change.items()}))
