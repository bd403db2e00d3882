"""The block's differentiable operators on fake tensors that require grad: shapes and a graph,
without a GPU."""

from __future__ import annotations

import importlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


@pytest.mark.parametrize("name", ["residual_adaln", "adaln", "gelu8", "lora_down8"])
def test_forward_with_gradients(pkg, name):
    adaln, ckpt8 = (importlib.import_module("anima_flat_amd.kernels." + n) for n in ("adaln", "ckpt8"))
    with FakeTensorMode():
        x = torch.empty(2, 5, 64, dtype=BF, device="cuda", requires_grad=True)
        m, a = torch.empty(2, 64, device="cuda", requires_grad=True), torch.empty(8, 64, dtype=BF, device="cuda", requires_grad=True)
        out = {
            "residual_adaln": lambda: adaln.residual_adaln(x * 2, x, m, m, m)[1], "adaln": lambda: adaln.adaln(x, m, m),
            "gelu8": lambda: ckpt8.gelu8(x + x), "lora_down8": lambda: ckpt8.lora_down8(x, a),
        }[name]()
        assert out.shape == (2, 5, 8 if name == "lora_down8" else 64) and out.dtype == BF and out.requires_grad
