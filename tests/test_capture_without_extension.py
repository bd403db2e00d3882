"""The Python autograd setups of the block's ops, which run where the torch extension does not:
they cannot look for a live eager graph, so a captured forward with gradients is refused."""

from __future__ import annotations

import importlib
from types import SimpleNamespace

import pytest
import torch

BF = torch.bfloat16


def _setups():
    adaln, ckpt8 = (importlib.import_module("anima_flat_amd.kernels." + n) for n in ("adaln", "ckpt8"))
    x, m, low = torch.zeros(1, 4, 64, dtype=BF), torch.zeros(1, 64), torch.zeros(1, 4, 8, dtype=BF)
    a, stats, none = torch.zeros(8, 64, dtype=BF), torch.zeros(4, 4), torch.zeros(0)
    return {
        "residual_adaln": (adaln._residual_adaln_setup, (x, x, m, m, m, None, 1e-6, 1.0, True), (x, x, stats)),
        "adaln": (adaln._adaln_setup, (x, m, m, 1e-6, True), (x, stats)),
        "gelu8": (ckpt8._gelu8_setup, (x, True), (x, none, none)),
        "lora_down8": (ckpt8._lora_down8_setup, (x, a, True), (low, none, none)),
    }


@pytest.mark.parametrize("name", ["residual_adaln", "adaln", "gelu8", "lora_down8"])
def test_refused(pkg, monkeypatch, name):
    setup, inputs, output = _setups()[name]
    saved = []
    ctx = SimpleNamespace(needs_input_grad=(True,) * len(inputs), set_materialize_grads=lambda on: None,
                          save_for_backward=lambda *t: saved.append(t))
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match=f"{name}: .* only with the torch extension"):
        setup(ctx, inputs, output)
    assert not saved
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    setup(ctx, inputs, output)
    assert saved
