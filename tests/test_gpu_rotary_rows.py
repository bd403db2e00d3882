"""As many positions as the tables' entry point takes."""

from __future__ import annotations

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_most_positions(pkg):
    """2^32 - 1 of one pair: 4 bytes each in, 8 out, 52 GB in all."""
    rot = importlib.import_module("anima_flat_amd.kernels.rotary")
    rows, step = (1 << 32) - 1, 1 << 30
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    positions = torch.zeros(rows, dtype=torch.int32, device="cuda")
    at = torch.tensor([0, 5, step - 1, step, 2 * step - 1, 2 * step, 3 * step - 1, 3 * step, rows - 2, rows - 1], device="cuda")
    positions[at] = torch.arange(1, 11, dtype=torch.int32, device="cuda")
    cos, sin = rot.rotary_tables(positions, 2)
    assert cos.shape == sin.shape == (rows, 1)
    want = rot.rotary_tables(positions[at], 2)
    assert torch.equal(cos[at], want[0]) and torch.equal(sin[at], want[1])
    for i in range(0, rows, step):  # every other position is 0
        part = slice(i, min(i + step, rows))
        here = ((at >= i) & (at < i + step)).sum().item()
        assert (sin[part] != 0).sum().item() == (cos[part] != 1).sum().item() == here
    del positions, cos, sin
    torch.cuda.empty_cache()
    with pytest.raises(ValueError, match="too many positions"):
        rot.rotary_tables(torch.empty(1, dtype=torch.int32, device="cuda").expand(rows + 1).contiguous(), 2)
    torch.cuda.empty_cache()
