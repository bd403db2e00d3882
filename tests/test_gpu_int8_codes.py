"""Int8 codes against the rule in 64 bits: round(127 y / max|y|) to nearest even, every tie as the
rule has it. A bf16 value at half its row's largest magnitude is such a tie."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import BF, bf, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="session")
def mods(pkg):
    return [importlib.import_module("anima_flat_amd.kernels." + n) for n in ("adaln", "int8")]


def _rule(y):
    """Codes of rows of bf16 values above 1e-12, in exact arithmetic: 127 y has 15 bits, and its
    quotient by the row's largest is a tie or 2^-17 (relative) away from one."""
    y = y.cpu().double()
    return torch.round(127 * y / y.abs().amax(-1, keepdim=True)).to(torch.int8)


@pytest.mark.parametrize("S,K", [(300, 264), (666, 1024), (64, 4096), (33, 8192)])
def test_tokens(mods, S, K):
    g = gen(S + K)
    x = bf(g, 2, S, K, scale=3.0)
    q, s = mods[1].rowquant_int8(x)
    assert torch.equal(q.cpu(), _rule(x))
    assert torch.equal(s.view(2, S).cpu(), x.cpu().float().abs().amax(-1) / 127)


def test_every_largest_value(mods):
    """Rows for each bf16 mantissa as the largest magnitude, over all of the exponent's range:
    every mantissa at 0 to 9 powers of two below it, both signs."""
    top = (128 + torch.arange(128.0))[:, None, None]
    below = (128 + torch.arange(128.0)) * torch.exp2(-torch.arange(10.0))[:, None]
    row = torch.where(below <= top, below, below / 2).flatten(1)
    row = torch.cat([row, -row, top[..., 0], torch.zeros(128, 7)], 1)
    for e in (-40, -7, 0, 60, 119):
        x = (row * 2.0**e).to(BF)
        assert torch.equal(x.double(), row.double() * 2.0**e)
        q, _ = mods[1].rowquant_int8(x[None].cuda())
        assert torch.equal(q[0].cpu(), _rule(x)), e


def test_weights(mods):
    w = bf(gen(1), 512, 2048, scale=2048**-0.5)
    q, s = mods[1].quantize_weight(w)
    assert torch.equal(q.cpu(), _rule(w)) and torch.equal(s.cpu(), w.cpu().float().abs().amax(-1) / 127)


@pytest.mark.parametrize("D", [264, 2048, 8192])
def test_norm(mods, D):
    """With a scale of -1 the norm's output is the shift, exactly."""
    g = gen(D)
    x, y, shift = bf(g, 64, 2, D), bf(g, 64, 2, D), bf(g, 64, D)
    one = torch.ones(1, D, dtype=BF, device="cuda")
    _, q, _ = mods[0].residual_adaln_int8(x, y, one, -one, shift)
    assert torch.equal(q.cpu(), _rule(shift)[:, None].expand(-1, 2, -1))
