"""Training with queries whose tokens lie far apart."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import gen
from sparse_cases import BF, heads, random_blocks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sp(pkg):
    return importlib.import_module("anima_flat_amd.kernels.sparse")


@pytest.mark.parametrize("stride", [1 << 24, (1 << 24) - 8, (1 << 24) + 1024])
def test_queries_far_apart(sp, stride):
    """The forward takes any sequence stride of the queries, and so does a step."""
    g = gen(65)
    S, H = 70, 2
    q, k, dout = heads(g, 1, S, H), heads(g, 1, 100, H), heads(g, 1, S, H)
    blocks = random_blocks(g, 1, H, S, 100, 2)
    store = torch.empty((S - 1) * stride + H * 128, dtype=BF, device="cuda")
    wide = store.as_strided(q.shape, (stride, stride, 128, 1)).copy_(q)
    wide_dout = torch.empty_like(store).as_strided(q.shape, (stride, stride, 128, 1)).copy_(dout)
    results = []
    for x, d in ((q, dout), (wide, wide_dout)):
        x = x.detach().requires_grad_(True)
        out = sp.sparse_attention(x, k, k, blocks)
        results.append([out, *torch.autograd.grad(out.unflatten(2, (H, 128)), [x], d)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_keys_far_apart_are_refused(sp):
    """Before anything is computed, with and without gradients."""
    g = gen(66)
    q = heads(g, 1, 5, 1)
    far = torch.empty((1 << 24) + 128, dtype=BF, device="cuda").as_strided((1, 2, 1, 128), (1 << 24, 1 << 24, 128, 1))
    blocks = torch.zeros(1, 1, 1, 1, dtype=torch.int32, device="cuda")
    for needs in (False, True):
        with pytest.raises(ValueError, match="sequence stride of k or v"):
            sp.sparse_attention(q.detach().requires_grad_(needs), far, far, blocks)
