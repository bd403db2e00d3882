"""dQ where the keys end in the first half of a block: the mean key of its correction."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import gen
from sparse_cases import BF, attend, heads

pytestmark = pytest.mark.gpu

# Two roundings, of dz and of dq, of half a step of 2^-8 each (what the keys have in common
# would multiply the first, uncorrected: about 25 in a thousand below).
TWO_ROUNDINGS = 2 * 2.0**-8


@pytest.fixture(scope="module")
def sp(pkg):
    return importlib.import_module("anima_flat_amd.kernels.sparse")


def _dq(sp, q, k, v, blocks, dout):
    q = q.clone().requires_grad_(True)
    return torch.autograd.grad(sp.sparse_attention(q, k, v, blocks), [q], dout.flatten(2))[0].double()


@pytest.mark.parametrize("sk", [84, 64 * 3 + 20, 64 * 5 + 1, 128, 64 * 2 + 50])
@pytest.mark.parametrize("sq", [64, 33000])
def test_keys_that_end_in_the_first_half_of_a_block(sp, sq, sk):
    """The weights are in the second half of the last whole block, whose mean key is as far from
    the others' as can be: the mean that is taken off has to be that block's own."""
    g = gen(64)
    m, e = torch.randn(128, generator=g), torch.randn(128, generator=g)
    e /= e.norm()
    m -= (m @ e) * e
    last = (sk - 1) // 64 * 64
    near = torch.zeros(sk, dtype=torch.bool)
    near[last - 64 : last] = True
    heavy = torch.zeros(sk, dtype=torch.bool)
    heavy[last - 32 : last] = True
    k = torch.randn(sk, 128, generator=g) + torch.where(near, 8.0, -8.0)[:, None] * m
    k -= 20 * (~heavy)[:, None] * e  # a score 17 lower
    q = torch.randn(sq, 128, generator=g)
    q += 10 * e - (q @ m)[:, None] * m / (m @ m)
    q, k = (t.to("cuda", BF)[None, :, None] for t in (q, k))
    v, dout = heads(g, 1, sk, 1), heads(g, 1, sq, 1)
    nk = -(-sk // 64)
    blocks = torch.arange(nk, dtype=torch.int32, device="cuda").expand(1, 1, -(-sq // 64), nk).contiguous()
    ref = attend(q, k, v, blocks, None, dout)[0]["dq"]
    assert (_dq(sp, q, k, v, blocks, dout) - ref).norm() <= TWO_ROUNDINGS * ref.norm()
