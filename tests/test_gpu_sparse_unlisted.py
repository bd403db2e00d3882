"""What a list does not name stays out of the gradients, also beside the end of the keys."""

from __future__ import annotations

import importlib
import math

import pytest
import torch

from block_cases import gen
from sparse_cases import heads

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sp(pkg):
    return importlib.import_module("anima_flat_amd.kernels.sparse")


@pytest.mark.parametrize("sq", [70, 33000])
@pytest.mark.parametrize("sk,listed", [(70, [1]), (95, [1]), (96, [1]), (97, [1]), (20, [0]), (300, [1, 4]), (1500, list(range(0, 22)) + [23])])
def test_unlisted_rows_are_not_read(sp, sq, sk, listed):
    """NaN in every row of blocks that no list names changes no bit; sq: lists split over
    workgroups where they are long, and not."""
    g = gen(61)
    q, k, v, dout = heads(g, 1, sq, 2), heads(g, 1, sk, 1), heads(g, 1, sk, 1), heads(g, 1, sq, 2)
    blocks = torch.tensor(listed, dtype=torch.int32, device="cuda").expand(1, 2, -(-sq // 64), len(listed)).contiguous()
    named = torch.zeros(-(-sk // 64), dtype=torch.bool)
    named[listed] = True
    out_of = ~named.repeat_interleave(64)[:sk]
    results = []
    for bad in (None, math.nan, math.inf):
        kk, vv = (t.clone() for t in (k, v))
        if bad is not None:
            kk[0, out_of], vv[0, out_of] = bad, bad
        leaves = [t.requires_grad_(True) for t in (q.clone(), kk, vv)]
        out = sp.sparse_attention(*leaves, blocks)
        results.append([out, *torch.autograd.grad(out, leaves, dout.flatten(2))])
    assert all(torch.isfinite(t).all() for t in results[0])
    for name, *same in zip(("out", "dq", "dk", "dv"), *results):
        assert all(torch.equal(same[0], t) for t in same[1:]), name


def test_rows_past_the_length_beside_an_unlisted_block(sp):
    """Lengths that end in the first rows of a block whose neighbour no list names."""
    g = gen(62)
    lens = [70, 128 + 31, 192 + 33, 5]
    B, sk = len(lens), 300
    q, k, v, dout = heads(g, B, 64, 1), heads(g, B, sk, 1), heads(g, B, sk, 1), heads(g, B, 64, 1)
    blocks = torch.tensor([[(n - 1) // 64] for n in lens], dtype=torch.int32, device="cuda").view(B, 1, 1, 1)
    seqused = torch.tensor(lens, dtype=torch.int32, device="cuda")
    results = []
    for bad in (False, True):
        kk, vv = (t.clone() for t in (k, v))
        for b, n in enumerate(lens):
            if bad:
                first = (n - 1) // 64 * 64
                for t in (kk, vv):
                    t[b, :first], t[b, n:] = math.nan, math.nan
        leaves = [t.requires_grad_(True) for t in (q.clone(), kk, vv)]
        out = sp.sparse_attention(*leaves, blocks, seqused)
        results.append([out, *torch.autograd.grad(out, leaves, dout.flatten(2))])
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(*results))
