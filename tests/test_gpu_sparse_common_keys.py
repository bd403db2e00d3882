"""dQ where keys have much in common: its correction beside rows that are not finite."""

from __future__ import annotations

import importlib
import math

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


@pytest.mark.parametrize("sq,bad", [(64, range(0, 16)), (64, range(48, 64)), (64, [5]), (70, [69]), (33000, [32999]), (33000, range(0, 16))])
@pytest.mark.parametrize("where", ["q", "dout"])
def test_other_rows_keep_their_digits(sp, sq, bad, where):
    """A query or gradient that is not finite spoils its own row of dq; the others stay as exact
    as they are."""
    g = gen(63)
    sk = 256
    q, v, dout = heads(g, 1, sq, 1), heads(g, 1, sk, 1), heads(g, 1, sq, 1)
    k = (8 * heads(g, 1, 1, 1).float() + heads(g, 1, sk, 1).float()).to(BF)
    blocks = torch.arange(4, dtype=torch.int32, device="cuda").expand(1, 1, -(-sq // 64), 4).contiguous()
    ref = attend(q, k, v, blocks, None, dout)[0]["dq"]
    spoilt = {"q": q.clone(), "dout": dout.clone()}
    spoilt[where][0, list(bad)] = math.nan
    got = _dq(sp, spoilt["q"], k, v, blocks, spoilt["dout"])
    assert torch.isnan(got[0, list(bad)]).all()
    for i in bad:
        # The rows that share a matrix instruction's lanes with it, and all of its block.
        first = i // 64 * 64
        for rows in ([first + (i - first + 16) % 64], [first + (i - first + 48) % 64], range(first, first + 64)):
            rows = [r for r in rows if r < sq and r not in bad]
            if rows:
                assert (got[0, rows] - ref[0, rows]).norm() <= TWO_ROUNDINGS * ref[0, rows].norm(), (i, rows)
