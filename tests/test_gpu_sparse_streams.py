"""Gradients of the attention over selected blocks on two streams at once."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import gen
from sparse_cases import heads, random_blocks

pytestmark = pytest.mark.gpu


def test_gradients_on_two_streams(pkg):
    """Lists of queries and of keys split over workgroups on one stream (their partial sums share
    a workspace), whole ones on the other: the bits of each alone."""
    sparse = importlib.import_module("anima_flat_amd.kernels.sparse")
    lib = pkg._lib.lib()
    g = gen(68)
    sets = []
    for B, Sq, Sk, H, Hk, count in ((1, 1000, 1900, 2, 1, 20), (1, 34000, 4500, 2, 2, 3)):
        q, k, v, dout = heads(g, B, Sq, H), heads(g, B, Sk, Hk), heads(g, B, Sk, Hk), heads(g, B, Sq, H)
        blocks = random_blocks(g, B, H, Sq, Sk, count)
        sets.append(([t.requires_grad_(True) for t in (q, k, v)], blocks, dout.flatten(2)))
        # Statistics, turned lists and mean keys alone; with partial sums there is more.
        nq, nk = -(-Sq // 64), -(-Sk // 64)
        whole = B * H * (nq * 1024 + nk * -(-nq // 64) * 8) + B * Hk * nk * 512
        split = lib.aa_sparse_bwd_workspace(B, Sq, Sk, H, Hk, count) - (whole + 15) // 16 * 16
        assert (split > 0) == (lib.aa_sparse_fwd_workspace(B, Sq, H, count) > 0) == (Sq == 1000)

    def step(leaves, blocks, dout):
        out = sparse.sparse_attention(*leaves, blocks)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for stream, s, to in zip(streams, sets, got):
            with torch.cuda.stream(stream):
                to.append(step(*s))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for steps, ref in zip(got, want) for one in steps for a, b in zip(one, ref))
