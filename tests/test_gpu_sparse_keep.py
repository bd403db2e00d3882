"""sparse_fwd called without its statistics where a gradient is needed."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import gen
from sparse_cases import heads

pytestmark = pytest.mark.gpu


def test_a_call_that_needs_gradients_keeps_its_statistics(pkg):
    """The op refuses it as its Python autograd does; its fake has no statistics either."""
    importlib.import_module("anima_flat_amd.kernels.sparse")
    op = torch.ops.anima_flat_amd.sparse_fwd
    q = heads(gen(67), 1, 70, 1)
    blocks = torch.zeros(1, 1, 2, 1, dtype=torch.int32, device="cuda")
    for i in range(3):
        args = [q, q.clone(), q.clone()]
        args[i] = args[i].clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="keeps its statistics"):
            op(*args, blocks, None, False)
        with torch.no_grad():
            assert op(*args, blocks, None, False)[1].shape == (0,)
        out, lse = op(*args, blocks, None, True)
        assert out.requires_grad and not lse.requires_grad and lse.shape == (1, 1, 70)
