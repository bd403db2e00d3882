"""The block's ops keep the contract of torch.library: inputs unchanged, no output that is an
input's or another output's memory, fakes of the same shapes, types and layout."""

from __future__ import annotations

import importlib

import pytest
import torch

from test_gpu_block_native import _cases

pytestmark = pytest.mark.gpu


def test_contract(pkg):
    for module in ("adaln", "int8", "ckpt8"):
        importlib.import_module("anima_flat_amd.kernels." + module)
    for name, calls in _cases().items():
        for args in calls:
            torch.library.opcheck(getattr(torch.ops.anima_flat_amd, name).default, args, test_utils=("test_schema", "test_faketensor"))
