"""What the backward cannot take is refused by the forward that keeps statistics for it."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib(pkg):
    if not pkg._lib.LIB_PATH.exists():
        pytest.skip("libanima_attn.so not built (run __graft_entry__.build())")
    return pkg._lib.lib()


# B, Sq, Sk, H, Hk: more than a launch of the turned lists, of these and the mean keys, and of the
# blocks of keys holds.
TOO_MANY = [(1048576, 1, 1, 16, 1), (1048575, 1, 1, 16, 8), (300000, 1, 4096, 1, 1), (1 << 20, 64, 64 * 4096, 1, 1)]


@pytest.mark.parametrize("size", TOO_MANY)
def test_forward_with_statistics(pkg, lib, size):
    """Nothing is launched: the pointers are never read."""
    L, fake = pkg._lib, 1 << 20
    codes = []
    for cls, fn, tensors in ((L.SparseFwdArgs, lib.aa_sparse_fwd, ("q", "k", "v", "out")),
                             (L.SparseBwdArgs, lib.aa_sparse_bwd, ("dout", "q", "k", "v", "out", "dq", "dk", "dv"))):
        a = cls(blocks=fake, lse=fake, count=1, hd=128, **dict(zip(("B", "Sq", "Sk", "H", "Hk"), size)))
        for name in tensors:
            setattr(a, name, fake)
            setattr(a, name + "_stride", L.c_strides((2048, 2048, 128)))
        codes.append(fn(ctypes.byref(a), fake, 1 << 50, None))
        assert b"too many" in lib.aa_last_error()
    assert codes == [L.AA_EUNSUPPORTED] * 2
