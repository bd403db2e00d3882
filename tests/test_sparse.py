"""Refusals, shapes and the token order of the attention over selected blocks, without a GPU."""

from __future__ import annotations

import ctypes
import importlib
import re
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


@pytest.fixture(scope="module")
def sp(pkg):
    return importlib.import_module("anima_flat_amd.kernels.sparse")


@pytest.fixture(scope="module")
def lib(pkg):
    if not pkg._lib.LIB_PATH.exists():
        pytest.skip("libanima_attn.so not built (run __graft_entry__.build())")
    return pkg._lib.lib()


def _meta(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_cpu_tensors(sp):
    q, blocks = torch.zeros(1, 4, 1, 128, dtype=BF), torch.zeros(1, 1, 1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors required"):
        sp.select_blocks(q, q, 1)
    with pytest.raises(ValueError, match="CUDA tensors required"):
        sp.sparse_attention(q, q, q, blocks)


def test_shapes(sp):
    q, k = _meta(2, 130, 6, 128), _meta(2, 70, 3, 128)
    blocks = sp.select_blocks(q, k, 5, _meta(2, dtype=torch.int32))
    assert blocks.shape == (2, 6, 3, 5) and blocks.dtype == torch.int32
    assert sp.sparse_attention(q, k, k, blocks).shape == (2, 130, 768)
    with FakeTensorMode():
        q, k = (torch.empty(1, 65, h, 128, dtype=BF, device="cuda", requires_grad=True) for h in (4, 2))
        blocks = sp.select_blocks(q, k, 3)
        out = sp.sparse_attention(q, k * 2, k, blocks)
        assert out.requires_grad and not blocks.requires_grad and blocks.shape == (1, 4, 2, 3)


@pytest.mark.parametrize("q,k,v,match", [
    ((2, 5, 128), (2, 5, 1, 128), (2, 5, 1, 128), "must be \\[B, Sq, H, hd\\]"),
    ((2, 5, 4, 128), (2, 5, 2, 128), (2, 6, 2, 128), "must be \\[B, Sq, H, hd\\]"),
    ((2, 5, 4, 128), (1, 5, 2, 128), (1, 5, 2, 128), "disagree on batch"),
    ((2, 5, 4, 128), (2, 5, 3, 128), (2, 5, 3, 128), "no multiple"),
    ((2, 5, 4, 128), (2, 5, 0, 128), (2, 5, 0, 128), "no multiple"),
    ((2, 5, 4, 64), (2, 5, 4, 64), (2, 5, 4, 64), "head_dim 64 is not supported"),
    ((2, 5, 4, 128), (2, 262145, 1, 128), (2, 262145, 1, 128), "at most 262144 keys"),
])
def test_refused_shapes(sp, q, k, v, match):
    blocks = _meta(2, 4, 1, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match=match):
        sp.sparse_attention(_meta(*q), _meta(*k), _meta(*v), blocks)
    if q[1:] != (5, 4, 128) or v == k:
        with pytest.raises(ValueError, match=match):
            sp.select_blocks(_meta(*q), _meta(*k), 1)


def test_refused_lists(sp):
    q, k = _meta(2, 65, 4, 128), _meta(2, 70, 2, 128)
    for shape in ((2, 4, 1, 3), (2, 2, 2, 3), (1, 4, 2, 3), (2, 4, 2, 0), (2, 4, 2, 4097), (2, 4, 2)):
        with pytest.raises(ValueError, match="blocks must be"):
            sp.sparse_attention(q, k, k, _meta(*shape, dtype=torch.int32))
    with pytest.raises(ValueError, match="blocks must be int32"):
        sp.sparse_attention(q, k, k, _meta(2, 4, 2, 3, dtype=torch.int64))
    for count in (0, -1, 4097):
        with pytest.raises(ValueError, match="count must be 1 to 4096"):
            sp.select_blocks(q, k, count)
    for lens in (_meta(3, dtype=torch.int32), _meta(2), _meta(2, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="seqused_k must be"):
            sp.select_blocks(q, k, 1, lens)
    with pytest.raises(ValueError, match="only bfloat16"):
        sp.select_blocks(_meta(2, 65, 4, 128, dtype=torch.float16), k, 1)


def test_library_refusals(pkg, lib):
    """Nothing is launched: every pointer below is never read."""
    L, fake = pkg._lib, 1 << 20
    strides = (1 << 15, 2048, 128)
    kinds = {
        "select": (L.BlockSelectArgs, lib.aa_block_select, ("q", "k")),
        "fwd": (L.SparseFwdArgs, lib.aa_sparse_fwd, ("q", "k", "v", "out")),
        "bwd": (L.SparseBwdArgs, lib.aa_sparse_bwd, ("dout", "q", "k", "v", "out", "dq", "dk", "dv")),
    }

    def call(kind, ws=fake, ws_bytes=1 << 40, **change):
        cls, fn, tensors = kinds[kind]
        a = cls(blocks=fake, B=1, Sq=4096, Sk=4096, H=16, Hk=4, hd=128, count=3)
        if kind == "bwd":
            a.lse = fake
        for name in tensors:
            setattr(a, name, fake)
            setattr(a, name + "_stride", L.c_strides(strides))
        for name, value in change.items():
            setattr(a, name, value)
        return fn(ctypes.byref(a), ws, ws_bytes, None)

    for kind, (_, fn, tensors) in kinds.items():
        assert fn(None, None, 0, None) == L.AA_EINVAL
        assert call(kind, B=0) == call(kind, Sq=0) == L.AA_OK
        assert call(kind, hd=64) == call(kind, dtype=1) == call(kind, count=0) == call(kind, count=4097) == L.AA_EUNSUPPORTED
        assert call(kind, Sk=262145) == call(kind, Sq=1 << 31) == call(kind, H=1 << 20, Hk=1) == L.AA_EUNSUPPORTED
        assert call(kind, H=15) == call(kind, Hk=0) == call(kind, Sk=-1) == L.AA_EINVAL
        assert call(kind, blocks=None) == L.AA_EINVAL
        for name in tensors:
            assert call(kind, **{name: None}) == call(kind, **{name: fake + 8}) == L.AA_EINVAL, (kind, name)
            assert call(kind, **{name + "_stride": L.c_strides((1 << 15, 2044, 128))}) == L.AA_EINVAL, (kind, name)
    assert call("bwd", B=1048575, Hk=8, Sq=1, Sk=1) == L.AA_EUNSUPPORTED
    assert call("select", ws=None) == call("select", ws_bytes=64) == call("select", ws=fake + 8) == L.AA_EINVAL
    assert call("bwd", ws=None) == call("bwd", ws_bytes=64) == call("bwd", ws=fake + 8) == call("bwd", lse=None) == L.AA_EINVAL
    for kind, names in (("fwd", ("k", "v")), ("bwd", ("dout", "q", "k", "v"))):
        for name in names:
            for bad in (-2048, 1 << 24):
                assert call(kind, **{name + "_stride": L.c_strides((1 << 15, bad, 128))}) == L.AA_EUNSUPPORTED


def test_workspaces(lib):
    assert lib.aa_block_select_workspace(2, 65, 64, 6, 3) == 2 * (6 * 2 + 3 * 1) * 128 * 8
    # No device here, so no split: 1 KB a query block, 8 bytes a key block and 64 query blocks.
    if not torch.cuda.is_available():
        assert lib.aa_sparse_bwd_workspace(2, 65, 130, 6, 3, 2) == 2 * 6 * (2 * 1024 + 3 * 8) + 2 * 3 * 3 * 512
        assert lib.aa_sparse_fwd_workspace(2, 65, 6, 100) == 0
    assert lib.aa_block_select_workspace(1, 64, 64, 3, 2) == lib.aa_sparse_bwd_workspace(1, 0, 64, 1, 1, 1) == 0
    assert lib.aa_sparse_bwd_workspace(1, 64, 64, 3, 2, 1) == lib.aa_sparse_fwd_workspace(0, 1, 1, 1) == 0


def test_structs_match_header(pkg):
    text = (Path(__file__).resolve().parents[1] / "include" / "anima_attn.h").read_text()
    L = pkg._lib
    for struct, cls in (("aa_block_select_args", L.BlockSelectArgs), ("aa_sparse_fwd_args", L.SparseFwdArgs), ("aa_sparse_bwd_args", L.SparseBwdArgs)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S)[1], flags=re.S)
        assert [f[0] for f in cls._fields_] == re.findall(r"([A-Za-z_0-9]+)(?:\[\d+\])?\s*[,;]", body)


@pytest.mark.parametrize("h,w", [(16, 24), (8, 8), (13, 21), (1, 5), (64, 9)])
def test_tile_order(sp, h, w):
    order, back = sp.tile_order(h, w)
    x = torch.arange(h * w)
    assert torch.equal(x[order].sort()[0], x) and torch.equal(x[order][back], x)
    if h % 8 == 0 and w % 8 == 0:
        y, c = x[order].view(-1, 64) // w, x[order].view(-1, 64) % w
        assert ((y // 8) == (y[:, :1] // 8)).all() and ((c // 8) == (c[:, :1] // 8)).all()
        assert torch.equal(x[order][:3], torch.tensor([0, 1, 2])) and x[order][8] == w


def test_captured_training_without_the_extension(pkg, sp, monkeypatch):
    """The Python autograd setups cannot look for a live eager graph: they refuse a captured
    forward with gradients, and an op call that kept no statistics."""
    from types import SimpleNamespace

    rotary = importlib.import_module("anima_flat_amd.kernels.rotary")
    x, t, blocks = torch.zeros(1, 4, 1, 128, dtype=BF), torch.zeros(4, 64), torch.zeros(1, 1, 1, 1, dtype=torch.int32)
    cases = [
        ("rotary", rotary._rotary_setup, (x, None, t, t, False, False), (x, x[:0])),
        ("sparse_attention", sp._sparse_setup, (x, x, x, blocks, None, True), (x, t)),
    ]
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    for name, setup, inputs, output in cases:
        saved = []
        needs = tuple(isinstance(i, torch.Tensor) and i.dtype == BF for i in inputs)
        ctx = SimpleNamespace(needs_input_grad=needs, set_materialize_grads=lambda on: None, mark_non_differentiable=lambda *a: None,
                              save_for_backward=lambda *a: saved.append(a))
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match=f"{name}: .* only with the torch extension"):
            setup(ctx, inputs, output)
        assert not saved
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        setup(ctx, inputs, output)
        assert saved
    with pytest.raises(RuntimeError, match="keeps its statistics"):
        sp._sparse_setup(ctx, (x, x, x, blocks, None, False), (x, t))
