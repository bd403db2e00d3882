"""Refusals and shapes of the rotary operators, without a GPU."""

from __future__ import annotations

import ctypes
import importlib
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


@pytest.fixture(scope="module")
def rot(pkg):
    return importlib.import_module("anima_flat_amd.kernels.rotary")


@pytest.fixture(scope="module")
def lib(pkg):
    if not pkg._lib.LIB_PATH.exists():
        pytest.skip("libanima_attn.so not built (run __graft_entry__.build())")
    return pkg._lib.lib()


def _meta(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_cpu_tensors(rot):
    t = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA tensors required"):
        rot.rotary(torch.zeros(1, 4, 1, 16), t, t)
    with pytest.raises(ValueError, match="CUDA tensors required"):
        rot.rotary_tables(torch.arange(4), 16)


def test_shapes(rot):
    t = _meta(2, 5, 6, dtype=torch.float32)
    q, k = rot.rotary_qk(_meta(2, 5, 4, 16), _meta(2, 5, 1, 16), t, t, True)
    assert q.shape == (2, 5, 4, 16) and k.shape == (2, 5, 1, 16) and q.dtype == k.dtype == BF
    assert rot.rotary(_meta(2, 5, 4, 16), t, t).shape == (2, 5, 4, 16)
    cos, sin = rot.rotary_tables(_meta(3, 7, dtype=torch.int64), 10)
    assert cos.shape == sin.shape == (3, 7, 5) and cos.dtype == torch.float32
    assert rot.rotary_tables(_meta(7, 2, dtype=torch.int32), (4, 6))[1].shape == (7, 5)


def test_fake_tensors_with_gradients(rot):
    with FakeTensorMode():
        q, k = (torch.empty(1, 5, h, 32, dtype=BF, device="cuda", requires_grad=True) for h in (4, 2))
        t = torch.empty(5, 16, device="cuda")
        out = rot.rotary_qk(q * 2, k, t, t)
        assert out[0].requires_grad and out[1].shape == k.shape


@pytest.mark.parametrize("q,k,t,match", [
    ((2, 5, 4), (2, 5, 1, 16), (5, 4), "must be \\[B, S, H, hd\\]"),
    ((2, 5, 4, 16), (2, 6, 1, 16), (5, 4), "one batch, length"),
    ((2, 5, 4, 16), (2, 5, 1, 24), (5, 4), "one batch, length"),
    ((2, 5, 4, 20), (2, 5, 1, 20), (5, 4), "multiple of 8"),
    ((2, 5, 4, 520), (2, 5, 1, 520), (5, 4), "multiple of 8, at most 512"),
    ((2, 5, 4, 16), (2, 5, 1, 16), (4, 4), "cos and sin must be"),
    ((2, 5, 4, 16), (2, 5, 1, 16), (3, 5, 4), "cos and sin must be"),
    ((2, 5, 4, 16), (2, 5, 1, 16), (5, 9), "turn 2 to head_dim"),
    ((2, 5, 4, 16), (2, 5, 1, 16), (5, 0), "turn 2 to head_dim"),
])
def test_refused_turns(rot, q, k, t, match):
    table = _meta(*t, dtype=torch.float32)
    with pytest.raises(ValueError, match=match):
        rot.rotary_qk(_meta(*q), _meta(*k), table, table)


def test_refused_types(rot):
    t = _meta(5, 4, dtype=torch.float32)
    with pytest.raises(ValueError, match="unsupported dtype"):
        rot.rotary(_meta(2, 5, 4, 16, dtype=torch.float64), t, t)
    with pytest.raises(ValueError, match="unsupported dtype"):
        rot.rotary_qk(_meta(2, 5, 4, 16), _meta(2, 5, 4, 16, dtype=torch.float16), t, t)
    with pytest.raises(ValueError, match="must be float32"):
        rot.rotary(_meta(2, 5, 4, 16), _meta(5, 4), _meta(5, 4))
    with pytest.raises(ValueError, match="positions must be int32"):
        rot.rotary_tables(_meta(5), 16)


@pytest.mark.parametrize("dims,more,match", [
    ((3, 5), {}, "even"), ((), {}, "1 to 4 axes"), ((2, 2, 2, 2, 2), {}, "1 to 4 axes"), ((0, 0), {}, "2 to 512"),
    ((512, 2), {}, "2 to 512"), ((8, 8), {"scale": 0.5}, "at least 1"), ((8, 8), {"scale": math.nan}, "at least 1"),
    ((8, 8), {"theta": 0.0}, "theta positive"), ((8, 8), {"scale": [1.0]}, "one value each"),
    ((8, 8), {"scaling": "yarn"}, "trained length"), ((8, 8), {"scaling": "cubic"}, "scaling must be one of"),
])
def test_refused_tables(rot, dims, more, match):
    with pytest.raises(ValueError, match=match):
        rot.rotary_tables(_meta(4, len(dims), dtype=torch.int64), dims, **more)
    with pytest.raises(ValueError, match="\\[..., axes\\]"):
        rot.rotary_tables(_meta(4, 3, dtype=torch.int64), (8, 8))


def test_library_refusals(pkg, lib):
    """Nothing is launched: every pointer below is never read."""
    L, fake = pkg._lib, 1 << 20
    assert lib.aa_rotary(None, None) == lib.aa_rotary_tables(None, None) == L.AA_EINVAL

    def turn(**change):
        a = L.RotaryArgs(q=fake, k=fake, q_out=fake, k_out=fake, cos=fake, sin=fake, B=1, S=4, H=2, Hk=2, hd=64, part=64)
        for name in ("q_stride", "k_stride", "q_out_stride", "k_out_stride"):
            setattr(a, name, L.c_strides((512, 128, 64)))
        for name, value in change.items():
            setattr(a, name, value)
        return lib.aa_rotary(ctypes.byref(a), None)

    assert turn(B=0) == turn(S=0) == turn(H=0, Hk=0) == L.AA_OK
    assert turn(hd=60) == turn(hd=520) == turn(part=0) == turn(part=66) == turn(part=31) == turn(dtype=3) == L.AA_EUNSUPPORTED
    assert turn(q=None) == turn(k_out=None) == turn(cos=None) == turn(q=fake + 8) == turn(sin=fake + 4) == L.AA_EINVAL
    assert turn(q_stride=L.c_strides((512, 128, 60))) == turn(table_stride=-1) == turn(table_stride=130) == L.AA_EINVAL
    assert turn(S=1 << 31) == turn(B=1 << 31) == turn(H=1 << 20) == L.AA_EUNSUPPORTED

    def tables(**change):
        a = L.RotaryTablesArgs(positions=fake, cos=fake, sin=fake, rows=4, axes=2)
        for i in range(2):
            a.dims[i], a.theta[i], a.scale[i] = 16, 1e4, 1.0
        for name, value in change.items():
            if isinstance(value, list):
                for i, v in enumerate(value):
                    getattr(a, name)[i] = v
            else:
                setattr(a, name, value)
        return lib.aa_rotary_tables(ctypes.byref(a), None)

    assert tables(rows=0) == L.AA_OK
    assert tables(axes=0) == tables(axes=5) == tables(dims=[3]) == tables(dims=[0, 0]) == tables(dims=[-2]) == L.AA_EUNSUPPORTED
    assert tables(dims=[1 << 40]) == tables(rows=1 << 40) == tables(position_type=4) == L.AA_EUNSUPPORTED
    assert tables(scale=[0.5]) == tables(theta=[-1.0]) == tables(scaling=2) == tables(scaling=3) == tables(cos=None) == L.AA_EINVAL
    assert tables(rows=-1) == tables(sin=fake + 4) == tables(positions=fake + 2) == L.AA_EINVAL


def test_structs_match_header(pkg):
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "anima_attn.h").read_text()
    for struct, cls in (("aa_rotary_args", pkg._lib.RotaryArgs), ("aa_rotary_tables_args", pkg._lib.RotaryTablesArgs)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S)[1], flags=re.S)
        names = re.findall(r"([A-Za-z_0-9]+)(?:\[\d+\])?\s*[,;]", body)
        assert [f[0] for f in cls._fields_] == names
