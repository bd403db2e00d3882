"""CPU tests of the block's operators (kernels.adaln, kernels.int8, kernels.ckpt8): refusals of
the C ABI and of the Python layer, fake implementations, the oracle itself. No kernel runs."""

from __future__ import annotations

import ctypes
import importlib
import math
import re
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import block_oracle as ref

HEADER = Path(__file__).resolve().parents[1] / "include" / "anima_attn.h"
BF = torch.bfloat16
FAKE = 1 << 20  # a 16-byte aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib(pkg):
    if not pkg._lib.LIB_PATH.exists():
        pytest.skip("libanima_attn.so not built (run __graft_entry__.build())")
    return pkg._lib.lib()


@pytest.fixture(scope="module")
def mods(pkg):
    return [importlib.import_module("anima_flat_amd.kernels." + n) for n in ("adaln", "int8", "ckpt8")]


def test_structs_match_header_field_order(pkg):
    text = HEADER.read_text()
    for struct, cls in (("aa_adaln_args", pkg._lib.AdalnArgs), ("aa_adaln_bwd_args", pkg._lib.AdalnBwdArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        types = {"const", "void", "float", "int", "int64_t"}
        fields = [t for t in re.findall(r"[A-Za-z_][A-Za-z0-9_]*", body) if t not in types]
        assert [f[0] for f in cls._fields_] == fields


# -------------------------------------------------------------- C ABI refusals --


def _adaln_args(L, **over):
    a = L.AdalnArgs(x=FAKE, y=FAKE, gate=FAKE, scale=FAKE, shift=FAKE, gate_stride=256, scale_stride=256,
                    shift_stride=0, r=FAKE, h=FAKE, B=2, S=3, D=256, eps=1e-6, branch_scale=1.0)
    for k, v in over.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("over,code,says", [
    ({"dtype": 1}, -2, "only bf16"),
    ({"mod_dtype": 1}, -2, "modulation must be"),
    ({"D": 0}, -1, "bad B/S/D"),
    ({"B": -1}, -1, "bad B/S/D"),
    ({"D": 260}, -2, "multiple of 8"),
    ({"D": 8200}, -2, "at most 8192"),
    ({"B": 1 << 20, "S": 1 << 20}, -2, "too many tokens"),
    ({"x": None}, -1, "null pointer"),
    ({"h": None}, -1, "null pointer"),
    ({"q": FAKE, "h": None}, -1, "null pointer"),
    ({"q": FAKE, "q_scale": FAKE}, -1, "exclude"),
    ({"r": None}, -1, "null pointer"),
    ({"y": None, "weight": FAKE}, -1, "weight without y"),
    ({"gate": None}, -1, "null pointer"),
    ({"scale": None}, -1, "null pointer"),
    ({"shift": None}, -1, "null pointer"),
    ({"gate": FAKE + 2}, -1, "16-byte aligned"),
    ({"gate_stride": 260}, -1, "16-byte aligned"),
    ({"scale_stride": -256}, -1, "stride"),
    ({"shift_stride": 128}, -1, "stride"),
    ({"x": FAKE + 8}, -1, "16-byte aligned"),
    ({"h": None, "q": FAKE + 4, "q_scale": FAKE}, -1, "8-byte aligned"),
])
def test_adaln_refusals(pkg, lib, over, code, says):
    assert lib.aa_adaln_fwd(_adaln_args(pkg._lib, **over), None) == code
    assert says in lib.aa_last_error().decode()


def _adaln_bwd_args(L, **over):
    a = L.AdalnBwdArgs(dr=FAKE, dh=FAKE, x=FAKE, y=FAKE, gate=FAKE, scale=FAKE, gate_stride=256, scale_stride=256,
                       stats=FAKE, dx=FAKE, dy=FAKE, gate_rows=2, scale_rows=1, shift_rows=2, B=2, S=3, D=256,
                       branch_scale=1.0)
    for k, v in over.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("over,code,says", [
    ({"dtype": 1}, -2, "only bf16"),
    ({"D": 12}, -2, "multiple of 8"),
    ({"stats": None}, -1, "null pointer"),
    ({"dy": None}, -1, "null pointer"),
    ({"y": None, "weight": FAKE}, -1, "weight without y"),
    ({"y": None, "dgate": FAKE}, -1, "not there"),
    ({"dweight": FAKE}, -1, "not there"),
    ({"dr": FAKE + 4}, -1, "16-byte aligned"),
    ({"dgate": FAKE, "gate_rows": 3}, -1, "rows must be 1 or B"),
    ({"dgate": FAKE}, -1, "workspace too small"),
    ({"dscale": FAKE, "S": 0}, -1, "no tokens"),
    ({"dscale": FAKE, "B": 70000, "gate_rows": 1, "shift_rows": 1}, -2, "too many batch items"),
])
def test_adaln_bwd_refusals(pkg, lib, over, code, says):
    assert lib.aa_adaln_bwd(_adaln_bwd_args(pkg._lib, **over), None, 0, None) == code
    assert says in lib.aa_last_error().decode()


def test_other_refusals(lib):
    bad, no = -1, -2
    assert lib.aa_adaln_fwd(None, None) == bad and lib.aa_adaln_bwd(None, None, 0, None) == bad

    def rowquant(rows=4, K=64, x=FAKE, q=FAKE, s=FAKE, dtype=0):
        return lib.aa_rowquant_int8(x, rows, K, 0, q, s, dtype, None)

    assert rowquant(dtype=1) == no and rowquant(K=60) == no and rowquant(K=8200) == no
    assert rowquant(rows=-1) == bad and rowquant(s=None) == bad and rowquant(x=FAKE + 8) == bad
    assert rowquant(rows=1 << 31) == no and rowquant(rows=0, x=None) == 0

    def linear(q=FAKE, s=FAKE, w=FAKE, ws=FAKE, y=FAKE, M=4, N=64, K=64, dtype=0):
        return lib.aa_int8_linear(q, s, w, ws, y, M, N, K, dtype, None)

    assert linear(dtype=2) == no and linear(K=40) == no and linear(K=65552) == no and linear(N=60) == no
    assert linear(M=-1) == bad and linear(N=0) == bad and linear(ws=None) == bad and linear(w=FAKE + 8) == bad
    assert linear(M=0, q=None) == 0

    def gelu(x=FAKE, y=FAKE, c=FAKE, e=FAKE, rows=4, K=64, dtype=0):
        return lib.aa_gelu8_fwd(x, y, c, e, rows, K, dtype, None)

    assert gelu(dtype=1) == no and gelu(K=20) == no and gelu(K=65544) == no and gelu(rows=-1) == bad
    assert gelu(e=None) == bad and gelu(c=FAKE + 8) == bad and gelu(rows=0, x=None) == 0
    assert lib.aa_gelu8_bwd(FAKE, None, FAKE, FAKE, 4, 64, 0, None) == bad
    assert lib.aa_gelu8_bwd(FAKE + 2, FAKE, FAKE, FAKE, 4, 64, 0, None) == bad

    def lora(x=FAKE, a=FAKE, t=FAKE, c=FAKE, e=FAKE, ws=None, n=0, M=4, K=64, R=16, dtype=0):
        return lib.aa_lora8_fwd(x, a, t, c, e, ws, n, M, K, R, dtype, None)

    assert lora(dtype=1) == no and lora(R=12) == no and lora(R=72) == no and lora(R=0) == no and lora(K=4) == no
    assert lora(e=None) == bad and lora(a=FAKE + 2) == bad and lora(M=0, x=None) == 0
    big = lib.aa_lora8_bwd_workspace(1 << 20, 64, 16)
    assert big > 0

    def lora_bwd(dt=FAKE, a=FAKE, c=FAKE, e=FAKE, dx=FAKE, da=FAKE, ws=FAKE, n=big, M=1 << 20, K=64, R=16):
        return lib.aa_lora8_bwd(dt, a, c, e, dx, da, ws, n, M, K, R, 0, None)

    assert lora_bwd(n=big - 4) == bad and "workspace" in lib.aa_last_error().decode()
    assert lora_bwd(ws=None) == bad and lora_bwd(c=None) == bad and lora_bwd(a=None) == bad
    assert lora_bwd(R=4) == no and lora_bwd(M=0) == bad and lora_bwd(M=0, da=None) == 0
    assert lora_bwd(dt=FAKE + 4) == bad


# ------------------------------------------------------------- Python refusals --


def test_cpu_tensors_are_rejected(mods):
    adaln, int8, ckpt8 = mods
    x, m = torch.zeros(1, 4, 64, dtype=BF), torch.zeros(1, 64)
    i = torch.zeros(1, 4, 64, dtype=torch.int8)
    for call in (
        lambda: adaln.residual_adaln(x, x, m, m, m), lambda: adaln.adaln(x, m, m),
        lambda: adaln.residual_adaln_int8(x, x, m, m, m), lambda: int8.rowquant_int8(x),
        lambda: int8.quantize_weight(x[0]), lambda: int8.int8_linear(i, torch.ones(4), i[0], torch.ones(4)),
        lambda: ckpt8.gelu8(x), lambda: ckpt8.lora_down8(x, x[0]),
    ):
        with pytest.raises(ValueError, match="CUDA tensors required"):
            call()


def test_shapes_and_types_are_checked(mods):
    adaln, int8, ckpt8 = mods
    with FakeTensorMode():
        def t(*shape, dtype=BF, **kw):
            return torch.empty(*shape, dtype=dtype, device="cuda", **kw)

        x, m = t(2, 5, 64), t(2, 64)
        for args, says in (
            ((x.half(), x.half(), m, m, m), "only bfloat16"),
            ((x, t(2, 5, 72), m, m, m), "x's shape"),
            ((x[0], x[0], m, m, m), "must be .B, S, D"),
            ((t(2, 5, 60), t(2, 5, 60), m, m, m), "multiple of 8"),
            ((t(1, 2, 8200), t(1, 2, 8200), m, m, m), "at most 8192"),
            ((x, x, t(3, 64), m, m), "gate must be"),
            ((x, x, m, t(2, 5, 64), m), "scale must be"),
            ((x, x, m, m, t(2, 32)), "shift must be"),
            ((x, x, m, m, m.half()), "shift must be bfloat16 or float32"),
            ((x, x, m, m, m, t(32)), "weight must be"),
            ((x, x, m, m, m.to("cuda:1")), "one device"),
        ):
            for call in (adaln.residual_adaln, adaln.residual_adaln_int8):
                with pytest.raises(ValueError, match=says):
                    call(*args)
        with pytest.raises(RuntimeError, match="no backward"):
            adaln.residual_adaln_int8(x, x, m, m, t(2, 64, requires_grad=True))
        with pytest.raises(RuntimeError, match="no backward"):
            int8.rowquant_int8(t(2, 5, 64, requires_grad=True))
        with pytest.raises(ValueError, match="B, S, K"):
            int8.rowquant_int8(m)
        with pytest.raises(ValueError, match="N, K"):
            int8.quantize_weight(x)
        q, s, w, ws = t(2, 5, 64, dtype=torch.int8), t(10, 1, dtype=torch.float32), t(8, 64, dtype=torch.int8), t(8, dtype=torch.float32)
        for args in ((x, s, w, ws), (q[0], s, w, ws), (q, s[:9], w, ws), (q, s.half(), w, ws), (q, s, w[:, :48], ws),
                     (q, s, w.float(), ws), (q, s, w, ws[:4]), (q, s, w, ws.double()), (q, s, w, ws.to("cuda:1"))):
            with pytest.raises(ValueError):
                int8.int8_linear(*args)
        for call in (lambda: ckpt8.gelu8(x.float()), lambda: ckpt8.gelu8(x[0]), lambda: ckpt8.gelu8(t(1, 1, 12)),
                     lambda: ckpt8.gelu8(t(1, 1, 65544)), lambda: ckpt8.lora_down8(x, t(12, 64)),
                     lambda: ckpt8.lora_down8(x, t(72, 64)), lambda: ckpt8.lora_down8(x, t(0, 64)),
                     lambda: ckpt8.lora_down8(x, t(8, 72)), lambda: ckpt8.lora_down8(x, t(8, 64).float()),
                     lambda: ckpt8.lora_down8(x, t(8, 64).to("cuda:1"))):
            with pytest.raises(ValueError):
                call()


def test_fakes(mods):
    """Shapes and types without a GPU, forward (fake tensors) and the raw ops (meta)."""
    adaln, int8, ckpt8 = mods
    with FakeTensorMode():
        def t(*shape, dtype=BF):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        x, m = t(2, 5, 64), t(2, 64, dtype=torch.float32)
        r, h = adaln.residual_adaln(x, x, m, m, m, t(64))
        assert r.shape == h.shape == x.shape and h.dtype == BF
        assert adaln.adaln(x, m, m).shape == x.shape
        r, q, s = adaln.residual_adaln_int8(x, x, m, m, m)
        assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == (10, 1)
        q, s = int8.rowquant_int8(x, gelu=True)
        y = int8.int8_linear(q, s, *int8.quantize_weight(t(24, 64)))
        assert y.shape == (2, 5, 24) and y.dtype == BF
        assert ckpt8.gelu8(x).shape == x.shape and ckpt8.lora_down8(x, t(16, 64)).shape == (2, 5, 16)
    ops = torch.ops.anima_flat_amd
    x, m = torch.empty(2, 5, 72, dtype=BF, device="meta"), torch.empty(2, 72, device="meta")
    *_, stats = ops.residual_adaln(x, x, m, m, m, None, 1e-6, 1.0, True)
    assert stats.shape == (10, 4)
    one = torch.empty(1, 72, device="meta")
    out = ops.adaln_bwd(x, None, x, x, one, m, one[0], stats, 1, 1.0, True)
    assert [tuple(o.shape) for o in out] == [(2, 5, 72), (2, 5, 72), (1, 72), (2, 72), (1, 72), (72,)]
    out = ops.adaln_bwd(None, x, x, None, None, m, None, stats, 2, 1.0, False)
    assert [o.numel() for o in out] == [720, 0, 0, 0, 0, 0]
    _, codes, exps = ops.gelu8(x, True)
    assert codes.shape == (10, 96) and exps.shape == (10, 3)
    assert ops.gelu8_bwd(x, codes, exps).shape == x.shape
    a = torch.empty(16, 72, dtype=BF, device="meta")
    low, codes, exps = ops.lora_down8(x, a, True)
    assert low.shape == (2, 5, 16) and codes.shape == (10, 96) and exps.shape == (3, 16)
    dx, da = ops.lora_down8_bwd(low, a, codes, exps, True, False)
    assert dx.shape == x.shape and da.numel() == 0


def test_names_stay_out_of_the_references_namespace(mods):
    for name in ("residual_adaln", "adaln", "rowquant_int8", "int8_linear", "gelu8", "lora_down8"):
        assert hasattr(torch.ops.anima_flat_amd, name) and not hasattr(torch.ops.anima_flat, name)


# ------------------------------------------------------------------ the oracle --


def test_oracle_gradients():
    """The oracle's forward is differentiable and agrees with differences."""
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randn(2, 3, 8, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    m = [torch.randn(n, 8, generator=g, dtype=torch.float64, requires_grad=True) for n in (2, 1, 2)]
    w = torch.randn(8, generator=g, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda *a: ref.residual_adaln(*a, eps=1e-3, branch_scale=0.7), (x, y, *m, w))


def test_oracle_gelu():
    x = torch.linspace(-9, 9, 2001, dtype=torch.float64)
    torch.testing.assert_close(ref.gelu(x), torch.nn.functional.gelu(x), rtol=1e-9, atol=1e-15)
    torch.testing.assert_close(ref.gelu_slope(x), (ref.gelu(x + 1e-6) - ref.gelu(x - 1e-6)) / 2e-6, rtol=1e-6, atol=1e-8)


def test_oracle_checkpoint():
    """Within half a step, at most 2^-7 of the group's largest, exact in bf16, marks non-finite."""
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(50, 72, generator=g) * torch.exp2(torch.randint(-60, 60, (50, 1), generator=g).float())).to(BF)
    x[3, 40] = math.inf
    codes, exps, kept = ref.checkpoint(x)
    assert codes.shape == (50, 96) and exps.shape == (50, 3) and exps[3].tolist().count(255) == 1
    assert torch.isnan(kept[3, 32:64]).all() and torch.isfinite(kept[3, :32]).all()
    fine = torch.isfinite(kept)
    assert torch.equal(kept.to(BF).double()[fine], kept[fine])
    top = torch.nn.functional.pad(x.double().abs(), (0, 24)).unflatten(1, (3, 32)).amax(-1).repeat_interleave(32, 1)[:, :72]
    assert ((kept - x.double()).abs() <= top * 2.0**-7)[fine].all()
    # A tie and the clamp at the largest magnitude: 1.9921875 / 2^-6 = 127.5.
    v = torch.tensor([[1.9921875, -1.9921875, 0.5 / 64, 1.5 / 64]]).to(BF)
    assert ref.checkpoint(v)[0][0, :4].tolist() == [127, -127, 0, 2]


def test_int8_rule_for_every_bf16_value():
    """The quantiser's arithmetic (an exact product with 127 / max rounded up to float32, then to
    an integer) gives the oracle's codes for each bf16 mantissa of the largest value and every
    smaller value, ties included."""
    bits = torch.arange(0x7F80, dtype=torch.int32)
    values = (bits << 16).view(torch.float32)  # finite and not negative
    for e in (-39, -30, 0, 40, 110):
        for m in (128 + torch.arange(128.0)) * 2.0 ** (e - 7):
            y = values[(values <= m) & (values >= m * 2.0**-11)]
            rcp = 127 / m
            if rcp.double() * m.double() < 127:
                rcp = torch.nextafter(rcp, torch.tensor(math.inf))
            q, s = ref.int8_rows(y[None])
            assert torch.equal(torch.round(y.double() * rcp.double()).to(torch.int8), q[0]) and s == m / 127
    y = values[values <= 1e-12]
    m = torch.tensor(1e-12)
    rcp = 127 / m
    rcp = rcp if rcp.double() * m.double() >= 127 else torch.nextafter(rcp, torch.tensor(math.inf))
    assert torch.equal(torch.round(y.double() * rcp.double()).to(torch.int8), ref.int8_rows(y[None])[0][0])
    half = torch.tensor([[255.0, 127.5, -127.5, 1.0]])
    assert ref.int8_rows(half)[0].tolist() == [[127, 64, -64, 0]]
