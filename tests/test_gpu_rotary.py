"""Rotary tables and turns against their 64-bit formulas."""

from __future__ import annotations

import importlib
import math

import pytest
import torch

from block_cases import gen, within
from rotary_cases import U32, tables, turn, turn_bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rot(pkg):
    return importlib.import_module("anima_flat_amd.kernels.rotary")


def _heads(g, B, S, H, hd, dtype):
    return (torch.randn(B, S, H, hd, generator=g) * 1.5).to("cuda", dtype)


def _angles(g, *shape):
    a = 6.3 * torch.rand(*shape, generator=g).cuda()
    return a.cos(), a.sin()


# ------------------------------------------------------------------ tables --

# An angle's fraction of a turn is rounded to fp32 once (relative 2^-24 of at most pi
# radians); sincospif is good to 4 ulp (2^-24 below 1), the factor is one more rounding. The
# product in 64 bits is off by 4 2^-53 of itself (frequency, its turns, product, reference):
# 2^-51 2 10^5 turns at most here, under 10^-9.
TABLE_BOUND = (math.pi + 4 + 1) * U32 + 2e-9


@pytest.mark.parametrize("scaling", ["ntk", "linear", "yarn"])
@pytest.mark.parametrize("dims,shape", [((128,), (37,)), ((44, 42, 42), (2, 9)), ((6, 0, 2), (5,)), ((10,), (1,)), ((2,), (3, 3)), ((512,), (4,))])
def test_tables(rot, scaling, dims, shape):
    positions = torch.randint(-(10**6), 10**6, (*shape, len(dims)), generator=gen(3)).cuda()
    theta, scale = [10000.0, 500.0, 1e6][: len(dims)], [7.3, 1.0, 2.5][: len(dims)]
    cos, sin = rot.rotary_tables(positions, dims, theta=theta, scale=scale, scaling=scaling, original=4096)
    c, s, factor = tables(positions, dims, theta, scale, scaling, 4096)
    bound = torch.tensor(TABLE_BOUND * factor, dtype=torch.float64, device="cuda")
    for got, want in ((cos, c), (sin, s)):
        assert got.shape == (*shape, sum(dims) // 2) and got.dtype == torch.float32
        within(got, want, bound, f"{scaling} {dims}")


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_tables_of_one_axis_and_every_type(rot, dtype):
    positions = torch.tensor([[0, 1, 5, 99999], [7, -3, 2**20, 10**8]], dtype=torch.float64).cuda().to(dtype)
    if dtype.is_floating_point:
        positions += 0.25
    cos, sin = rot.rotary_tables(positions, 64)
    c, s, _ = tables(positions[..., None], [64], [10000.0], [1.0], "ntk")
    # 10^8 positions are 1.6 10^7 turns: 4 2^-53 of them are 2 pi 7 10^-9 radians.
    bound = torch.tensor(TABLE_BOUND + 5e-8, dtype=torch.float64, device="cuda")
    within(cos, c, bound, "cos")
    within(sin, s, bound, "sin")


def test_tables_are_the_models(pkg, rot):
    """rope_tables' grid, whose angles are formed in fp32: off by 4 2^-24 of up to 63 radians."""
    y, x = torch.meshgrid(torch.arange(48), torch.arange(64), indexing="ij")
    positions = torch.stack((torch.zeros_like(x), y, x), -1).reshape(-1, 3).cuda()
    cos, sin = rot.rotary_tables(positions, (44, 42, 42), scale=(1.0, 4.0, 4.0))
    c, s = pkg.rope_tables(48, 64, 128, "cuda", (4.0, 4.0))
    assert (cos - c).abs().max() < 63 * 4 * U32 + 1e-6 and (sin - s).abs().max() < 63 * 4 * U32 + 1e-6


def test_no_positions(rot):
    cos, sin = rot.rotary_tables(torch.empty(0, 2, dtype=torch.int64, device="cuda"), (8, 8))
    assert cos.shape == sin.shape == (0, 8)


# -------------------------------------------------------------------- turn --

SIZES = [  # B, S, H, Hk, hd, part
    (1, 1, 1, 1, 128, 128), (2, 37, 16, 16, 128, 128), (1, 130, 12, 4, 80, 36), (3, 5, 6, 2, 256, 64), (2, 9, 3, 1, 40, 10),
    (1, 3, 5, 5, 8, 2), (2, 3, 7, 2, 96, 94), (1, 65, 9, 0, 64, 64), (1, 2, 2, 1, 512, 512),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_turn(rot, dtype, interleaved, size):
    B, S, H, Hk, hd, part = size
    g = gen(5)
    q, k = _heads(g, B, S, H, hd, dtype), _heads(g, B, S, Hk, hd, dtype)
    cos, sin = _angles(g, B, S, part // 2) if S % 2 else _angles(g, S, part // 2)
    got = rot.rotary_qk(q, k, cos, sin, interleaved) if Hk else [rot.rotary(q, cos, sin, interleaved)]
    for x, y in zip((q, k), got):
        ref, width = turn(x, cos, sin, interleaved)
        assert y.dtype == dtype and y.is_contiguous()
        within(y, ref, turn_bound(ref, width, dtype), f"{size}")
        assert torch.equal(y[..., part:], x[..., part:])
    if Hk:
        assert torch.equal(got[0], rot.rotary(q, cos, sin, interleaved)) and torch.equal(got[1], rot.rotary(k, cos, sin, interleaved))


@pytest.mark.parametrize("form", ["fused", "head_major", "last_dim_strided", "misaligned", "expanded", "odd_stride"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_views(rot, form, interleaved):
    """Views in place or copied, the same bits; tables that are views."""
    g = gen(6)
    B, S, H, hd = 2, 33, 4, 64
    q = _heads(g, B, S, H, hd, torch.bfloat16)
    cos, sin = _angles(g, S, 16)
    if form == "fused":  # q and v side by side, as a projection gives them
        x = torch.cat((q, q.flip(1)), -1)[..., :hd]
    elif form == "head_major":
        x = q.transpose(1, 2).contiguous().transpose(1, 2)
    elif form == "last_dim_strided":
        x = torch.stack((q, q), -1)[..., 0]
    elif form == "misaligned":
        x = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    elif form == "expanded":
        q = q[:1].expand(B, S, H, hd)
        x = q
    else:
        x = torch.empty(B, S, H, hd + 3, dtype=q.dtype, device="cuda")[..., :hd].copy_(q)
    want = rot.rotary(q.contiguous(), cos, sin, interleaved)
    assert torch.equal(rot.rotary(x, cos, sin, interleaved), want)
    wide = torch.stack((cos, cos), -1)[..., 0], torch.cat((sin, sin), -1)[:, : sin.shape[1]]
    assert torch.equal(rot.rotary(x, *wide, interleaved), want)
    assert torch.equal(rot.rotary(x, cos[None], sin[None], interleaved), want)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(rot, interleaved, dtype):
    """The formula's, and differences: the turn is linear, so a step of any size gives them."""
    g = gen(7)
    B, S, H, Hk, hd, part = 2, 19, 6, 2, 48, 20
    q, k, dq, dk = (_heads(g, B, S, n, hd, dtype) for n in (H, Hk, H, Hk))
    cos, sin = _angles(g, B, S, part // 2)
    q.requires_grad_(True), k.requires_grad_(True)
    out = rot.rotary_qk(q, k, cos, sin, interleaved)
    got = torch.autograd.grad(out, [q, k], [dq, dk])
    for x, y in zip((dq, dk), got):
        ref, width = turn(x, cos, -sin, interleaved)
        within(y, ref, turn_bound(ref, width, dtype), "gradient")
    if dtype == torch.float32:
        step = _heads(g, B, S, H, hd, dtype)
        with torch.no_grad():
            change = rot.rotary(q + step, cos, sin, interleaved) - rot.rotary(q - step, cos, sin, interleaved)
        along, by = (change.double() * dq.double() / 2).sum(), (got[0].double() * step.double()).sum()
        size = (dq.double().abs().sum() * 4 * (q.abs().max() + step.abs().max()).double())
        assert (along - by).abs() < 6 * U32 * size
    # one of two outputs only; twice
    only = torch.autograd.grad(rot.rotary_qk(q, k, cos, sin, interleaved)[1], [k], dk)[0]
    assert torch.equal(only, got[1])
    none = torch.autograd.grad(rot.rotary_qk(q, k, cos, sin, interleaved)[1], [q], dk, allow_unused=True)[0]
    assert none is None or not none.any()
    first = torch.autograd.grad(rot.rotary(q, cos, sin, interleaved), [q], dq.requires_grad_(True), create_graph=True)[0]
    second = torch.autograd.grad(first, [dq], q.detach())[0]
    assert torch.equal(second, rot.rotary(q.detach(), cos, sin, interleaved))


def test_tables_need_no_gradient(rot):
    q = torch.ones(1, 2, 1, 8, device="cuda")
    cos, sin = torch.ones(2, 4, device="cuda", requires_grad=True), torch.zeros(2, 4, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        rot.rotary(q, cos, sin)
    with torch.no_grad():
        assert torch.equal(rot.rotary(q, cos, sin), q)


def test_special_values_stay_in_their_pair(rot):
    q = torch.ones(1, 2, 1, 16, device="cuda", dtype=torch.bfloat16)
    q[0, 0, 0, 3], q[0, 1, 0, 15] = math.nan, math.inf
    cos, sin = torch.full((2, 4), 0.6, device="cuda"), torch.full((2, 4), 0.8, device="cuda")
    y = rot.rotary(q, cos, sin)
    assert torch.isnan(y[0, 0, 0]).nonzero().flatten().tolist() == [3, 7]
    assert torch.isfinite(y[0, 1, 0, :15]).all() and y[0, 1, 0, 15] == math.inf


def test_strides_of_single_elements(rot):
    """Dimensions of size 1 have strides that address nothing, and that contiguous() keeps."""
    g = gen(8)
    base = torch.randn(1, 5, 3, 67, generator=g).cuda().to(torch.bfloat16)
    x = base[:, :1, :1, :64]
    x = x.as_strided(x.shape, (7, 3, 5, 1))
    cos, sin = _angles(g, 1, 32)
    assert torch.equal(rot.rotary(x, cos, sin), rot.rotary(x.clone(memory_format=torch.contiguous_format), cos, sin))


def test_empty(rot):
    cos = torch.ones(0, 4, device="cuda")
    q, k = rot.rotary_qk(torch.empty(2, 0, 3, 8, device="cuda"), torch.empty(2, 0, 1, 8, device="cuda"), cos, cos)
    assert q.shape == (2, 0, 3, 8) and k.shape == (2, 0, 1, 8)
