"""kernels.ckpt8 against its oracle: the 8-bit copies bit for bit, results and gradients."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import BF, U16, U32, bf, gen, within
from oracle import block_oracle as ref

pytestmark = pytest.mark.gpu

# The fit of GELU's tail is off by 3.1e-5, relative; the exponential's argument x^2 / 2 (at most
# 100 where anything is left) by 2^-23 of itself, and a handful of float32 roundings.
GELU_REL = 3.1e-5 + 100 * 2.0**-23 + 16 * U32


@pytest.fixture(scope="session")
def ckpt8(pkg):
    return importlib.import_module("anima_flat_amd.kernels.ckpt8")


def _values(shape, seed, spread=False):
    g = gen(seed)
    x = torch.randn(*shape, generator=g) * 1.5
    if spread:
        x = x * torch.exp2(torch.randint(-100, 101, (*shape[:-1], 1), generator=g).float())
        x = x * torch.exp2(torch.randint(-12, 1, shape, generator=g).float())
    return x.to("cuda", BF)


KS = [8, 24, 32, 40, 56, 64, 248, 256, 264, 1000, 2048, 8192]


@pytest.mark.parametrize("K", KS)
@pytest.mark.parametrize("spread", [False, True])
@pytest.mark.parametrize("op", ["gelu8", "lora_down8"])
def test_copies_bit_exact(ckpt8, K, spread, op):
    rows = 37
    x = _values((1, rows, K), K + spread, spread)
    x[0, 3] = 0
    x[0, 5, K // 2] = float("inf")
    x[0, 7, 0] = float("nan")
    x[0, 9] = 1e-40  # below bf16's normal range
    codes, exps, _ = ref.checkpoint(x[0].cpu())
    if op == "gelu8":
        _, c, e = ckpt8._gelu8(x, True)
    else:
        _, c, e = ckpt8._lora_down8(x, torch.zeros(8, K, dtype=BF, device="cuda"), True)
        assert e.shape == (codes.shape[1] // 32, 48)
        e = e[:, :rows].t()
    assert torch.equal(e.cpu(), exps)
    fine = (exps != 255).repeat_interleave(32, 1)  # a marked group's codes are not read
    assert torch.equal(c.cpu()[fine], codes[fine])
    assert (c.cpu()[:, K:] == 0)[fine[:, K:]].all()


@pytest.mark.parametrize("B,S,K", [(1, 1, 8), (2, 3, 40), (1, 33, 256), (2, 17, 1000), (1, 9, 8192), (3, 301, 264)])
def test_gelu(ckpt8, B, S, K):
    x = _values((B, S, K), B + S + K).requires_grad_(True)
    y = ckpt8.gelu8(x)
    want = ref.gelu(x.detach().double())
    within(y, want, (U16 + GELU_REL) * want.abs(), "y")
    dy = bf(gen(K), B, S, K)
    (dx,) = torch.autograd.grad(y, [x], dy)
    kept = ref.checkpoint(x.detach().flatten(0, 1))[2].view(B, S, K)
    slope = ref.gelu_slope(kept)
    part = ref.normal_cdf(kept) + (slope - ref.normal_cdf(kept)).abs()
    want = dy.double() * slope
    within(dx, want, U16 * want.abs() + GELU_REL * dy.double().abs() * part, "dx")
    with torch.no_grad():
        assert torch.equal(ckpt8.gelu8(x), y)


def test_gelu_whole_range(ckpt8):
    """Every finite bf16 value: the lower tail keeps its digits until it leaves the normal range."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    x = x[torch.isfinite(x)].view(1, 1, -1).cuda()
    y = ckpt8.gelu8(x).double()
    want = ref.gelu(x.double())
    bound = (U16 + GELU_REL) * want.abs() + 2.0**-126 * x.double().abs().clamp(1, 16)
    within(y, want, bound, "y")
    inf = torch.tensor([float("inf"), float("-inf")] * 4, dtype=BF, device="cuda").view(1, 1, 8)
    assert ckpt8.gelu8(inf).flatten()[:2].tolist() == [float("inf"), 0.0]
    assert torch.isnan(ckpt8.gelu8(torch.full_like(inf, float("nan")))).all()


def test_gelu_slope_against_differences(ckpt8):
    """dx of a copied value against a central difference of GELU there."""
    x = torch.linspace(-6, 6, 4096).to("cuda", BF).view(1, 64, 64).requires_grad_(True)
    (dx,) = torch.autograd.grad(ckpt8.gelu8(x), [x], torch.ones_like(x))
    kept = ref.checkpoint(x.detach()[0])[2]
    slope = (ref.gelu(kept + 1e-5) - ref.gelu(kept - 1e-5)) / 2e-5
    within(dx[0], slope, U16 * slope.abs() + 1.2 * GELU_REL * 1.2 + 1e-9, "dx")


def _lora_bounds(x, a):
    return (x.abs() @ a.abs().t())


@pytest.mark.parametrize("R", [8, 16, 24, 40, 64])
@pytest.mark.parametrize("B,S,K", [(1, 1, 8), (2, 7, 264), (1, 130, 2048), (1, 17, 8192), (1, 300, 40)])
def test_lora(ckpt8, B, S, K, R):
    """t: fp32 over chains of at most K / 8 + 16 additions in a wave and across them. dx: R.
    da: one per token. All of exact bf16 products."""
    g = gen(B + S + K + R)
    x = _values((B, S, K), K + R).requires_grad_(True)
    a = bf(g, R, K, scale=K**-0.5).requires_grad_(True)
    t = ckpt8.lora_down8(x, a)
    xd, ad = x.detach().double().flatten(0, 1), a.detach().double()
    want = xd @ ad.t()
    within(t.flatten(0, 1), want, U16 * want.abs() + (K / 8 + 32) * U32 * (xd.abs() @ ad.abs().t()), "t")
    dt = bf(g, B, S, R)
    dx, da = torch.autograd.grad(t, [x, a], dt)
    dtd = dt.double().flatten(0, 1)
    want = dtd @ ad
    within(dx.flatten(0, 1), want, U16 * want.abs() + (R + 2) * U32 * (dtd.abs() @ ad.abs()), "dx")
    kept = ref.checkpoint(x.detach().flatten(0, 1))[2]
    want = dtd.t() @ kept
    within(da, want, U16 * want.abs() + (B * S + 8) * U32 * (dtd.abs().t() @ kept.abs()), "da")
    with torch.no_grad():
        assert torch.equal(ckpt8.lora_down8(x, a), t)


@pytest.mark.parametrize("M,K,R", [(8200, 520, 16), (9000, 256, 48), (2050, 8192, 32), (8250, 264, 64)])
def test_lora_many_rows(ckpt8, M, K, R):
    """Row tiles of 32, several ranges of rows in da."""
    test_lora(ckpt8, 1, M, K, R)


def test_lora_one_gradient(ckpt8):
    """Only what requires grad is computed; nothing of x is kept where a is frozen."""
    x, a = _values((1, 50, 264), 3), bf(gen(4), 16, 264)
    dt = bf(gen(5), 1, 50, 16)
    both = [v.clone().requires_grad_(True) for v in (x, a)]
    want = torch.autograd.grad(ckpt8.lora_down8(*both), both, dt)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(t.numel()), t)[1], lambda t: t):
        t = ckpt8.lora_down8(both[0], a)
    assert sum(seen) == a.numel()
    assert torch.equal(torch.autograd.grad(t, [both[0]], dt)[0], want[0])
    assert torch.equal(torch.autograd.grad(ckpt8.lora_down8(x, both[1]), [both[1]], dt)[0], want[1])


def test_saved_bytes(ckpt8):
    """The graph keeps 33/32 bytes a value and no bf16 copy."""
    x = _values((1, 64, 2048), 6).requires_grad_(True)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(t.numel() * t.element_size()), t)[1], lambda t: t):
        ckpt8.gelu8(x)
    assert sum(seen) == x.numel() * 33 // 32


def test_not_finite(ckpt8):
    """A value that is not finite marks its group of 32: the gradients that read it are NaN, all
    others are untouched."""
    x = _values((1, 40, 96), 7)
    dt, dy = bf(gen(8), 1, 40, 8), bf(gen(9), 1, 40, 96)
    a = bf(gen(10), 8, 96).requires_grad_(True)

    def grads(x):
        x = x.clone().requires_grad_(True)
        t = ckpt8.lora_down8(x, a)
        return t, *torch.autograd.grad(t, [x, a], dt), *torch.autograd.grad(ckpt8.gelu8(x), [x], dy)

    clean = grads(x)
    x = x.clone()
    x[0, 33, 40] = float("inf")
    t, dx, da, dg = grads(x)
    rows = torch.arange(40) != 33
    assert torch.equal(t[0, rows], clean[0][0, rows]) and torch.equal(dx, clean[1])
    cols = torch.ones(96, dtype=torch.bool)
    cols[32:64] = False
    assert torch.equal(da[:, cols], clean[2][:, cols]) and torch.isnan(da[:, ~cols]).all()
    assert torch.equal(dg[0, rows], clean[3][0, rows]) and torch.equal(dg[0, 33, cols], clean[3][0, 33, cols])
    assert torch.isnan(dg[0, 33, ~cols]).all()


def test_layouts(ckpt8):
    x, a, dt = _values((2, 19, 264), 11), bf(gen(12), 24, 264), bf(gen(13), 2, 19, 24)
    dy = bf(gen(14), 2, 19, 264)

    def off(v):
        return torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v)

    def strided(v):
        return torch.stack((v, v), -1)[..., 0]

    def turned(v):
        return v.transpose(0, -1).contiguous().transpose(0, -1)

    def step(form):
        xs, as_ = (form(v).detach().requires_grad_(True) for v in (x, a))
        t, y = ckpt8.lora_down8(xs, as_), ckpt8.gelu8(xs)
        return [t, y, *torch.autograd.grad([t, y], [xs, as_], [form(dt), form(dy)])]

    want = step(lambda v: v)
    for form in (off, strided, turned):
        assert all(torch.equal(p, q) for p, q in zip(want, step(form))), form.__name__


def test_no_tokens(ckpt8):
    x = torch.empty(2, 0, 64, dtype=BF, device="cuda", requires_grad=True)
    a = torch.ones(8, 64, dtype=BF, device="cuda", requires_grad=True)
    t = ckpt8.lora_down8(x, a)
    y = ckpt8.gelu8(x)
    dx, da = torch.autograd.grad([t, y], [x, a], [torch.empty_like(t), torch.empty_like(y)])
    assert t.shape == (2, 0, 8) and dx.shape == x.shape and not da.any()


def test_repeatable(ckpt8):
    x, a = _values((1, 3000, 520), 15).requires_grad_(True), bf(gen(16), 16, 520).requires_grad_(True)
    dt = bf(gen(17), 1, 3000, 16)
    first = torch.autograd.grad(ckpt8.lora_down8(x, a), [x, a], dt)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(ckpt8.lora_down8(x, a), [x, a], dt)))
