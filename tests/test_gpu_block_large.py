"""The block's operators where element offsets pass 2^31: the last rows of a large call have the
bits of a call with them alone."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import BF

pytestmark = pytest.mark.gpu

TAIL = 48


@pytest.fixture(scope="module")
def mods(pkg):
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip("needs 100 GB of GPU memory")
    yield [importlib.import_module("anima_flat_amd.kernels." + n) for n in ("adaln", "int8", "ckpt8")]
    torch.cuda.empty_cache()


def _x(rows, K, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(1, rows, K, generator=g, device="cuda", dtype=BF)


def _same(large, small):
    for a, b in zip(large, small):
        assert torch.equal(a[:, -TAIL:], b)


def test_adaln(mods):
    adaln = mods[0]
    rows, D = 270_000, 8192  # 2.2e9 values
    x, y = _x(rows, D, 1), _x(rows, D, 2)
    m = torch.randn(3, D, device="cuda")
    tail = [v[:, -TAIL:].clone() for v in (x, y)]
    _same(adaln.residual_adaln(x, y, *m), adaln.residual_adaln(*tail, *m))
    r, q, s = adaln.residual_adaln_int8(x, y, *m)
    r0, q0, s0 = adaln.residual_adaln_int8(*tail, *m)
    _same((r, q, s[None]), (r0, q0, s0[None]))
    del r, q, s

    def grads(x, y):
        x, y = x.requires_grad_(True), y.requires_grad_(True)
        out = adaln.residual_adaln(x, y, *m)
        return torch.autograd.grad(out, [x, y], [x.detach(), y.detach()])

    _same(grads(x, y), grads(*tail))


def test_int8(mods):
    int8 = mods[1]
    x = _x(270_000, 8192)
    tail = x[:, -TAIL:].clone()
    q, s = int8.rowquant_int8(x, gelu=True)
    q0, s0 = int8.rowquant_int8(tail, gelu=True)
    _same((q, s[None]), (q0, s0[None]))
    del x
    w = torch.randint(-127, 128, (8200, 32), device="cuda", dtype=torch.int8)
    ws = torch.rand(8200, device="cuda")
    _same([int8.int8_linear(q[:, :, :32].contiguous(), s, w, ws)], [int8.int8_linear(q0[:, :, :32].contiguous(), s0, w, ws)])
    w = torch.randint(-127, 128, (64, 8192), device="cuda", dtype=torch.int8)
    _same([int8.int8_linear(q, s, w, ws[:64])], [int8.int8_linear(q0, s0, w, ws[:64])])


def test_gelu8(mods):
    ckpt8 = mods[2]
    x = _x(34_000, 65536)
    tail = x[:, -TAIL:].clone()

    def both(x):
        x = x.requires_grad_(True)
        y = ckpt8.gelu8(x)
        return y.detach(), *torch.autograd.grad(y, [x], x.detach())

    _same(both(x), both(tail))


def test_lora_down8(mods):
    ckpt8 = mods[2]
    rows = 34_000
    x, a, dt = _x(rows, 65536), _x(16, 65536, 1)[0], _x(rows, 16, 2)
    dt[:, :-TAIL] = 0  # da is that of the last rows, in the same 256 of a range
    tail = x[:, -TAIL:].clone()

    def both(x, dt):
        x, w = x.requires_grad_(True), a.clone().requires_grad_(True)
        t = ckpt8.lora_down8(x, w)
        return t.detach(), *torch.autograd.grad(t, [x, w], dt)

    t, dx, da = both(x, dt)
    t0, dx0, da0 = both(tail, dt[:, -TAIL:].clone())
    _same((t, dx), (t0, dx0))
    torch.testing.assert_close(da.float(), da0.float(), rtol=2.0**-7, atol=1e-6)  # other orders of one sum each
