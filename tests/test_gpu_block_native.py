"""The block operators' native dispatcher kernels against their Python functions, and how they
behave under autograd, transforms and tracing."""

from __future__ import annotations

import importlib

import pytest
import torch
import torch._dynamo.compiled_autograd
from torch._subclasses.fake_tensor import FakeTensorMode

from block_cases import BF, bf, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="session")
def mods(pkg):
    return [importlib.import_module("anima_flat_amd.kernels." + n) for n in ("adaln", "int8", "ckpt8")]


def _cases():
    """Arguments of every op with native kernels, by name."""
    g = gen(1)
    x, y, dr, dh = (bf(g, 2, 30, 264) for _ in range(4))
    gate, scale = bf(g, 2, 528)[:, 264:], bf(g, 2, 264)
    shift, weight = bf(g, 1, 264), bf(g, 264).float()
    a, dt = bf(g, 16, 264), bf(g, 2, 30, 16)
    ops = torch.ops.anima_flat_amd
    stats = ops.residual_adaln(x, y, gate, scale, shift, weight, 1e-6, 0.5, True)[2]
    own = ops.adaln(x, scale, shift, 1e-6, True)[1]
    wide = bf(g, 2, 30, 272)
    q, s = ops.rowquant_int8(wide, True)
    w, ws = torch.randint(-127, 128, (24, 272), generator=g, dtype=torch.int8).cuda(), torch.rand(24, generator=g).cuda()
    _, codes, exps = ops.gelu8(x, True)
    _, lcodes, lexps = ops.lora_down8(x, a, True)
    return {
        "residual_adaln": [(x, y, gate, scale, shift, weight, 1e-6, 0.5, True), (x, y, gate, scale, shift, None, 1e-6, 0.5, False)],
        "adaln": [(x, scale, shift, 1e-6, True), (x, scale, shift, 1e-6, False)],
        "residual_adaln_int8": [(x, y, gate, scale, shift, weight, 1e-6, 0.5)],
        "adaln_bwd": [(dr, dh, x, y, gate, scale, weight, stats, 1, 0.5, True), (None, dh, x, y, gate, scale, None, stats, 1, 0.5, False),
                      (None, dh, x, None, None, scale, None, own, 1, 1.0, True)],
        "rowquant_int8": [(x, False), (x, True)],
        "int8_linear": [(q, s, w, ws)],
        "gelu8": [(x, True), (x, False)],
        "gelu8_bwd": [(dh, codes, exps)],
        "lora_down8": [(x, a, True), (x, a, False)],
        "lora_down8_bwd": [(dt, a, lcodes, lexps, True, True), (dt, a, lcodes, lexps, False, True), (dt, a, lcodes, lexps, True, False)],
    }


def _off(v):
    """The same values one element past a 16-byte boundary."""
    return torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v)


@pytest.mark.parametrize("form", ["plain", "misaligned"])
def test_python_functions_give_the_same_bits(mods, form):
    cases = _cases()
    native = importlib.import_module("anima_flat_amd._native")
    assert {"anima_flat_amd::" + n for n in cases} == native.NATIVE_BLOCK_OPS
    for name, calls in cases.items():
        (impl,) = [op._init_fn for m in mods for op in vars(m).values()
                   if isinstance(op, torch.library.CustomOpDef) and op._qualname == "anima_flat_amd::" + name]
        for args in calls:
            want = getattr(torch.ops.anima_flat_amd, name)(*args)
            cast = args if form == "plain" else [
                _off(a) if isinstance(a, torch.Tensor) and a.dtype == BF and a.is_contiguous() else a for a in args]
            for got in (impl(*cast), getattr(torch.ops.anima_flat_amd, name)(*cast)):
                pairs = list(zip([want] if isinstance(want, torch.Tensor) else want, [got] if isinstance(got, torch.Tensor) else got))
                assert all(p.shape == q.shape and p.dtype == q.dtype and torch.equal(p, q) for p, q in pairs), name


def _calls(mods):
    """Each differentiable operator as a function of its first argument."""
    adaln, _, ckpt8 = mods
    g = gen(2)
    y, m, a = bf(g, 1, 40, 256), bf(g, 1, 256), bf(g, 8, 256)
    return {
        "residual_adaln": lambda x: torch.cat(adaln.residual_adaln(x, y, m, m, m), -1),
        "adaln": lambda x: adaln.adaln(x, m, m),
        "gelu8": ckpt8.gelu8,
        "lora_down8": lambda x: ckpt8.lora_down8(x, a),
    }


NAMES = ["residual_adaln", "adaln", "gelu8", "lora_down8"]


@pytest.mark.parametrize("name", NAMES)
def test_autograd_behaviour(mods, name):
    """A second backward needs retain_graph; a double backward raises; graphs can be recorded by
    compiled autograd; outputs of calls without gradients have none."""
    run = _calls(mods)[name]
    x = bf(gen(3), 1, 40, 256).requires_grad_(True)
    out = run(x)
    seed = torch.ones_like(out)
    (want,) = torch.autograd.grad(out, [x], seed, retain_graph=True)
    assert torch.equal(torch.autograd.grad(out, [x], seed)[0], want)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, [x], seed)
    (first,) = torch.autograd.grad(run(x), [x], seed.clone().requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="no autograd formula"):
        first.float().sum().backward()
    with torch._dynamo.compiled_autograd._enable(torch.compile(backend="eager")):
        run(x).backward(seed)
    assert torch.equal(x.grad, want)
    with torch.no_grad():
        assert not run(x).requires_grad


@pytest.mark.parametrize("name", NAMES)
def test_fake_backward(mods, name):
    run = _calls(mods)[name]
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.empty(1, 40, 256, dtype=BF, device="cuda", requires_grad=True)
        out = run(x)
        (dx,) = torch.autograd.grad(out, [x], torch.empty_like(out))
        assert dx.shape == x.shape


@pytest.mark.parametrize("name", NAMES)
def test_functional_transforms_are_refused(mods, name):
    run = _calls(mods)[name]
    x = bf(gen(4), 1, 40, 256)
    with pytest.raises(RuntimeError, match="functorch transforms"):
        torch.func.grad(lambda v: run(v).float().sum())(x)


def test_changed_inputs_are_noticed(mods):
    """Autograd raises where a saved input was changed in place before the backward."""
    adaln = mods[0]
    x, y, m = bf(gen(5), 1, 4, 64).requires_grad_(True), bf(gen(6), 1, 4, 64), bf(gen(7), 1, 64)
    h = adaln.residual_adaln(x, y, m, m, m)[1]
    y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def test_no_gradient_through_int8(mods):
    adaln, int8, _ = mods
    m = bf(gen(8), 1, 64)
    x = bf(gen(9), 1, 4, 64).requires_grad_(True)
    for call in (lambda: adaln.residual_adaln_int8(x, x, m, m, m), lambda: int8.rowquant_int8(x)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()
