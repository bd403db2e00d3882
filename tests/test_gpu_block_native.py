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


def test_refusals_on_the_gpu(mods):
    """What the native kernels do not take is refused as the fakes refuse it, before any launch."""
    adaln, int8, ckpt8 = mods

    def t(*shape, dtype=BF):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    x, m = t(2, 5, 64), t(2, 64)
    cases = [
        (f, args, says) for f in (adaln.residual_adaln, adaln.residual_adaln_int8) for args, says in (
            ((x.half(), x.half(), m, m, m), "only bfloat16"),
            ((x, t(2, 5, 72), m, m, m), "x's shape"),
            ((x, x.cpu(), m, m, m), "CUDA tensors"),
            ((x[0], x[0], m, m, m), "must be .B, S, D"),
            ((t(2, 5, 60), t(2, 5, 60), t(2, 60), t(2, 60), t(2, 60)), "multiple of 8"),
            ((t(1, 2, 8200), t(1, 2, 8200), t(8200), t(8200), t(8200)), "at most 8192"),
            ((x, x, t(3, 64), m, m), "gate must be"),
            ((x, x, m, t(2, 5, 64), m), "scale must be"),
            ((x, x, m, m, t(2, 32)), "shift must be"),
            ((x, x, m, m, m.half()), "must be bfloat16 or float32"),
            ((x, x, m, m, m, t(32)), "weight must be"),
            ((x, x, m, m, m, t(1, 64)), "weight must be"),
            ((x, x, m, m, m, t(64).half()), "weight must be"),
            ((x, x, m, m, m, t(64).double()), "weight must be"),
        )
    ]
    q, s, w, ws = t(2, 5, 64, dtype=torch.int8), t(10, 1, dtype=torch.float32), t(8, 64, dtype=torch.int8), t(8, dtype=torch.float32)
    cases += [(int8.int8_linear, args, says) for args, says in (
        ((x, s, w, ws), "q must be"), ((q[0], s, w, ws), "q must be"), ((q, s[:9], w, ws), "s must be"),
        ((q, s.half(), w, ws), "s must be"), ((q, s, w[:, :48], ws), "weight must be"),
        ((q, s, w.float(), ws), "weight must be"), ((q, s, w, ws[:4]), "weight_scale must be"),
        ((q, s, w, ws.double()), "weight_scale must be"), ((q, s, w, ws.cpu()), "CUDA tensors"),
        ((q[..., :24], s, w[:, :24], ws), "multiple of 16"), ((q, s, w[:4], ws[:4]), "multiple of 8"),
    )]
    cases += [
        (int8.rowquant_int8, (m,), "B, S, K"), (int8.rowquant_int8, (x.half(),), "only bfloat16"),
        (int8.rowquant_int8, (t(1, 1, 12),), "multiple of 8"), (int8.rowquant_int8, (t(1, 1, 8200),), "at most 8192"),
        (ckpt8.gelu8, (x.float(),), "only bfloat16"), (ckpt8.gelu8, (x[0],), "B, S, K"),
        (ckpt8.gelu8, (t(1, 1, 12),), "multiple of 8"), (ckpt8.gelu8, (t(1, 1, 65544),), "at most 65536"),
    ] + [(ckpt8.lora_down8, (x, a), says) for a, says in (
        (t(12, 64), "rank"), (t(72, 64), "rank"), (t(0, 64), "rank"), (t(8, 72), "a must be"),
        (t(8, 64).float(), "a must be"), (t(8, 64).cpu(), "CUDA tensors"),
    )]
    for call, args, says in cases:
        with pytest.raises(ValueError, match=says):
            call(*args)


@pytest.mark.parametrize("name", NAMES)
def test_inference_mode(mods, name):
    run = _calls(mods)[name]
    x = bf(gen(12), 1, 40, 256)
    want = run(x)
    with torch.inference_mode():
        assert torch.equal(run(x), want)
    assert torch.equal(run(x), want)


def test_backward_refuses_what_is_not_the_forwards(mods):
    """The backward ops take only statistics and copies of the sizes that their forward makes."""
    ops = torch.ops.anima_flat_amd
    cases = _cases()

    def refused(name, args, *changes):
        for at, value in changes:
            changed = list(args)
            changed[at] = value
            with pytest.raises(ValueError):
                getattr(ops, name)(*changed)

    args = cases["adaln_bwd"][0]
    dr, x, stats = args[0], args[2], args[7]
    refused("adaln_bwd", args, (0, dr[:1]), (0, dr.float()), (1, dr[..., :256]), (3, None), (4, None), (7, stats[:-1]),
            (7, stats.half()), (7, stats.cpu()), (8, 3), (2, x[:1]))
    dy, codes, exps = cases["gelu8_bwd"][0]
    refused("gelu8_bwd", (dy, codes, exps), (0, dy.float()), (0, dy[:1]), (1, codes[:-1]), (1, codes.cpu()), (2, exps[:, :-1]),
            (2, exps.float()))
    args = cases["lora_down8_bwd"][0]
    dt, a, codes, exps = args[:4]
    refused("lora_down8_bwd", args, (0, dt.float()), (0, dt[..., :8]), (0, dt[:1]), (1, a[:8]), (1, a.cpu()), (2, codes[:-1]),
            (3, exps[:-1]))
