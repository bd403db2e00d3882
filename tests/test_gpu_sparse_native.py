"""Rotary positions and sparse attention: native dispatcher kernels against the Python functions,
autograd, transforms, captures, streams, and a run of them together."""

from __future__ import annotations

import importlib
import math

import pytest
import torch
import torch._dynamo.compiled_autograd
from torch._subclasses.fake_tensor import FakeTensorMode

from block_cases import BF, bf, gen
from conftest import REL_L2
from rotary_cases import turn
from sparse_cases import attend, heads, random_blocks, selected

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="session")
def mods(pkg):
    return [importlib.import_module("anima_flat_amd.kernels." + n) for n in ("rotary", "sparse")]


def _angles(g, *shape):
    a = 6.3 * torch.rand(*shape, generator=g).cuda()
    return a.cos(), a.sin()


def _cases():
    """Arguments of every op with native kernels, by name."""
    g = gen(31)
    q, k, v, dout = heads(g, 2, 130, 4), heads(g, 2, 200, 2), heads(g, 2, 200, 2), heads(g, 2, 130, 4)
    lens = torch.tensor([200, 70], dtype=torch.int32, device="cuda")
    blocks = random_blocks(g, 2, 4, 130, 200, 3, lens)
    cos, sin = _angles(g, 130, 32)
    k2 = heads(g, 2, 130, 2)
    few, short = blocks[:, :, :1].contiguous(), q[:, :64].contiguous()
    wide = torch.arange(9, dtype=torch.int32, device="cuda").expand(2, 4, 1, 9).contiguous()
    many = heads(g, 2, 600, 2)
    out, lse = torch.ops.anima_flat_amd.sparse_fwd(q, k, v, blocks, lens, True)
    positions = torch.randint(0, 1000, (2, 7, 3), generator=g).cuda()
    return {
        "rotary_tables": [(positions, [4, 6, 8], [1e4] * 3, [1.0, 2.0, 2.0], 0, 0.0), (positions[..., :1].float().contiguous(), [8], [1e4], [4.0], 2, 64.0)],
        "rotary": [(q, k2, cos, sin, False, False), (q, None, cos, sin, True, True), (q.float(), None, cos, sin, False, False)],
        "select_blocks": [(q, k, 2, lens), (q, k, 9, None)],
        "sparse_fwd": [(q, k, v, blocks, lens, True), (q, k, v, blocks, None, False), (short, k, v, few, lens, False), (short, many, many, wide, None, True)],
        "sparse_bwd": [(dout, q, k, v, out, lse, blocks, lens)],
    }


def _off(v):
    """The same values one element past a 16-byte boundary."""
    return torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v)


@pytest.mark.parametrize("form", ["plain", "misaligned"])
def test_python_functions_give_the_same_bits(mods, form):
    cases = _cases()
    native = importlib.import_module("anima_flat_amd._native")
    assert {"anima_flat_amd::" + n for n in cases} == native.NATIVE_SPARSE_OPS
    for name, calls in cases.items():
        (impl,) = [op._init_fn for m in mods for op in vars(m).values()
                   if isinstance(op, torch.library.CustomOpDef) and op._qualname == "anima_flat_amd::" + name]
        for args in calls:
            want = getattr(torch.ops.anima_flat_amd, name)(*args)
            cast = args if form == "plain" else [_off(a) if isinstance(a, torch.Tensor) and a.dtype in (BF, torch.float32) else a for a in args]
            for got in (impl(*cast), getattr(torch.ops.anima_flat_amd, name)(*cast)):
                pairs = list(zip([want] if isinstance(want, torch.Tensor) else want, [got] if isinstance(got, torch.Tensor) else got))
                assert all(p.shape == q.shape and p.dtype == q.dtype and torch.equal(p, q) for p, q in pairs), name


def test_contract(mods):
    """Inputs unchanged, outputs of their own memory, fakes of the same shapes, types, layout."""
    for name, calls in _cases().items():
        for args in calls:
            torch.library.opcheck(getattr(torch.ops.anima_flat_amd, name).default, args, test_utils=("test_schema", "test_faketensor"))


def _calls(mods):
    """Each differentiable operator as a function of its first argument [1, 130, 4, 128]."""
    rotary, sparse = mods
    g = gen(32)
    k, blocks = heads(g, 1, 200, 2), random_blocks(g, 1, 4, 130, 200, 3)
    cos, sin = _angles(g, 130, 64)
    return {
        "rotary": lambda x: rotary.rotary(x, cos, sin),
        "rotary_qk": lambda x: torch.cat(rotary.rotary_qk(x, x, cos, sin, True), 2),
        "sparse_attention": lambda x: sparse.sparse_attention(x, k, k, blocks),
        "selected": lambda x: sparse.sparse_attention(x, x, x, sparse.select_blocks(x, x, 2)),
    }


NAMES = ["rotary", "rotary_qk", "sparse_attention", "selected"]


def _x(seed):
    return heads(gen(seed), 1, 130, 4)


@pytest.mark.parametrize("name", NAMES)
def test_autograd_behaviour(mods, name):
    run = _calls(mods)[name]
    x = _x(33).requires_grad_(True)
    out = run(x)
    seed = torch.ones_like(out)
    (want,) = torch.autograd.grad(out, [x], seed, retain_graph=True)
    assert torch.equal(torch.autograd.grad(out, [x], seed)[0], want)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, [x], seed)
    if not name.startswith("rotary"):
        (first,) = torch.autograd.grad(run(x), [x], seed.clone().requires_grad_(True), create_graph=True)
        with pytest.raises(RuntimeError, match="no autograd formula"):
            first.float().sum().backward()
    with torch._dynamo.compiled_autograd._enable(torch.compile(backend="eager")):
        run(x).backward(seed)
    assert torch.equal(x.grad, want)
    with torch.no_grad():
        assert not run(x).requires_grad
    with torch.inference_mode():
        assert torch.equal(run(x.detach()), out)


@pytest.mark.parametrize("name", NAMES)
def test_fake_backward_and_transforms(mods, name):
    run = _calls(mods)[name]
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.empty(1, 130, 4, 128, dtype=BF, device="cuda", requires_grad=True)
        out = run(x)
        assert torch.autograd.grad(out, [x], torch.empty_like(out))[0].shape == x.shape
    with pytest.raises(RuntimeError, match="functorch transforms"):
        torch.func.grad(lambda v: run(v).float().sum())(_x(34))


def test_changed_inputs_are_noticed(mods):
    sparse = mods[1]
    q, k = _x(35).requires_grad_(True), _x(36)
    out = sparse.sparse_attention(q, k, k, sparse.select_blocks(q, k, 2))
    k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_refusals_on_the_gpu(mods):
    """What the native kernels do not take is refused as the fakes refuse it, before any launch."""
    rotary, sparse = mods

    def t(*shape, dtype=BF):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    q, k, blocks, table = t(2, 70, 4, 128), t(2, 90, 2, 128), t(2, 4, 2, 3, dtype=torch.int32), t(70, 64, dtype=torch.float32)
    cases = [(sparse.sparse_attention, args, says) for args, says in (
        ((q.half(), k.half(), k.half(), blocks), "only bfloat16"), ((q, k, k[:, :5], blocks), "must be"), ((q, k, k.float(), blocks), "only bfloat16"),
        ((q, k[..., :64], k[..., :64], blocks), "disagree"), ((q, t(2, 90, 3, 128), t(2, 90, 3, 128), blocks), "no multiple"),
        ((q, k, k, blocks[:, :, :1]), "blocks must be"), ((q, k, k, blocks.long()), "int32"), ((q, k, k, blocks.cpu()), "CUDA tensors"),
        ((q, k, k, blocks, t(2)), "seqused_k"), ((q, k, k, blocks, t(3, dtype=torch.int32)), "seqused_k"), ((q, k.cpu(), k, blocks), "CUDA tensors"),
    )]
    cases += [(sparse.select_blocks, args, says) for args, says in (
        ((q, k, 0), "count"), ((q, k, 4097), "count"), ((q.float(), k.float(), 1), "only bfloat16"), ((q[0], k, 1), "must be"), ((q, k[:1], 1), "disagree"),
    )]
    cases += [(rotary.rotary, args, says) for args, says in (
        ((q, table[:69], table[:69]), "cos and sin"), ((q, table, table.half()), "float32"), ((q, table.double(), table.double()), "float32"),
        ((q.double(), table, table), "unsupported dtype"), ((q[..., :60], table[:, :8], table[:, :8]), "multiple of 8"), ((q, table.cpu(), table), "CUDA tensors"),
    )]
    for call, args, says in cases:
        with pytest.raises(ValueError, match=says):
            call(*args)
    # Lengths of another integer type are read as they are.
    for values in ([5, 90], [-(2**40), 2**40]):
        lens = torch.tensor(values, device="cuda")
        assert torch.equal(sparse.select_blocks(q, k, 2, lens), sparse.select_blocks(q, k, 2, lens.clamp(0, 90).int()))


def _refused(call, *tensors):
    with pytest.raises(ValueError):
        call(*tensors)


def test_backward_refuses_what_is_not_the_forwards(mods):
    (args,) = _cases()["sparse_bwd"]
    dout, q, k, v, out, lse, blocks, lens = args
    op = torch.ops.anima_flat_amd.sparse_bwd
    for at, value in ((0, dout[:, :5]), (0, dout.float()), (4, out[:1]), (4, out.half()), (5, lse[:, :1]), (5, lse.half()), (5, lse.cpu()), (6, blocks[..., :0])):
        changed = list(args)
        changed[at] = value
        _refused(op, *changed)


# ---------------------------------------------------------------- captures --


@pytest.mark.parametrize("name", NAMES)
def test_captured_steps(mods, name):
    """Two graphs of whole steps, replayed in turn with eager work between, give the eager bits."""
    run = _calls(mods)[name]
    leaves = [_x(37).requires_grad_(True), _x(38).requires_grad_(True)]

    def step(x):
        out = run(x)
        return out.detach(), torch.autograd.grad(out, [x], torch.ones_like(out))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in leaves:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(x))
    for turn_ in range(4):
        with torch.no_grad():
            for i, x in enumerate(leaves):
                x.copy_(_x(40 + 2 * turn_ + i))
        want = [step(x) for x in leaves]
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for got, ref in zip(outs, want) for a, b in zip(got, ref)), turn_


@pytest.mark.parametrize("name", NAMES)
def test_capture_beside_a_live_graph(mods, name):
    run = _calls(mods)[name]
    p, q = _x(50).requires_grad_(True), _x(51).requires_grad_(True)
    live = run(p + q)
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run(p + q)
    torch.cuda.synchronize()
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(p + q)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, live)


def test_streams(mods):
    """Calls on two other streams at once, with split lists and their workspaces."""
    sparse = mods[1]
    g = gen(52)
    sets = [(heads(g, 1, 64, 2), heads(g, 1, 2000, 2), heads(g, 1, 2000, 2)) for _ in range(2)]
    want = [sparse.sparse_attention(q, k, v, sparse.select_blocks(q, k, 20)) for q, k, v in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, (q, k, v), to in zip(streams, sets, got):
            with torch.cuda.stream(s):
                to.append(sparse.sparse_attention(q, k, v, sparse.select_blocks(q, k, 20)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for outs, w in zip(got, want) for o in outs)


# ---------------------------------------------------------------- together --


@pytest.mark.parametrize("h,w", [(24, 40), (13, 21)])
def test_a_layer(pkg, mods, h, w):
    """What a layer does with an image's tokens, in patch order: tables of its rows and columns
    stretched to the size, turned queries and keys, the selection, the attention, back through
    all of it. Each step against 64 bits of what it was given; the whole against the dense
    attention where every block is selected."""
    rotary, sparse = mods
    g = gen(53)
    order, back = sparse.tile_order(h, w, "cuda")
    S, H, Hk = h * w, 4, 2
    positions = torch.stack((torch.zeros_like(order), order // w, order % w), -1)
    cos, sin = rotary.rotary_tables(positions, (44, 42, 42), scale=(1.0, 4.0, 4.0))
    c, s = pkg.rope_tables(h, w, 128, "cuda", (4.0, 4.0))
    assert (cos[back] - c).abs().max() < 1e-5 and (sin[back] - s).abs().max() < 1e-5
    qkv = bf(g, 1, S, (H + 2 * Hk) * 128).requires_grad_(True)
    x = qkv[:, order].unflatten(-1, (H + 2 * Hk, 128))
    q, k, v = x[:, :, :H], x[:, :, H : H + Hk], x[:, :, H + Hk :]
    tq, tk = rotary.rotary_qk(q, k, cos, sin)
    blocks = sparse.select_blocks(tq, tk, 3)
    out = sparse.sparse_attention(tq, tk, v, blocks)
    dout = heads(g, 1, S, H)
    (grad,) = torch.autograd.grad(out, [qkv], dout.flatten(2))

    assert torch.equal(blocks.cpu(), selected(tq.detach().cpu(), tk.detach().cpu(), 3))
    ref, err = attend(tq, tk, v, blocks, dout=dout)
    assert ((out.double().unflatten(-1, (H, 128)) - ref["out"]).abs() <= err["out"]).all()
    want = torch.cat((turn(ref["dq"], cos, -sin, False)[0], turn(ref["dk"], cos, -sin, False)[0], ref["dv"]), 2).flatten(2)
    got = grad.double()[:, order]
    # A turn keeps norms: the attention's gradients are off by REL_L2, their turn rounds once
    # more, and is of values rounded to bf16 before.
    assert (got - want).norm() <= (REL_L2 + 2 * 2.0**-8) * want.norm()

    every = torch.arange(-(-S // 64), dtype=torch.int32, device="cuda")
    with torch.no_grad():
        full = sparse.sparse_attention(tq, tk, v, every.expand(1, H, len(every), len(every)))
        dense = pkg.attention(tq[:, back], *(t[:, back].repeat_interleave(H // Hk, 2) for t in (tk, v)))
    assert (full[:, back].double() - dense.double()).norm() <= 2 * REL_L2 * dense.double().norm()
