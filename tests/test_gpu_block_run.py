"""The block's operators as they are used: an int8 inference block around attention, a LoRA
training step, both under graph capture, on several streams, with block checkpointing."""

from __future__ import annotations

import importlib
import threading

import pytest
import torch
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

from block_cases import BF, U16, bf, gen, within
from oracle import block_oracle as ref

pytestmark = pytest.mark.gpu

H, HD, D, MLP, RANK = 2, 128, 256, 1024, 16
EPS = 1e-6


@pytest.fixture(scope="session")
def mods(pkg):
    return [importlib.import_module("anima_flat_amd.kernels." + n) for n in ("adaln", "int8", "ckpt8")]


def _weights(int8, seed=0):
    g = gen(seed)
    shapes = {"qkv": (3 * D, D), "o": (D, D), "up": (MLP, D), "down": (D, MLP)}
    w = {k: bf(g, *s, scale=s[1] ** -0.5) for k, s in shapes.items()}
    return w, {k: int8.quantize_weight(v) for k, v in w.items()}


def _modulation(B, seed):
    m = bf(gen(seed), B, 8 * D, scale=0.3)
    return m.chunk(8, -1)


def _int8_block(pkg, mods, x, y, mod, w8, qw, cos, sin):
    """Norm -> QKV -> attention -> output projection -> norm -> MLP -> norm, projections in int8."""
    adaln, int8, _ = mods
    sh1, sc1, g1, sh2, sc2, g2, sh3, sc3 = mod
    r, q, s = adaln.residual_adaln_int8(x, y, g1, sc1, sh1, eps=EPS)
    qkv = int8.int8_linear(q, s, *w8["qkv"])
    qh, kh, vh = pkg.qkv_norm_rope(qkv, qw, qw, cos, sin, H, EPS)
    att = pkg.attention(qh, kh, vh)
    o = int8.int8_linear(*int8.rowquant_int8(att), *w8["o"])
    r2, q2, s2 = adaln.residual_adaln_int8(r, o, g2, sc2, sh2, eps=EPS)
    up = int8.int8_linear(q2, s2, *w8["up"])
    down = int8.int8_linear(*int8.rowquant_int8(up, gelu=True), *w8["down"])
    r3, h3 = adaln.residual_adaln(r2, down, g2, sc3, sh3, eps=EPS)
    return {"r": r, "q": q, "s": s, "qkv": qkv, "att": att, "o": o, "r2": r2, "q2": q2, "s2": s2, "up": up,
            "down": down, "r3": r3, "h3": h3}


def _block_inputs(pkg, mods, B, S, seed):
    g = gen(seed)
    x, y = bf(g, B, S, D), bf(g, B, S, D)
    qw = (1 + 0.02 * torch.randn(HD, generator=g)).cuda()
    cos, sin = pkg.rope_tables(1, S, HD, "cuda")
    return x, y, _modulation(B, seed + 1), _weights(mods[1], seed + 2)[1], qw, cos, sin


@pytest.mark.parametrize("B,S", [(1, 1), (2, 75), (1, 300)])
def test_int8_block(pkg, mods, B, S):
    """Every int8 step of the run against 64 bits on the tensors that reached it."""
    args = _block_inputs(pkg, mods, B, S, 3)
    x, y, mod, w8 = args[:4]
    t = _int8_block(pkg, mods, *args)

    def product(q, s, w):
        return (q.double().flatten(0, 1) @ w[0].double().t()).view(*q.shape[:2], -1) * s.double().view(*q.shape[:2], 1) * w[1].double()

    for q, s, w, out in ((t["q"], t["s"], "qkv", "qkv"), (t["q2"], t["s2"], "up", "up")):
        want = product(q, s, w8[w])
        within(t[out], want, 1.001 * U16 * want.abs(), out)
    q, s = ref.int8_rows(t["att"].float())
    want = product(q, s, w8["o"])
    within(t["o"], want, 1.001 * U16 * want.abs(), "o")
    # After GELU a code may fall on the other side of a tie: a step times the largest weight each,
    # for at most 1 code in 1000.
    q, s = ref.int8_rows(ref.gelu(t["up"].double()).float())
    want = product(q, s, w8["down"])
    flips = s.double().view(B, S, 1) * 127 * w8["down"][1].double() * (1 + MLP // 1000)
    within(t["down"], want, 1.001 * U16 * want.abs() + 1e-4 * want.abs() + flips, "down")
    r, h = ref.residual_adaln(t["r2"].double(), t["down"].double(), mod[5].double(), mod[7].double(), mod[6].double(), eps=EPS)
    within(t["r3"], r, 1.001 * U16 * r.abs() + 1e-5, "r3")
    within(t["h3"], h, 1.001 * U16 * h.abs() + 1e-4, "h3")


def _lora(seed, names=("up", "down")):
    g = gen(seed)
    out = {}
    for n, (o, i) in zip(names, ((MLP, D), (D, MLP))):
        out[n + "_a"] = (torch.randn(RANK, i, generator=g) * i**-0.5).cuda().requires_grad_(True)
        out[n + "_b"] = (torch.randn(o, RANK, generator=g) * 0.1).cuda().requires_grad_(True)
    return out


def _lora_block(mods, x, y, mod, w, lora):
    """The MLP half of a block with LoRA adapters (fp32 parameters, bf16 compute)."""
    adaln, _, ckpt8 = mods
    sh1, sc1, g1, sh2, sc2, g2 = mod[:6]

    def linear(h, n):
        low = ckpt8.lora_down8(h, lora[n + "_a"].to(BF))
        return F.linear(h, w[n]) + F.linear(low, lora[n + "_b"].to(BF))

    r, h = adaln.residual_adaln(x, y, g1, sc1, sh1, eps=EPS)
    return adaln.residual_adaln(r, linear(ckpt8.gelu8(linear(h, "up")), "down"), g2, sc2, sh2, eps=EPS)


def _lora_block64(x, y, mod, w, lora):
    sh1, sc1, g1, sh2, sc2, g2 = (m.detach().double() for m in mod[:6])

    def linear(h, n):
        return h @ w[n].double().t() + h @ lora[n + "_a"].t() @ lora[n + "_b"].t()

    r, h = ref.residual_adaln(x, y, g1, sc1, sh1, eps=EPS)
    return ref.residual_adaln(r, linear(ref.gelu(linear(h, "up")), "down"), g2, sc2, sh2, eps=EPS)


def _train_inputs(mods, B, S, seed):
    g = gen(seed)
    x, y = (bf(g, B, S, D).requires_grad_(True) for _ in range(2))
    w, _ = _weights(mods[1], seed + 2)
    return x, y, _modulation(B, seed + 1), w, _lora(seed + 3), bf(g, B, S, D), bf(g, B, S, D)


def _train_step(mods, x, y, mod, w, lora, dr, dh, wrap=None):
    run = lambda x, y: _lora_block(mods, x, y, mod, w, lora)  # noqa: E731
    out = run(x, y) if wrap is None else wrap(run, x, y)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, [x, y, *lora.values()], [dr, dh]))


@pytest.mark.parametrize("B,S", [(1, 1), (2, 75), (1, 520)])
def test_lora_step(mods, B, S):
    """Outputs and gradients against 64 bits without any rounding. On the way of a value stand at
    most 14 roundings to bf16 (2^-8 at most, each) and, in a's gradients and through GELU's
    slope, one 8-bit copy (2^-7 of its group's largest, at most 4 times a value's usual size):
    14 * 2^-8 + 4 * 2^-7 = 0.086 of the norm at the very most."""
    args = _train_inputs(mods, B, S, 11)
    got = _train_step(mods, *args)
    x, y, mod, w, lora, dr, dh = args
    xd, yd = (v.detach().double().requires_grad_(True) for v in (x, y))
    ld = {k: v.detach().to(BF).double().requires_grad_(True) for k, v in lora.items()}
    out = _lora_block64(xd, yd, mod, w, ld)
    want = [o.detach() for o in out] + list(torch.autograd.grad(out, [xd, yd, *ld.values()], [dr.double(), dh.double()]))
    names = ["r", "h", "dx", "dy", *lora]
    for n, a, b in zip(names, got, want):
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off < 0.086, (n, off)


def test_block_checkpointing(mods):
    """torch.utils.checkpoint runs the forward again in the backward: the same bits."""
    args = _train_inputs(mods, 2, 33, 21)
    want = _train_step(mods, *args)
    got = _train_step(mods, *args, wrap=lambda run, x, y: checkpoint(run, x, y, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def _captured(step):
    """A graph of step() and the outputs that replays fill."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


def test_graph_replays(pkg, mods):
    """An inference block and a training step, two sizes each, captured: replays in turn, with
    eager work between them and new values in the inputs, give the eager bits."""
    cases = []
    for B, S in ((1, 40), (2, 300)):
        args = _block_inputs(pkg, mods, B, S, B + S)
        cases.append((args[0], lambda a=args: list(_int8_block(pkg, mods, *a).values())))
        targs = _train_inputs(mods, B, S, B + S)
        cases.append((targs[5], lambda a=targs: _train_step(mods, *a)))
    graphs = [(v, step, *_captured(step)) for v, step in cases]
    for turn in range(3):
        for changed, step, graph, out in graphs:
            changed.copy_(bf(gen(100 + turn), *changed.shape))
            want = [t.clone() for t in step()]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_streams_and_threads(mods):
    """Training steps from several threads, each on its own stream, workspaces in use at once."""
    args = [_train_inputs(mods, 1, 700, 31 + i) for i in range(4)]
    want = [_train_step(mods, *a) for a in args]
    torch.cuda.synchronize()
    got = [None] * len(args)

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(8):
                got[i] = _train_step(mods, *args[i])
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(args))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_trained_modulation(mods):
    """Gradients reach a modulation projection through the chunked rows of both norms."""
    adaln, _, _ = mods
    g = gen(41)
    x, y = bf(g, 2, 60, D), bf(g, 2, 60, D)
    emb, w = torch.randn(2, 32, generator=g).cuda(), (torch.randn(3 * D, 32, generator=g) * 0.05).cuda().requires_grad_(True)
    dr, dh = bf(g, 2, 60, D), bf(g, 2, 60, D)

    def loss(run, w, emb, *ts):
        x, y, dr, dh = ts
        shift, scale, gate = F.linear(emb, w).chunk(3, -1)
        r, h = run(x, y, gate, scale, shift, eps=EPS)
        return (r * dr).sum() + (h * dh).sum()

    out = torch.autograd.grad(loss(lambda *a, **k: tuple(v.float() for v in adaln.residual_adaln(*a, **k)), w, emb, x, y, dr, dh), [w])[0]
    wd = w.detach().double().requires_grad_(True)
    want = torch.autograd.grad(loss(ref.residual_adaln, wd, emb.double(), *(v.double() for v in (x, y, dr, dh))), [wd])[0]
    # Sums of 60 tokens in fp32, of bf16 gradients that are exact inputs: dr and dh pass a cast.
    torch.testing.assert_close(out.double(), want, rtol=1e-4, atol=1e-4 * want.abs().max().item())


def test_two_norms_of_one_stream(mods):
    """The residual stream used by two operators: their gradients add up in autograd."""
    adaln, _, _ = mods
    g = gen(42)
    x, y = bf(g, 1, 9, D).requires_grad_(True), bf(g, 1, 9, D)
    m = torch.zeros(1, D, device="cuda")
    r, h = adaln.residual_adaln(x, y, m + 1, m, m, eps=EPS)
    h2 = adaln.adaln(r, m, m, eps=EPS)
    assert (h.float() - h2.float()).abs().max() < 0.05  # of the fp32 r, of the bf16 r
    dx, dr = torch.autograd.grad([h, h2], [x, r], [torch.ones_like(h), torch.ones_like(h)])
    assert torch.isfinite(dx.float()).all() and torch.isfinite(dr.float()).all()


def test_capture_beside_a_live_graph(mods):
    """A captured forward with gradients is refused while an eager graph of its leaves lives on
    the default stream (whose accumulators could not join the capture), and taken after it."""
    adaln, _, ckpt8 = mods
    g = gen(61)
    x, a, m = bf(g, 1, 40, 64).requires_grad_(True), torch.randn(8, 64, generator=g).cuda().requires_grad_(True), bf(g, 1, 64)
    dt = bf(g, 1, 40, 8)
    steps = [
        lambda: torch.autograd.grad(adaln.residual_adaln(x, x, m, m, m)[1], [x], x.detach()),
        lambda: torch.autograd.grad(adaln.adaln(x, m, m), [x], x.detach()),
        lambda: torch.autograd.grad(ckpt8.gelu8(x), [x], x.detach()),
        lambda: torch.autograd.grad(ckpt8.lora_down8(x.detach(), a.to(BF)), [a], dt),
    ]
    want = [[t.clone() for t in step()] for step in steps]
    live = x.float() * 2, a.to(BF)
    for step in steps:
        with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                step()
        torch.cuda.synchronize()
    del live
    for step, first in zip(steps, want):
        graph, out = _captured(step)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, first))
            assert all(torch.equal(p, q) for p, q in zip(step(), first))
