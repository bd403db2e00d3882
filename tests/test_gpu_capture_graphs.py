"""Captured forwards with gradients beside a live eager graph that reaches their inputs through
operations of several inputs. Only forwards are captured there: they must raise before a backward
could make the default stream wait for the capture."""

from __future__ import annotations

import importlib

import pytest
import torch
import torch.nn.functional as F

from block_cases import BF, bf, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods(pkg):
    return [importlib.import_module("anima_flat_amd.kernels." + n) for n in ("adaln", "int8", "ckpt8")]


def _leaves():
    g = gen(71)
    t = {k: bf(g, 1, 40, 64).requires_grad_(True) for k in ("p", "q")}
    t["emb"], t["w"] = bf(g, 1, 32), bf(g, 3 * 64, 32).requires_grad_(True)
    t["a"], t["b"] = (bf(g, 8, 64).requires_grad_(True) for _ in range(2))
    return t


def _calls(mods, t):
    """Each operator on inputs that several leaves or a product make."""
    adaln, _, ckpt8 = mods
    plain = bf(gen(72), 1, 40, 64)

    def rows():
        return F.linear(t["emb"], t["w"]).chunk(3, -1)

    def stacked():  # through another of these operators
        m = rows()
        return adaln.adaln(adaln.residual_adaln(plain, t["p"], *m)[0], m[0], m[1])

    return {
        "sum": lambda: ckpt8.gelu8(t["p"] + t["q"]),
        "projected modulation": lambda: adaln.residual_adaln(plain, plain, *rows())[1],
        "modulation alone": lambda: adaln.adaln(plain, *rows()[:2]),
        "sum of adapters": lambda: ckpt8.lora_down8(plain, t["a"] + t["b"]),
        "operators in turn": stacked,
    }


NAMES = ["sum", "projected modulation", "modulation alone", "sum of adapters", "operators in turn"]


@pytest.mark.parametrize("name", NAMES)
def test_refused_beside_a_live_graph(mods, name):
    t = _leaves()
    run = _calls(mods, t)[name]
    live = run()  # an eager graph of the same leaves
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run()
    torch.cuda.synchronize()
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, live)


@pytest.mark.parametrize("name", ["x", "adapter"])
def test_refused_behind_an_eager_operation(mods, name):
    """The input itself is the live graph's."""
    t = _leaves()
    x, a = t["p"] * t["q"], t["a"] + t["b"]
    run = {"x": lambda: mods[2].gelu8(x), "adapter": lambda: mods[2].lora_down8(x.detach(), a)}[name]
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run()
    torch.cuda.synchronize()


@pytest.mark.parametrize("name", NAMES)
def test_taken_without_one(mods, name):
    """The whole step is captured once no eager graph lives, and replays give the eager bits."""
    t = _leaves()
    run = _calls(mods, t)[name]
    leaves = [v for v in t.values() if v.requires_grad]

    def step():
        out = run()
        return out.detach(), *(g for g in torch.autograd.grad(out, leaves, torch.ones_like(out), allow_unused=True) if g is not None)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        with torch.no_grad():
            for v in leaves:
                v.copy_(bf(gen(80 + turn), *v.shape))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert len(want) > 1 and all(torch.equal(p, q) for p, q in zip(out, want)), turn
