"""The block's operators around attention, as cases that a timing program can run.

`own` chooses between the plain form (elementary torch operations in 32 bits,
rounded once at the end) and the framework's operators. `kind` says which:

  norm         residual_adaln, no grad: x + gate * y, LayerNorm, modulation
  norm_train   the same, forward and backward; `mods`: gradients of the
               modulation too, `post`: an RMSNorm on the block's output before
               the gate, `bm`: rows of modulation (B, or 1 for all of a batch)
  norm_linear  residual_adaln_int8 and the int8 projection of its tokens
  linear       rowquant_int8 (after GELU where `gelu`) and int8_linear
  gelu_train   gelu8 forward and backward: the input kept in 8 bits
  lora_train   lora_down8 forward and backward: the input kept in 8 bits

Sizes are the model's (width 2048, MLP width 8192, 512 text tokens of width
1024, one token per 16 x 16 pixels: 256 to 9216 tokens an image; batch 2 is
classifier-free guidance's two branches) or generic.
"""

from __future__ import annotations

import math

import torch

own = False

BF = torch.bfloat16
EPS = 1e-6
GROUP = 32  # channels that share a power of two in an 8-bit checkpoint


def listed():
    return [
        # Between two sublayers at 256 x 256, one branch: the smallest call,
        # where a launch's fixed cost weighs most.
        {"name": "norm_256", "kind": "norm", "B": 1, "S": 256, "D": 2048},
        # ... of a guided step at 1024 x 1024, the model's native size.
        {"name": "norm_1024", "kind": "norm", "B": 2, "S": 4096, "D": 2048},
        # The same place in LoRA training at 1024 x 1024: the modulation is frozen.
        {"name": "norm_train_1024", "kind": "norm_train", "B": 1, "S": 4096, "D": 2048, "mods": False, "post": False, "bm": 1},
        # Training of a whole block with norms before and after its sublayers:
        # gradients of the modulation (one for the batch) and of the norm's
        # weight; odd sizes.
        {"name": "norm_train_all", "kind": "norm_train", "B": 3, "S": 1001, "D": 1544, "mods": True, "post": True, "bm": 1},
        # The norm and the QKV projection in int8, guided step at 832 x 1216
        # (3952 tokens, ragged in every tile size).
        {"name": "norm_qkv_832x1216", "kind": "norm_linear", "B": 2, "S": 3952, "K": 2048, "N": 6144},
        # A modulation's projection of the time embedding: one token per branch.
        {"name": "linear_time", "kind": "linear", "B": 2, "S": 1, "K": 2048, "N": 6144, "gelu": False},
        # One layer's text keys and values, a trimmed context of 333 tokens.
        {"name": "linear_text", "kind": "linear", "B": 2, "S": 333, "K": 1024, "N": 4096, "gelu": False},
        # The MLP's first product at 1024 x 1024, one branch.
        {"name": "linear_up_1024", "kind": "linear", "B": 1, "S": 4096, "K": 2048, "N": 8192, "gelu": False},
        # The MLP's second product with its GELU, guided step at 1536 x 1536:
        # the largest.
        {"name": "linear_down_1536", "kind": "linear", "B": 2, "S": 9216, "K": 8192, "N": 2048, "gelu": True},
        # The MLP's GELU in LoRA training at 1024 x 1024.
        {"name": "gelu_train_1024", "kind": "gelu_train", "B": 1, "S": 4096, "K": 8192},
        # LoRA training: the low-rank product of a projection of the block's
        # width at 1024 x 1024, rank 16.
        {"name": "lora_train_1024", "kind": "lora_train", "B": 1, "S": 4096, "K": 2048, "R": 16},
        # ... of the MLP's second product, two items at 832 x 1216, a higher rank.
        {"name": "lora_train_mlp", "kind": "lora_train", "B": 2, "S": 3952, "K": 8192, "R": 40},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def _wide(rng, a, b, step):
    return max(step, _log(rng, a, b) // step * step)


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1.5e15)


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    kind = rng.choice(("norm", "norm_train", "norm_train", "norm_linear", "linear", "linear", "gelu_train", "lora_train"))
    while True:
        c = {"kind": kind, "B": rng.choice((1, 1, 2, 2, 3, 4)), "S": _log(rng, 1, 9216)}
        if kind in ("norm", "norm_train"):
            c["D"] = _wide(rng, 256, 4096, 8)
        if kind == "norm_train":
            c |= {"mods": rng.random() < 0.5, "post": rng.random() < 0.5, "bm": rng.choice((1, c["B"]))}
        if kind in ("norm_linear", "linear"):
            c |= {"K": _wide(rng, 256, 4096 if kind == "norm_linear" else 8192, 16), "N": _wide(rng, 64, 8192, 8)}
        if kind == "linear":
            c["gelu"] = rng.random() < 0.3
        if kind == "gelu_train":
            c["K"] = _wide(rng, 256, 8192, 8)
        if kind == "lora_train":
            c |= {"K": _wide(rng, 256, 8192, 8), "R": 8 * rng.randint(1, 8)}
        if _cost(c) <= most[kind]:
            return c


# ------------------------------------------------------------------ inputs --


def prepare(case, seed):
    """The case's tensors on the GPU, from the seed alone. The residual stream
    has a few channels of large values, as a trained model's does; branch
    outputs, gradients and GELU inputs are N(0, 1) times a size per channel;
    the modulation is N(0, 0.3^2). Weights are in hand as int8 codes with a
    scale per output channel."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    def channels(*shape):
        return n(*shape) * (0.5 + torch.rand(shape[-1], generator=g, device="cuda"))

    kind, B, S = case["kind"], case["B"], case["S"]
    t = dict(case)
    if kind in ("norm", "norm_train", "norm_linear"):
        D = case["K"] if kind == "norm_linear" else case["D"]
        big = torch.ones(D, device="cuda")
        big[torch.randint(0, D, (4,), generator=g, device="cuda")] = 12.0
        x, y = (channels(B, S, D) * big).to(BF), channels(B, S, D).to(BF)
        bm = case.get("bm", B)
        # What the modulation's projection gives: shift, scale and gate side by
        # side in one row; in fp32 where it is trained.
        mod = n(bm, 3 * D, scale=0.3).to(torch.float32 if case.get("mods") else BF)
        shift, scale, gate = mod.chunk(3, -1)
        t |= {"x": x, "y": y, "shift": shift, "scale": scale, "gate": gate, "weight": None}
        if kind == "norm_train":
            if case["post"]:
                t["weight"] = 1 + 0.1 * n(D)
            t |= {"dr": n(B, S, D).to(BF), "dh": n(B, S, D).to(BF)}
            leaves = ["x", "y"]
            if case["mods"]:
                leaves += ["gate", "scale", "shift"]
                if case["post"]:
                    leaves.append("weight")
            for k in leaves:
                t[k] = t[k].detach().requires_grad_(True)
            t["leaves"] = leaves
    if kind in ("norm_linear", "linear"):
        w = n(case["N"], case["K"], scale=case["K"] ** -0.5)
        ws = w.abs().amax(1) / 127
        t |= {"wq": torch.round(w / ws[:, None]).to(torch.int8), "ws": ws}
    if kind == "linear":
        t["x"] = channels(B, S, case["K"]).to(BF)
    if kind in ("gelu_train", "lora_train"):
        t["x"] = (channels(B, S, case["K"]) * 1.3).to(BF).requires_grad_(True)
    if kind == "gelu_train":
        t["dy"] = n(B, S, case["K"]).to(BF)
    if kind == "lora_train":
        t["a"] = n(case["R"], case["K"], scale=case["K"] ** -0.5).to(BF).requires_grad_(True)
        t["dt"] = n(B, S, case["R"]).to(BF)
    return t


# -------------------------------------------------------------- plain form --


def _gelu(x):
    return 0.5 * x * torch.special.erfc(x * -(0.5**0.5))


def _norm(t):
    """(r, h) in 32 bits."""
    x, y = t["x"].float(), t["y"].float()
    gate, scale, shift = (t[k].float()[:, None] for k in ("gate", "scale", "shift"))
    if t["weight"] is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * t["weight"]
    r = x + gate * y
    c = r - r.mean(-1, keepdim=True)
    return r, c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * (1 + scale) + shift


def _int8_rows(x):
    s = x.abs().amax(-1, keepdim=True).clamp_min(1e-12) / 127
    return torch.round(x / s).clamp(-127, 127), s


def _int8_product(q, s, t):
    return ((q @ t["wq"].float().t()) * s * t["ws"]).to(BF)


def _checkpoint(x):
    """x as an 8-bit checkpoint holds it: codes of -127 to 127 times a power of
    two per GROUP channels, the one that puts the largest in 64 to 128."""
    K = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -K % GROUP)).unflatten(-1, (-1, GROUP))
    e = torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 7
    step = ((e.clamp(-126, 121) + 127) << 23).view(torch.float32)  # 2^e
    return (torch.round(v / step).clamp(-127, 127) * step).flatten(-2)[..., :K]


def _plain(t):
    kind = t["kind"]
    if kind == "norm":
        r, h = _norm(t)
        return [r.to(BF), h.to(BF)]
    if kind == "norm_train":
        r, h = _norm(t)
        grads = torch.autograd.grad([r, h], [t[k] for k in t["leaves"]], [t["dr"].float(), t["dh"].float()])
        return [r.detach().to(BF), h.detach().to(BF), *grads]
    if kind == "norm_linear":
        r, h = _norm(t)
        return [r.to(BF), _int8_product(*_int8_rows(h), t)]
    if kind == "linear":
        x = t["x"].float()
        return _int8_product(*_int8_rows(_gelu(x) if t["gelu"] else x), t)
    x = t["x"].detach()
    kept = _checkpoint(x)
    if kind == "gelu_train":
        y = _gelu(x.float())
        slope = 0.5 * torch.special.erfc(kept * -(0.5**0.5)) + kept * torch.exp(-0.5 * kept * kept) * (2 * math.pi) ** -0.5
        return [y.to(BF), (t["dy"].float() * slope).to(BF)]
    a, dt = t["a"].detach().float(), t["dt"].float()
    return [(x.float() @ a.t()).to(BF), (dt @ a).to(BF), (dt.flatten(0, 1).t() @ kept.flatten(0, 1)).to(BF)]


# ------------------------------------------------------------- the framework --


def _modules():
    import importlib

    import __graft_entry__

    __graft_entry__.load_package()
    return [importlib.import_module("anima_flat_amd.kernels." + m) for m in ("adaln", "int8", "ckpt8")]


_loaded = []


def _framework(t):
    if not _loaded:
        _loaded.extend(_modules())
    adaln, int8, ckpt8 = _loaded
    kind = t["kind"]
    if kind == "norm":
        return adaln.residual_adaln(t["x"], t["y"], t["gate"], t["scale"], t["shift"], eps=EPS)
    if kind == "norm_train":
        out = adaln.residual_adaln(t["x"], t["y"], t["gate"], t["scale"], t["shift"], weight=t["weight"], eps=EPS)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, [t[k] for k in t["leaves"]], [t["dr"], t["dh"]]))
    if kind == "norm_linear":
        r, q, s = adaln.residual_adaln_int8(t["x"], t["y"], t["gate"], t["scale"], t["shift"], eps=EPS)
        return [r, int8.int8_linear(q, s, t["wq"], t["ws"])]
    if kind == "linear":
        q, s = int8.rowquant_int8(t["x"], gelu=t["gelu"])
        return int8.int8_linear(q, s, t["wq"], t["ws"])
    if kind == "gelu_train":
        y = ckpt8.gelu8(t["x"])
        return [y.detach(), *torch.autograd.grad(y, [t["x"]], t["dy"])]
    low = ckpt8.lora_down8(t["x"], t["a"])
    return [low.detach(), *torch.autograd.grad(low, [t["x"], t["a"]], t["dt"])]


def run(state):
    return _framework(state) if own else _plain(state)


# -------------------------------------------------------------------- work --


def work(case):
    kind, rows = case["kind"], case["B"] * case["S"]
    if kind in ("norm", "norm_train"):
        n, bm = rows * case["D"], case.get("bm", case["B"])
        if kind == "norm":
            return {"bytes": 8 * n + 6 * bm * case["D"], "flops": 12 * n}
        # The inputs and both gradients once, both results and both gradients once.
        extra = (12 * bm * case["D"] if case["mods"] else 0) + 12 * bm * case["D"]
        return {"bytes": 16 * n + extra, "flops": (40 if case["post"] else 30) * n}
    if kind in ("norm_linear", "linear"):
        K, N = case["K"], case["N"]
        moved = (6 if kind == "norm_linear" else 2) * rows * K + N * K + 4 * N + 2 * rows * N
        return {"bytes": moved, "flops": 2 * rows * N * K}
    n = rows * case["K"]
    if kind == "gelu_train":  # x and dy in, y and dx out
        return {"bytes": 8 * n, "flops": 40 * n}
    return {"bytes": 4 * n + 4 * rows * case["R"] + 4 * case["R"] * case["K"], "flops": 6 * n * case["R"]}


# ------------------------------------------------------------------- exact --


def exact(case, seed):
    t = prepare(case, seed)
    f = {k: v.detach().double() for k, v in t.items() if isinstance(v, torch.Tensor)}
    kind = case["kind"]
    x = f["x"]
    if kind.startswith("norm"):
        y, D = f["y"], x.shape[-1]
        gate, scale, shift = f["gate"].unsqueeze(1), f["scale"].unsqueeze(1), f["shift"].unsqueeze(1)
        ry = yh = None
        branch = y
        if t["weight"] is not None:
            ry = (y.pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5)
            yh = y * ry
            branch = yh * f["weight"]
        r = x + gate * branch
        mu = r.sum(-1, keepdim=True) / D
        rstd = ((r - mu).pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5)
        xh = (r - mu) * rstd
        h = xh + xh * scale + shift
        if kind == "norm":
            return [r, h]
        if kind == "norm_train":
            u = f["dh"] * (1 + scale)
            d = f["dr"] + rstd * (u - u.sum(-1, keepdim=True) / D - xh * ((u * xh).sum(-1, keepdim=True) / D))
            db = gate * d
            if ry is None:
                dy = db
            else:
                v = db * f["weight"]
                dy = ry * (v - yh * ((v * yh).sum(-1, keepdim=True) / D))
            out = [r, h, d, dy]
            if case["mods"]:
                over = (0, 1) if case["bm"] == 1 else (1,)
                for grad in (d * branch, f["dh"] * xh, f["dh"]):
                    out.append(grad.sum(over).reshape(case["bm"], D))
                if case["post"]:
                    out.append((db * yh).sum((0, 1)))
            return out
        x = h
    if kind in ("norm_linear", "linear"):
        if case.get("gelu"):
            x = x * (1 + torch.erf(x / math.sqrt(2.0))) / 2
        s = torch.clamp(torch.amax(x.abs(), -1), min=1e-12) / 127
        codes = torch.clamp(torch.round(x / s.unsqueeze(-1)), -127, 127)
        out = torch.matmul(codes, f["wq"].T) * s.unsqueeze(-1) * f["ws"]
        return [r, out] if kind == "norm_linear" else out
    K = x.shape[-1]
    kept = torch.empty_like(x)
    powers = torch.tensor([math.ldexp(1.0, k) for k in range(-126, 122)], dtype=torch.float64, device=x.device)
    for c in range(0, K, GROUP):
        v = x[..., c : c + GROUP]
        top = v.abs().amax(-1, keepdim=True)
        power = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))) + 1e-9) - 6
        step = powers[power.clamp(-126, 121).long() + 126]
        kept[..., c : c + GROUP] = torch.clamp(torch.round(v / step), -127, 127) * step
    if kind == "gelu_train":
        slope = (1 + torch.erf(kept / math.sqrt(2.0))) / 2 + kept * torch.exp(kept * kept / -2) / math.sqrt(2 * math.pi)
        return [x * (1 + torch.erf(x / math.sqrt(2.0))) / 2, f["dy"] * slope]
    rows = x.shape[0] * x.shape[1]
    low = torch.matmul(x.reshape(rows, K), f["a"].T).reshape(*x.shape[:2], -1)
    dt = f["dt"].reshape(rows, -1)
    return [low, torch.matmul(dt, f["a"]).reshape(x.shape), torch.matmul(dt.T, kept.reshape(rows, K))]
