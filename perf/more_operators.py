"""Rotary positions and sparse attention over selected blocks, as cases that a timing program can run.

`own` chooses between the plain form (elementary torch operations in 32 bits, in
64 for angles and for scores that are only compared, rounded once at the end)
and the framework's operators. `kind` says which:

  rotary        rotary_qk, no grad: q and k turned by position
  rotary_train  the same, forward and backward
  tables        rotary_tables: cos and sin of positions on one or more axes
  select        select_blocks: for each block of 64 queries the `count` blocks of
                64 keys with the largest product of mean query and mean key
  attend        sparse_attention over given blocks, no grad
  attend_train  the same, forward and backward
  sparse        select_blocks and sparse_attention after it, no grad

Sizes are the model's (16 heads of 128, one token per 16 x 16 pixels: 256 to
9216 tokens an image up to 1536 x 1536; batch 2 is classifier-free guidance's
two branches), an image of 2048 x 2048 (16384 tokens), or generic: shared key
heads, parts of a head, lengths that end inside a block.
"""

from __future__ import annotations

import math

import torch

own = False

BF = torch.bfloat16
HD = 128  # head_dim of the attention
BLOCK = 64  # queries, and keys, that are selected together


def listed():
    return [
        # One layer's queries and keys at 256 x 256, one branch: the smallest
        # call, where a launch's fixed cost weighs most.
        {"name": "rotary_256", "kind": "rotary", "B": 1, "S": 256, "H": 16, "Hk": 16, "hd": 128, "part": 128, "interleaved": False, "dtype": "bfloat16", "rows": 1},
        # ... of a guided step at 1536 x 1536.
        {"name": "rotary_1536", "kind": "rotary", "B": 2, "S": 9216, "H": 16, "Hk": 16, "hd": 128, "part": 128, "interleaved": False, "dtype": "bfloat16", "rows": 1},
        # Training with the other layout, a part of each head, shared key heads
        # and positions of each item's own; odd sizes.
        {"name": "rotary_train_part", "kind": "rotary_train", "B": 3, "S": 1001, "H": 12, "Hk": 4, "hd": 80, "part": 36, "interleaved": True, "dtype": "bfloat16", "rows": 3},
        # The tables of an image of 2048 x 2048: rows and columns stretched as
        # the model does it beyond its native size.
        {"name": "tables_2048", "kind": "tables", "rows": 16384, "dims": "44 42 42", "far": 128, "scale": 4.0, "scaling": "ntk"},
        # A text's positions far beyond the trained length.
        {"name": "tables_far", "kind": "tables", "rows": 131072, "dims": "128", "far": 1000000, "scale": 32.0, "scaling": "yarn"},
        # The selection alone, guided step at 1024 x 1024: a quarter of the blocks.
        {"name": "select_1024", "kind": "select", "B": 2, "Sq": 4096, "Sk": 4096, "H": 16, "Hk": 16, "count": 16, "lens": False},
        # One query against the keys of a 2048 x 2048 image.
        {"name": "attend_1", "kind": "attend", "B": 1, "Sq": 1, "Sk": 16384, "H": 16, "Hk": 16, "count": 32, "lens": False},
        # Selection and attention, guided step at 1024 x 1024.
        {"name": "sparse_1024", "kind": "sparse", "B": 2, "Sq": 4096, "Sk": 4096, "H": 16, "Hk": 16, "count": 16, "lens": False},
        # ... of an image of 2048 x 2048, an eighth of the blocks: the largest.
        {"name": "sparse_2048", "kind": "sparse", "B": 1, "Sq": 16384, "Sk": 16384, "H": 16, "Hk": 16, "count": 32, "lens": False},
        # LoRA training at 1024 x 1024.
        {"name": "attend_train_1024", "kind": "attend_train", "B": 1, "Sq": 4096, "Sk": 4096, "H": 16, "Hk": 16, "count": 16, "lens": False},
        # ... at 1536 x 1536, a sixth of the blocks.
        {"name": "attend_train_1536", "kind": "attend_train", "B": 1, "Sq": 9216, "Sk": 9216, "H": 16, "Hk": 16, "count": 24, "lens": False},
        # Training with shared key heads, keys that end inside a block at
        # another place for each item, and rows that attend nothing.
        {"name": "attend_train_ragged", "kind": "attend_train", "B": 2, "Sq": 1001, "Sk": 777, "H": 12, "Hk": 4, "count": 5, "lens": True},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def _dims(case):
    """Values of a head that turn with each axis."""
    return [int(d) for d in case["dims"].split()]


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 1e15)


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    kind = rng.choice(("rotary", "rotary_train", "tables", "select", "attend", "attend_train", "attend_train", "sparse", "sparse"))
    most["attend"] = most["sparse"]
    while True:
        c = {"kind": kind}
        if kind.startswith("rotary"):
            Hk = rng.choice((1, 2, 4, 8, 16))
            hd = 8 * rng.randint(4, 32)
            c |= {"B": rng.choice((1, 1, 2, 3)), "S": _log(rng, 1, 9216), "H": Hk * rng.choice((1, 1, 2, 3)), "Hk": Hk, "hd": hd}
            c |= {"part": hd if rng.random() < 0.5 else 2 * rng.randint(4, hd // 2), "interleaved": rng.random() < 0.5}
            c |= {"dtype": rng.choice(("bfloat16", "bfloat16", "float16", "float32")), "rows": rng.choice((1, c["B"]))}
        elif kind == "tables":
            dims = rng.choice(("128", "64", "44 42 42", "16 56 56", str(2 * rng.randint(2, 64))))
            c |= {"rows": _log(rng, 1, 131072), "dims": dims, "far": _log(rng, 16, 1000000)}
            c |= {"scale": round(math.exp(rng.uniform(0, math.log(32))), 3), "scaling": rng.choice(("ntk", "linear", "yarn"))}
        else:
            Hk = rng.choice((1, 2, 4, 8, 16))
            c |= {"B": rng.choice((1, 1, 2, 3)), "Sq": _log(rng, 1, 16384), "Sk": _log(rng, 16 if kind == "attend_train" else 1, 16384), "H": Hk * rng.choice((1, 1, 2, 4)), "Hk": Hk}
            c["count"] = _log(rng, 1, max(1, min(64, -(-c["Sk"] // BLOCK))))
            c["lens"] = rng.random() < 0.4
        if _cost(c) <= most[kind]:
            return c


# ------------------------------------------------------------------ inputs --


def _heads(g, B, S, H, drift):
    """Normed heads [B, S, H, HD] as they come to the attention: a direction that
    changes slowly along the sequence (`drift`: its values at every 256th token)
    and a token's own part, at RMS 1."""
    at = torch.arange(S, device="cuda") / 256
    low = at.long()
    t = (at - low)[:, None, None]
    x = drift[:, low, :H] * (1 - t) + drift[:, low + 1, :H] * t
    x = x + torch.randn(B, S, H, HD, generator=g, device="cuda")
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)).to(BF)


def _some_blocks(g, case, lens):
    """Lists as a selection gives them: more blocks near a query's own place in the
    sequence than far away, in ascending order, -1 where there are no more; with
    lengths, a first of several blocks of queries that has none."""
    B, H, nq, nk = case["B"], case["H"], -(-case["Sq"] // BLOCK), -(-case["Sk"] // BLOCK)
    rows, cols = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
    near = (rows[:, None] * (nk / nq) - cols).abs() / 4
    score = torch.rand(B, H, nq, nk, generator=g, device="cuda") - 0.2 * near.clamp_max(4)
    if lens is not None:
        score = score.masked_fill(cols * BLOCK >= lens[:, None, None, None], -math.inf)
        if nq > 1:
            score[:, :, 0] = -math.inf
    best, at = score.topk(min(case["count"], nk), -1)
    at = torch.where(best == -math.inf, nk, at).sort(-1)[0]
    out = torch.full((B, H, nq, case["count"]), -1, dtype=torch.int32, device="cuda")
    out[..., : at.shape[-1]] = torch.where(at == nk, -1, at)
    return out


def prepare(case, seed):
    """The case's tensors on the GPU, from the seed alone. Queries and keys have
    RMS 1, as after their norms; neighbouring tokens are alike, and queries are
    like the keys at their place. Values and gradients are N(0, 1)."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind = case["kind"]
    t = dict(case)
    if kind == "tables":
        t["positions"] = torch.randint(0, case["far"], (case["rows"], len(_dims(case))), generator=g, device="cuda")
        return t
    if kind.startswith("rotary"):
        B, S, hd, dtype = case["B"], case["S"], case["hd"], getattr(torch, case["dtype"])
        t["q"], t["k"] = n(B, S, case["H"], hd).to(dtype), n(B, S, case["Hk"], hd).to(dtype)
        angle = 6.3 * torch.rand(*(() if case["rows"] == 1 else (B,)), S, case["part"] // 2, generator=g, device="cuda")
        t["cos"], t["sin"] = angle.cos(), angle.sin()
        if kind == "rotary_train":
            t["q"].requires_grad_(True)
            t["k"].requires_grad_(True)
            t["dq"], t["dk"] = n(B, S, case["H"], hd).to(dtype), n(B, S, case["Hk"], hd).to(dtype)
        return t
    B, Sq, Sk, H, Hk = (case[k] for k in ("B", "Sq", "Sk", "H", "Hk"))
    drift = n(B, max(Sq, Sk) // 256 + 2, H, HD)
    t["q"], t["k"] = _heads(g, B, Sq, H, drift), _heads(g, B, Sk, Hk, 0.7 * drift[:, :, :: H // Hk] + 0.7 * n(1, 1, Hk, HD))
    # (With one key the attention has gradients of zero for queries and keys.)
    least = min(8, Sk) if kind == "attend_train" else 0
    t["lens"] = torch.randint(least, Sk + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if case["lens"] else None
    if kind != "select":
        t["v"] = n(B, Sk, Hk, HD).to(BF)
    if kind.startswith("attend"):
        t["blocks"] = _some_blocks(g, case, t["lens"])
    if kind == "attend_train":
        t["dout"] = n(B, Sq, H * HD).to(BF)
        for k in ("q", "k", "v"):
            t[k].requires_grad_(True)
    return t


# -------------------------------------------------------------- plain form --


def _frequencies(case):
    """(radians a position of each pair, its axis, factor of both tables)."""
    scale, freqs, axes, factor = case["scale"], [], [], 1.0
    for axis, d in enumerate(_dims(case)):
        i = torch.arange(d // 2, dtype=torch.float64, device="cuda")
        base = torch.tensor(10000.0 * (scale ** (d / (d - 2)) if case["scaling"] == "ntk" and d > 2 else 1.0), dtype=torch.float64, device="cuda")
        f = torch.exp(torch.log(base) * (-2 * i / d))
        if case["scaling"] == "linear":
            f = f / scale
        if case["scaling"] == "yarn":
            turns = ORIGINAL * f / (2 * math.pi)  # in the trained length
            keep = ((turns - 1) / 31).clamp(0, 1)
            f = f * (keep + (1 - keep) / scale)
            factor = 0.1 * math.log(scale) + 1
        freqs.append(f)
        axes.append(torch.full((d // 2,), axis, device="cuda"))
    return torch.cat(freqs), torch.cat(axes), factor


ORIGINAL = 4096  # trained length of the scaled tables


def _turn(x, cos, sin, t):
    """x with its first `part` values of each head turned, in 32 bits."""
    x = x.float()
    part = t["part"]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    head, rest = x[..., :part], x[..., part:]
    if t["interleaved"]:
        a, b = head.unflatten(-1, (-1, 2)).unbind(-1)
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = head.chunk(2, -1)
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1)


def _means(x, ends):
    """Mean of each block of rows of [B, S, H, HD] in 64 bits, [B, H, blocks, HD];
    rows at or past `ends` [B] do not count."""
    B, S, H, _ = x.shape
    there = torch.arange(S, device=x.device)[None, :, None, None] < ends[:, None, None, None]
    x = torch.where(there, x.double(), 0.0)
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -S % BLOCK)).unflatten(1, (-1, BLOCK)).sum(2)
    first = torch.arange(x.shape[1], device=x.device) * BLOCK
    rows = (ends[:, None] - first).clamp(1, BLOCK)
    return (x / rows[:, :, None, None]).transpose(1, 2)


def _ends(t):
    q, k = t["q"], t["k"]
    full = torch.full((q.shape[0],), k.shape[1], dtype=torch.int32, device=q.device)
    return full if t["lens"] is None else t["lens"].clamp(0, k.shape[1])


def _select(t):
    q, k, count = t["q"].detach(), t["k"].detach(), t["count"]
    ends = _ends(t)
    qm = _means(q, torch.full_like(ends, q.shape[1]))
    km = _means(k, ends).repeat_interleave(q.shape[2] // k.shape[2], 1)
    score = qm @ km.transpose(-1, -2).contiguous()
    nk = score.shape[-1]
    out = (torch.arange(nk, device=q.device) * BLOCK)[None] >= ends[:, None]
    score = score.masked_fill(out[:, None, None], -math.inf)
    best, at = score.sort(dim=-1, descending=True, stable=True)
    at = torch.where(best == -math.inf, nk, at)[..., :count].sort(-1)[0]
    at = torch.where(at == nk, -1, at).to(torch.int32)
    return torch.nn.functional.pad(at, (0, count - at.shape[-1]), value=-1)


def _attend(t, blocks):
    """Attention of each block of queries over its listed blocks of keys, in 32
    bits: out, and with a `dout` the gradients."""
    q, k, v = (t[x].detach().float() for x in ("q", "k", "v"))
    B, Sq, H, _ = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    nq, nk, count = blocks.shape[2], -(-Sk // BLOCK), blocks.shape[3]

    def cut(x, blocks_of):  # [B, H, blocks, BLOCK, HD]
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, blocks_of * BLOCK - x.shape[1]))
        return x.unflatten(1, (blocks_of, BLOCK)).permute(0, 3, 1, 2, 4)

    heads = torch.arange(H, device=q.device) // (H // Hk)
    index = (torch.arange(B, device=q.device)[:, None] * Hk + heads)[:, :, None, None] * nk + blocks.clamp_min(0)

    def listed_rows(x):  # [B, H, nq, count * BLOCK, HD]
        return cut(x, nk).reshape(B * Hk * nk, BLOCK, HD)[index.long()].flatten(3, 4)

    keys = blocks[..., None] * BLOCK + torch.arange(BLOCK, device=q.device)
    out = (blocks < 0)[..., None] | (keys >= _ends(t)[:, None, None, None, None])
    qb, kb, vb = cut(q, nq), listed_rows(k), listed_rows(v)
    out = out.flatten(3)[:, :, :, None]
    s = (qb @ kb.transpose(-1, -2).contiguous() * HD**-0.5).masked_fill(out, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = p @ vb

    def rows(x):  # back to [B, Sq, H, HD]
        return x.permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :Sq]

    outs = [rows(o).flatten(2).to(BF)]
    if t["kind"] == "attend_train":
        do = cut(t["dout"].float().unflatten(-1, (H, HD)), nq)
        ds = p * (do @ vb.transpose(-1, -2).contiguous() - (do * o).sum(-1, keepdim=True)) * HD**-0.5
        outs.append(rows(ds @ kb).to(BF))
        for per_key, by in ((ds, qb), (p, do)):
            got = torch.zeros(B * Hk * nk, BLOCK, HD, device=q.device)
            part = per_key.transpose(-1, -2).contiguous() @ by
            got.index_add_(0, index.flatten().long(), part.reshape(-1, BLOCK, HD))
            got = got.unflatten(0, (B, Hk, nk)).permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :Sk]
            outs.append(got.to(BF))
    return outs


def _plain(t):
    kind = t["kind"]
    if kind == "tables":
        f, axes, factor = _frequencies(t)
        angle = t["positions"].double()[:, axes] * f
        return [(angle.cos() * factor).float(), (angle.sin() * factor).float()]
    if kind.startswith("rotary"):
        outs = [_turn(t[x].detach(), t["cos"], t["sin"], t) for x in ("q", "k")]
        if kind == "rotary_train":
            outs += [_turn(t[x], t["cos"], -t["sin"], t) for x in ("dq", "dk")]
        return [o.to(t["q"].dtype) for o in outs]
    if kind == "select":
        return [_select(t)]
    if kind == "sparse":
        blocks = _select(t)
        return [blocks, *_attend(t, blocks)]
    return _attend(t, t["blocks"])


# ------------------------------------------------------------- the framework --


def _modules():
    import importlib

    import __graft_entry__

    __graft_entry__.load_package()
    return [importlib.import_module("anima_flat_amd.kernels." + m) for m in ("rotary", "sparse")]


_loaded = []


def _framework(t):
    if not _loaded:
        _loaded.extend(_modules())
    rotary, sparse = _loaded
    kind = t["kind"]
    if kind == "tables":
        return rotary.rotary_tables(t["positions"], _dims(t), scale=t["scale"], scaling=t["scaling"], original=ORIGINAL)
    if kind.startswith("rotary"):
        out = rotary.rotary_qk(t["q"], t["k"], t["cos"], t["sin"], interleaved=t["interleaved"])
        if kind == "rotary":
            return out
        return [o.detach() for o in out] + list(torch.autograd.grad(out, [t["q"], t["k"]], [t["dq"], t["dk"]]))
    if kind == "select":
        return [sparse.select_blocks(t["q"], t["k"], t["count"], t["lens"])]
    if kind == "sparse":
        blocks = sparse.select_blocks(t["q"], t["k"], t["count"], t["lens"])
        return [blocks, sparse.sparse_attention(t["q"], t["k"], t["v"], blocks, t["lens"])]
    out = sparse.sparse_attention(t["q"], t["k"], t["v"], t["blocks"], t["lens"])
    if kind == "attend":
        return [out]
    return [out.detach(), *torch.autograd.grad(out, [t["q"], t["k"], t["v"]], t["dout"])]


def run(state):
    return _framework(state) if own else _plain(state)


# -------------------------------------------------------------------- work --


def work(case):
    kind = case["kind"]
    if kind == "tables":
        pairs = case["rows"] * sum(_dims(case)) // 2
        return {"bytes": 8 * case["rows"] * len(_dims(case)) + 8 * pairs, "flops": 20 * pairs}
    if kind.startswith("rotary"):
        size = {"bfloat16": 2, "float16": 2, "float32": 4}[case["dtype"]]
        n = case["B"] * case["S"] * (case["H"] + case["Hk"]) * case["hd"]
        both = 2 if kind == "rotary_train" else 1
        tables = 4 * case["S"] * case["part"] * (case["B"] if case["rows"] > 1 else 1)
        return {"bytes": both * (2 * size * n + tables), "flops": both * 3 * n}
    B, Sq, Sk, H, Hk, count = (case[k] for k in ("B", "Sq", "Sk", "H", "Hk", "count"))
    nq, nk = -(-Sq // BLOCK), -(-Sk // BLOCK)
    lists, q, k = 4 * B * H * nq * count, 2 * B * Sq * H * HD, 2 * B * Sk * Hk * HD
    w = {"bytes": 0, "flops": 0}
    if kind in ("select", "sparse"):
        w["bytes"] += q + k + lists
        w["flops"] += B * (Sq * H + Sk * Hk) * HD + 2 * B * H * nq * nk * HD
    if kind != "select":
        # Of the keys and values, the blocks that the lists can reach.
        there = min(1.0, nq * (H // Hk) * count / nk)
        pairs = B * H * Sq * min(count * BLOCK, Sk)
        w["bytes"] += int(2 * q + 2 * there * k) + (lists if kind != "sparse" else 0)
        w["flops"] += 4 * pairs * HD
        if kind == "attend_train":
            w["bytes"] += int(2 * q + 2 * k)  # dout in, dq out, dk and dv out
            w["flops"] += 8 * pairs * HD
    return w


# ------------------------------------------------------------------- exact --


def exact(case, seed):
    t = prepare(case, seed)
    kind = case["kind"]
    if kind == "tables":
        cols = []
        for axis, d in enumerate(_dims(case)):
            pos = t["positions"][:, axis].double()
            for i in range(d // 2):
                theta, s, grow = 10000.0, case["scale"], 1.0
                if case["scaling"] == "ntk" and d > 2:
                    theta = theta * s ** (d / (d - 2))
                f = theta ** (-2.0 * i / d)
                if case["scaling"] == "linear":
                    f = f / s
                if case["scaling"] == "yarn":
                    part = min(1.0, max(0.0, (ORIGINAL / (2 * math.pi / f) - 1) / (32 - 1)))
                    f = (1 - part) * f / s + part * f
                    grow = 1 + math.log(s) / 10
                cols.append((torch.cos(pos * f) * grow, torch.sin(pos * f) * grow))
        return [torch.stack([c[j] for c in cols], -1) for j in (0, 1)]
    if kind.startswith("rotary"):
        part = case["part"]
        i = torch.arange(part // 2, device="cuda")
        lo, hi = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + part // 2)
        c, s = (t[k].double().reshape(-1, case["S"], 1, part // 2) for k in ("cos", "sin"))
        outs = []
        for name, sign in (("q", 1), ("k", 1), ("dq", -1), ("dk", -1))[: 2 if kind == "rotary" else 4]:
            x = t[name].detach().double()
            y = x.clone()
            z = torch.complex(x[..., lo], x[..., hi]) * torch.complex(c, sign * s)
            y[..., lo], y[..., hi] = z.real, z.imag
            outs.append(y)
        return outs
    B, Sq, Sk, H, Hk, count = (case[k] for k in ("B", "Sq", "Sk", "H", "Hk", "count"))
    nq, nk, group = -(-Sq // BLOCK), -(-Sk // BLOCK), H // Hk
    q, k = t["q"].detach().double(), t["k"].detach().double()
    ends = [Sk] * B if t["lens"] is None else t["lens"].tolist()
    outs = []
    if kind in ("select", "sparse"):
        blocks = torch.full((B, H, nq, count), -1, dtype=torch.int32, device="cuda")
        for b in range(B):
            have = -(-ends[b] // BLOCK)
            if not have:
                continue
            km = torch.stack([k[b, i * BLOCK : min((i + 1) * BLOCK, ends[b])].mean(0) for i in range(have)])
            qm = torch.stack([q[b, i * BLOCK : (i + 1) * BLOCK].mean(0) for i in range(nq)])
            for h in range(H):
                order = torch.argsort(-(qm[:, h] @ km[:, h // group].t().contiguous()), dim=1, stable=True)[:, :count]
                blocks[b, h, :, : order.shape[1]] = torch.sort(order, dim=1)[0].to(torch.int32)
        outs.append(blocks)
        if kind == "select":
            return outs
    else:
        blocks = t["blocks"]
    v = t["v"].detach().double()
    out = torch.zeros(B, Sq, H, HD, dtype=torch.float64, device="cuda")
    grads = [torch.zeros_like(out), torch.zeros_like(k), torch.zeros_like(v)] if kind == "attend_train" else []
    rows, cols = torch.arange(Sq, device="cuda") // BLOCK, torch.arange(Sk, device="cuda")
    for b in range(B):
        for h in range(H):
            hk = h // group
            chosen = torch.zeros(nq, nk + 1, dtype=torch.bool, device="cuda")
            chosen.scatter_(1, torch.where(blocks[b, h] < 0, nk, blocks[b, h]).long(), True)
            seen = chosen[rows][:, cols // BLOCK] & (cols < ends[b])
            e = torch.where(seen, q[b, :, h] @ k[b, :, hk].t().contiguous() / math.sqrt(HD), -math.inf)
            top = e.amax(1, keepdim=True)
            e = torch.exp(e - torch.where(top == -math.inf, 0.0, top))
            e = e / e.sum(1, keepdim=True).clamp_min(1e-300)
            out[b, :, h] = e @ v[b, :, hk]
            if grads:
                d = t["dout"].double().view(B, Sq, H, HD)[b, :, h]
                w = d @ v[b, :, hk].t().contiguous()
                w = e * (w - (e * w).sum(1, keepdim=True)) / math.sqrt(HD)
                grads[0][b, :, h] = w @ k[b, :, hk]
                grads[1][b, :, hk] += w.t().contiguous() @ q[b, :, h]
                grads[2][b, :, hk] += e.t().contiguous() @ d
    return [*outs, out.flatten(2), *grads]
