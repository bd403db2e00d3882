"""The attention over selected blocks in 64 bits, with bounds of its kernels' errors; shared by
its tests.

Bounds, per element. u = 2^-24 and w = 2^-8 are half a step of float32 and bfloat16, relative.
A score is a sum of 128 exact products in fp32: off by 132 u of its summands' sizes. Its
exponential adds 4 u (|s| + |m|) for the product and difference with the maximum and 2^-21 for
the instruction; together eps. The probability that weights V is rounded to bf16 once (w), so
    |out - o| <= sum_j p_j (w + eps) |v_j - o| / (1 - w - eps) + n u sum_j p_j |v_j| + w |o|
(the sum of the same rounded probabilities divides). The backward forms p from the
log-sum-exp, off by eps + n u + 2^-20 (1 + |lse|), rounds p and dz once each, and takes D from
the rounded out. dq takes (sum of dz) x (a mean of keys) off: as the exact dz sum to 0, that
adds the sum of their errors times what a mean can be, the largest block's.
"""

from __future__ import annotations

import math

import torch

U32 = 2.0**-24
U16 = 2.0**-8
BF = torch.bfloat16
B64 = 64


def heads(g, B, S, H, scale=1.0, device="cuda"):
    return (torch.randn(B, S, H, 128, generator=g) * scale).to(device, BF)


def ends_of(lens, B, Sk):
    return [Sk] * B if lens is None else [max(0, min(int(n), Sk)) for n in lens.tolist()]


def seen_by(blocks, lens, Sq, Sk):
    """bool [B, H, Sq, Sk]: the pairs that are attended."""
    B, H = blocks.shape[:2]
    nk = -(-Sk // B64)
    chosen = torch.zeros(B, H, blocks.shape[2], nk + 1, dtype=torch.bool, device=blocks.device)
    index = torch.where((blocks < 0) | (blocks >= nk), nk, blocks).long()
    chosen.scatter_(3, index, True)
    rows = torch.arange(Sq, device=blocks.device) // B64
    cols = torch.arange(Sk, device=blocks.device)
    end = torch.tensor(ends_of(lens, B, Sk), device=blocks.device)
    return chosen[:, :, rows][..., cols // B64] & (cols < end[:, None, None, None])


def selected(q, k, count, lens=None):
    """select_blocks in 64 bits."""
    q, k = q.double(), k.double()
    B, Sq, H, _ = q.shape
    Sk, Hk = k.shape[1:3]
    nq = -(-Sq // B64)
    out = torch.full((B, H, nq, count), -1, dtype=torch.int32)
    for b, end in enumerate(ends_of(lens, B, Sk)):
        have = -(-end // B64)
        for h in range(H):
            km = [k[b, i * B64 : min(i * B64 + B64, end), h // (H // Hk)].mean(0) for i in range(have)]
            for i in range(nq):
                qm = q[b, i * B64 : i * B64 + B64, h].mean(0)
                score = [(qm @ m).item() for m in km]
                best = sorted(range(have), key=lambda j: (not math.isnan(score[j]), -score[j], j))[:count]
                for n, j in enumerate(sorted(best)):
                    out[b, h, i, n] = j
    return out


def attend(q, k, v, blocks, lens=None, dout=None):
    """(out, lse, gradients) in float64 and their bounds, as dicts of [B, S, H, 128] (lse [B, H, Sq])."""
    B, Sq, H, _ = q.shape
    Sk, Hk = k.shape[1:3]
    group, scale, n = H // Hk, 1 / math.sqrt(128), Sk
    seen = seen_by(blocks, lens, Sq, Sk)
    ref = {"out": torch.zeros(B, Sq, H, 128, dtype=torch.float64, device=q.device), "lse": torch.zeros(B, H, Sq, dtype=torch.float64, device=q.device)}
    err = {name: torch.zeros_like(t) for name, t in ref.items()}
    if dout is not None:
        for name, like in (("dq", q), ("dk", k), ("dv", v)):
            ref[name] = torch.zeros(like.shape, dtype=torch.float64, device=q.device)
            err[name] = torch.zeros_like(ref[name])
    for b in range(B):
        for h in range(H):
            Q, K, V = (t.detach()[b, :, i].double() for t, i in ((q, h), (k, h // group), (v, h // group)))
            m = seen[b, h]
            # Rows that nothing may read hold anything.
            used = m.any(0)
            K, V = (torch.where(used[:, None], t, 0.0) for t in (K, V))
            s = torch.where(m, Q @ K.t().contiguous() * scale, -math.inf)
            top = s.amax(1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            e = torch.exp(s - top)
            total = e.sum(1, keepdim=True)
            p = torch.where(total > 0, e / total, 0.0)
            o = p @ V
            lse = torch.log(total[:, 0]) + top[:, 0]
            size = torch.where(m, Q.abs() @ K.abs().t().contiguous() * scale, 0.0)
            far = torch.where(m & torch.isfinite(s), s.abs(), 0.0)
            eps = 132 * U32 * size + 4 * U32 * (far + far.amax(1, keepdim=True)) + 2.0**-21
            gap = torch.stack([(p * (U16 + eps) * (V[:, d][None] - o[:, d : d + 1]).abs()).sum(1) for d in range(128)], 1)
            eo = gap / (1 - U16 - eps.amax(1, keepdim=True)) + n * U32 * (p @ V.abs())
            ref["out"][b, :, h], err["out"][b, :, h] = o, eo + U16 * (o.abs() + eo)
            el = eps.amax(1) + n * U32 + 2.0**-20 * (1 + torch.where(torch.isfinite(lse), lse.abs(), 0.0))
            ref["lse"][b, h], err["lse"][b, h] = lse, el
            if dout is None:
                continue
            dO = dout.detach().view(B, Sq, H, 128)[b, :, h].double()
            eta = 1.01 * (eps + el[:, None])
            x = dO @ V.t().contiguous() - (dO * o).sum(1, keepdim=True)
            ed = (dO.abs() * err["out"][b, :, h]).sum(1, keepdim=True) + 130 * U32 * (dO.abs() * o.abs()).sum(1, keepdim=True)
            ex = 132 * U32 * (dO.abs() @ V.abs().t().contiguous()) + ed
            z = p * x
            ez = 1.01 * (z.abs() * (eta + U16) + p * (1 + eta) * ex)
            hk = h // group
            for name, at, val, bad, by in (
                ("dq", h, z, ez, K), ("dk", hk, z.t().contiguous(), ez.t().contiguous(), Q),
                ("dv", hk, p.t().contiguous(), (p * (eta + U16)).t().contiguous(), dO),
            ):
                by_scale = 1.0 if name == "dv" else scale
                ref[name][b, :, at] += by_scale * (val @ by)
                bad = bad + max(Sq, Sk) * U32 * val.abs()
                err[name][b, :, at] += by_scale * (bad @ by.abs())
                if name == "dq" and Sk:
                    means = torch.stack([r.mean(0) for r in K[: ends_of(lens, B, Sk)[b] or 1].split(B64)])
                    err[name][b, :, at] += by_scale * 1.01 * bad.sum(1, keepdim=True) * means.abs().amax(0)
    for name in ("dq", "dk", "dv"):
        if name in ref:
            err[name] = 1.01 * err[name] + U16 * ref[name].abs()
    return ref, err


def random_blocks(g, B, H, Sq, Sk, count, lens=None, device="cuda"):
    """Ascending lists of different blocks with a key, -1 behind them."""
    nq, nk = -(-Sq // B64), -(-Sk // B64)
    out = torch.full((B, H, nq, count), -1, dtype=torch.int32)
    for b, end in enumerate(ends_of(lens, B, Sk)):
        have = -(-end // B64)
        for h in range(H):
            for i in range(nq):
                got = torch.randperm(have, generator=g)[:count].sort()[0]
                out[b, h, i, : len(got)] = got
    return out.to(device)
