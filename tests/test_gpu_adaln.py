"""kernels.adaln against its 64-bit oracle: values, gradients, layouts, streams, refusals."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import BF, U16, U32, bf, gen, norm_bounds, within
from oracle import block_oracle as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture(scope="session")
def adaln(pkg):
    return importlib.import_module("anima_flat_amd.kernels.adaln")


def _inputs(B, S, D, seed, bm=None, mod=torch.float32, post=False, big=8.0):
    """Residual rows with two large channels, one chunked modulation, an RMSNorm weight."""
    g = gen(seed)
    x = torch.randn(B, S, D, generator=g)
    x[..., :2] *= big
    t = {"x": x.to("cuda", BF), "y": bf(g, B, S, D)}
    m = (torch.randn(B if bm is None else bm, 3 * D, generator=g) * 0.3).to("cuda", mod)
    t["shift"], t["scale"], t["gate"] = m.chunk(3, -1)
    t["weight"] = (1 + 0.1 * torch.randn(D, generator=g)).cuda() if post else None
    return t


def _ref_inputs(t, grad=()):
    out = {k: None if v is None else v.detach().double() for k, v in t.items()}
    for k in grad:
        out[k].requires_grad_(True)
    return out


def _check_forward(t, r, h, branch_scale=1.0):
    p = ref.norm_parts(**_ref_inputs(t), eps=EPS, branch_scale=branch_scale)
    within(r, p["r"], U16 * p["r"].abs() + 48 * U32 * p["size"], "r")
    _, xh = norm_bounds(p)
    s, b = t["scale"].double()[:, None], t["shift"].double()[:, None]
    size = p["xh"].abs() * (1 + s.abs()) + b.abs()
    within(h, p["h"], U16 * p["h"].abs() + (1 + s.abs()) * xh + 4 * U32 * size, "h")
    return p


# Widths of every kernel form (1, 2, 4 units a lane, rows of one, two, four and eight waves)
# and their edges; row counts around a workgroup's, one token, many.
SHAPES = [
    (1, 1, 8), (2, 1, 504), (1, 5, 512), (3, 7, 520), (1, 33, 1024), (2, 9, 1032), (1, 300, 2048),
    (2, 130, 2040), (1, 3, 2056), (2, 17, 4096), (1, 6, 4104), (1, 9, 8192), (5, 1, 2048), (1, 5000, 256),
]


@pytest.mark.parametrize("B,S,D", SHAPES)
@pytest.mark.parametrize("post", [False, True])
def test_forward(adaln, B, S, D, post):
    t = _inputs(B, S, D, B * 1000 + S + D, mod=BF if (B + S) % 2 else torch.float32, post=post)
    r, h = adaln.residual_adaln(**t, eps=EPS)
    _check_forward(t, r, h)
    assert not r.requires_grad


@pytest.mark.parametrize("D", [256, 1544, 2048, 4096])
def test_branch_scale_and_one_row_for_all(adaln, D):
    t = _inputs(3, 40, D, D, bm=1)
    r, h = adaln.residual_adaln(**t, eps=EPS, branch_scale=-0.37)
    _check_forward(t, r, h, branch_scale=-0.37)


@pytest.mark.parametrize("B,S,D", [(1, 1, 8), (2, 65, 2048), (1, 9, 4104)])
def test_adaln_alone(adaln, B, S, D):
    t = _inputs(B, S, D, 5) | {"y": None, "gate": None}
    h = adaln.adaln(t["x"], t["scale"], t["shift"], eps=EPS)
    p = ref.norm_parts(**_ref_inputs(t), eps=EPS)
    _, xh = norm_bounds(p)
    s, b = t["scale"].double()[:, None], t["shift"].double()[:, None]
    within(h, p["h"], U16 * p["h"].abs() + (1 + s.abs()) * xh + 4 * U32 * (p["xh"].abs() * (1 + s.abs()) + b.abs()), "h")
    # The same function with a gate of zero.
    zero = torch.zeros(1, D, device="cuda")
    r, h0 = adaln.residual_adaln(t["x"], t["x"], zero, t["scale"], t["shift"], eps=EPS)
    assert torch.equal(r, t["x"]) and torch.equal(h0, h)


# ---------------------------------------------------------------- backward --


def _gradients(adaln, t, names, dr, dh, branch_scale=1.0):
    leaves = [t[k].detach().requires_grad_(True) for k in names]
    args = t | dict(zip(names, leaves))
    if t["y"] is None:
        out = (adaln.adaln(args["x"], args["scale"], args["shift"], eps=EPS),)
        seeds = [dh]
    else:
        out = adaln.residual_adaln(**args, eps=EPS, branch_scale=branch_scale)
        seeds = [dr, dh]
    used = [(o, s) for o, s in zip(out, seeds) if s is not None]
    return torch.autograd.grad([o for o, _ in used], leaves, [s for _, s in used])


def _check_gradients(t, names, got, dr, dh, branch_scale=1.0):
    """Against autograd of the oracle. A gradient's summands have at most three factors that
    are off by (44 + 94 cond) u each, of the row's largest size; sums over rows add a chain of
    at most 64 + rows / 256 additions."""
    o = _ref_inputs(t, names)
    p = ref.norm_parts(**o, eps=EPS, branch_scale=branch_scale)
    outs = [(p["r"], dr), (p["h"], dh)] if t["y"] is not None else [(p["h"], dh)]
    used = [(a, s.double()) for a, s in outs if s is not None]
    want = torch.autograd.grad([a for a, _ in used], [o[k] for k in names], [s for _, s in used], allow_unused=True)
    with torch.no_grad():
        cond, _ = norm_bounds(p)
        k = U32 * (3 * (44 + 94 * cond) + 8)
        zero = torch.zeros_like(p["r"])
        g0 = zero if dr is None else dr.double()
        g1 = zero if dh is None else dh.double()
        u = (g1 * (1 + o["scale"][:, None])).abs()
        xh, rstd = p["xh"].abs(), p["rstd"]
        d = g0.abs() + rstd * (u + u.mean(-1, keepdim=True) + xh * (u * xh).mean(-1, keepdim=True))
        rows = d.shape[0] * d.shape[1]
        chain = U32 * (64 + rows / 256)
        # What xh's part that grows with cond alone (47 u cond) puts in, as a multiple of k.
        part = 47 * U32 * cond / k
        d = d + part * rstd * ((u * xh).mean(-1, keepdim=True) + xh * u.mean(-1, keepdim=True))
        size = {"x": d, "scale": g1.abs() * (xh + part), "shift": g1.abs()}
        if t["y"] is not None:
            gate = (branch_scale * o["gate"])[:, None].abs()
            size["y"] = gate * d
            size["gate"] = abs(branch_scale) * p["n"].abs() * d
            if t["weight"] is not None:
                ry = (o["y"].pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
                yh = (o["y"] * ry).abs()
                v = gate * d * o["weight"].abs()
                size["y"] = ry * (v + yh * (v * yh).mean(-1, keepdim=True))
                size["weight"] = gate * d * yh
    for name, a, w in zip(names, got, want):
        if w is None:
            w = torch.zeros_like(o[name])
        if name in ("x", "y"):
            within(a, w, U16 * w.abs() + k * size[name], "d" + name)
            continue
        assert a.dtype == t[name].dtype and a.shape == t[name].shape
        e = (k + chain) * size[name]
        e = e.sum((0, 1)) if name == "weight" else e.sum(1) if t[name].shape[0] == e.shape[0] else e.sum((0, 1))[None]
        within(a, w, (U16 if a.dtype == BF else U32) * w.abs() + e, "d" + name)


@pytest.mark.parametrize("B,S,D", SHAPES)
@pytest.mark.parametrize("kind", ["frozen", "mods", "post", "post_frozen"])
def test_gradients(adaln, B, S, D, kind):
    post = kind.startswith("post")
    t = _inputs(B, S, D, 7 * B + S + D, bm=1 if S % 2 else B, mod=BF if D % 16 else torch.float32, post=post)
    names = ["x", "y"] if kind.endswith("frozen") else ["x", "y", "gate", "scale", "shift"] + ["weight"] * post
    g = gen(B + S + D)
    dr, dh = bf(g, B, S, D), bf(g, B, S, D)
    _check_gradients(t, names, _gradients(adaln, t, names, dr, dh), dr, dh)


def test_weight_in_bf16(adaln):
    """Widened for the kernel; its gradient comes back in bf16."""
    t = _inputs(2, 21, 264, 31, post=True)
    t["weight"] = t["weight"].to(BF)
    names = ["x", "y", "gate", "scale", "shift", "weight"]
    g = gen(32)
    dr, dh = bf(g, 2, 21, 264), bf(g, 2, 21, 264)
    _check_gradients(t, names, _gradients(adaln, t, names, dr, dh), dr, dh)


@pytest.mark.parametrize("which", ["r", "h"])
def test_one_output_used(adaln, which):
    """The gradient of the other output is None inside: it counts as zero."""
    t = _inputs(2, 37, 520, 3, post=True)
    names = ["x", "y", "gate", "scale", "shift", "weight"]
    g = bf(gen(9), 2, 37, 520)
    dr, dh = (g, None) if which == "r" else (None, g)
    _check_gradients(t, names, _gradients(adaln, t, names, dr, dh, 0.5), dr, dh, 0.5)


@pytest.mark.parametrize("mods", [False, True])
def test_adaln_alone_gradients(adaln, mods):
    t = _inputs(2, 33, 2048, 4, bm=1) | {"y": None, "gate": None}
    names = ["x", "scale", "shift"] if mods else ["x"]
    dh = bf(gen(5), 2, 33, 2048)
    _check_gradients(t, names, _gradients(adaln, t, names, None, dh), None, dh)


def test_modulation_rows_of_different_numbers(adaln):
    """gate per batch item, scale one for all, shift expanded from one (its gradient comes
    back per batch item, through the expand)."""
    t = _inputs(3, 20, 264, 6)
    t["scale"] = t["scale"][:1]
    t["shift"] = t["shift"][:1].expand(3, -1)
    names = ["x", "y", "gate", "scale", "shift"]
    g = gen(8)
    dr, dh = bf(g, 3, 20, 264), bf(g, 3, 20, 264)
    got = _gradients(adaln, t, names, dr, dh)
    assert got[3].shape == (1, 264) and got[4].shape == (3, 264)
    _check_gradients(t, names, got, dr, dh)


def test_gradients_against_differences(adaln):
    """Along random directions: the kernel's gradient against a central difference of the
    oracle's forward. The kernel's rounding adds at most 2^-8 sum |g d| (and its float32 error,
    a hundredth of that); the difference's own error is O(step^2)."""
    B, S, D = 2, 24, 256
    t = _inputs(B, S, D, 12, post=True, big=2.0)
    names = ["x", "y", "gate", "scale", "shift", "weight"]
    g = gen(13)
    dr, dh = bf(g, B, S, D), bf(g, B, S, D)
    got = _gradients(adaln, t, names, dr, dh)
    o = _ref_inputs(t)
    for name, grad in zip(names, got):
        way = torch.randn(grad.shape, generator=g).cuda().double()
        value = []
        for sign in (1, -1):
            r, h = ref.residual_adaln(**(o | {name: o[name] + sign * 1e-4 * way}), eps=EPS)
            value.append((r * dr.double()).sum() + (h * dh.double()).sum())
        slope = (value[0] - value[1]) / 2e-4
        bound = 1.01 * U16 * (grad.double() * way).abs().sum() + 1e-5
        assert (slope - (grad.double() * way).sum()).abs() <= bound, name


# ---------------------------------------------------------------- int8 form --


@pytest.mark.parametrize("B,S,D", [(1, 1, 8), (2, 9, 520), (1, 77, 2048), (2, 5, 4096), (1, 3, 8192), (3, 1000, 256)])
def test_int8(adaln, B, S, D):
    """Codes are those of the oracle's h but for values within the float32 error of a tie."""
    t = _inputs(B, S, D, D + S, mod=BF if S % 2 else torch.float32, post=S % 3 == 0)
    r, q, s = adaln.residual_adaln_int8(**t, eps=EPS)
    assert torch.equal(r, adaln.residual_adaln(**t, eps=EPS)[0])
    p = ref.norm_parts(**_ref_inputs(t), eps=EPS)
    _, xh = norm_bounds(p)
    sc, b = t["scale"].double()[:, None], t["shift"].double()[:, None]
    e = (1 + sc.abs()) * xh + 4 * U32 * (p["xh"].abs() * (1 + sc.abs()) + b.abs())
    want_s = p["h"].abs().amax(-1, keepdim=True) / 127
    sd = s.view(B, S, 1).double()
    assert ((sd - want_s).abs() <= e.amax(-1, keepdim=True) / 127 + 2 * U32 * want_s).all()
    assert q.dtype == torch.int8 and q.abs().max() <= 127
    within(q.double() * sd, p["h"], sd * (0.5 + 2e-5) + e, "q s")


# ----------------------------------------------------------- odd situations --


def test_not_finite(adaln):
    """Infinities and NaN stay in their tokens; an int8 token that holds one has the scale NaN."""
    t = _inputs(1, 6, 512, 20)
    clean = adaln.residual_adaln(**t, eps=EPS)
    t["x"] = t["x"].clone()
    t["x"][0, 1, 7] = float("nan")
    t["x"][0, 3, 9] = float("inf")
    t["y"] = t["y"].clone()
    t["y"][0, 4, 0] = float("-inf")
    r, h = adaln.residual_adaln(**t, eps=EPS)
    for i in range(6):
        if i in (1, 3, 4):
            assert torch.isnan(h[0, i]).all()
        else:
            assert torch.equal(h[0, i], clean[1][0, i]) and torch.equal(r[0, i], clean[0][0, i])
    _, q, s = adaln.residual_adaln_int8(**t, eps=EPS)
    assert torch.isnan(s[:, 0]).tolist() == [False, True, False, True, True, False]
    assert (q[0, [1, 3, 4]] == 0).all()


def test_constant_rows(adaln):
    """A row of equal values has variance 0: h is the shift."""
    t = _inputs(1, 3, 264, 21)
    t["x"] = torch.full_like(t["x"], 3.0)
    r, h = adaln.residual_adaln(**(t | {"gate": torch.zeros(1, 264, device="cuda")}), eps=EPS)
    assert torch.equal(r, t["x"])
    assert torch.equal(h, t["shift"].to(BF)[:, None].expand_as(h))


def test_layouts(adaln):
    """Strided, misaligned and transposed tensors give the bits of plain ones."""
    t = _inputs(2, 19, 264, 22, mod=BF)
    want = adaln.residual_adaln(**t, eps=EPS)
    plain = {k: v.contiguous() for k, v in t.items() if v is not None}

    def off(v):  # one element past a 16-byte boundary
        return torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v)

    forms = {
        "plain": lambda v: v,
        "misaligned": off,
        "last_dim": lambda v: torch.stack((v, v), -1)[..., 0],
        "transposed": lambda v: v.transpose(0, -1).contiguous().transpose(0, -1),
        "3-d modulation": lambda v: v[:, None] if v.ndim == 2 else v,
    }
    for name, form in forms.items():
        got = adaln.residual_adaln(**{k: form(v) for k, v in plain.items()}, eps=EPS)
        assert all(torch.equal(a, b) for a, b in zip(want, got)), name
    one = {k: v[:1] if v.ndim == 2 else v for k, v in plain.items()}
    flat = {k: v[0] if v.ndim == 2 else v for k, v in one.items()}
    assert all(torch.equal(a, b) for a, b in zip(adaln.residual_adaln(**one), adaln.residual_adaln(**flat)))


def test_mixed_modulation_types(adaln):
    t = _inputs(1, 9, 264, 23, mod=BF)
    want = adaln.residual_adaln(**{k: v.float() if v is not None and v.ndim == 2 else v for k, v in t.items()}, eps=EPS)
    got = adaln.residual_adaln(**(t | {"gate": t["gate"].float()}), eps=EPS)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_no_tokens(adaln):
    t = _inputs(2, 0, 264, 24, post=True)
    r, h = adaln.residual_adaln(**t)
    assert r.shape == h.shape == (2, 0, 264)
    assert adaln.residual_adaln_int8(**t)[1].shape == (2, 0, 264)
    names = ["x", "y", "gate", "scale", "shift", "weight"]
    none = torch.empty(2, 0, 264, dtype=BF, device="cuda")
    for name, g in zip(names, _gradients(adaln, t, names, none, none)):
        assert g.shape == t[name].shape and not g.any()


def test_repeatable(adaln):
    t = _inputs(2, 700, 1032, 25, bm=1, post=True)
    names = ["x", "y", "gate", "scale", "shift", "weight"]
    g = gen(26)
    dr, dh = bf(g, 2, 700, 1032), bf(g, 2, 700, 1032)
    first = _gradients(adaln, t, names, dr, dh)
    again = _gradients(adaln, t, names, dr, dh)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_batch_item_is_its_own(adaln):
    """Item b of a batch gives the bits of a call with it alone, forward and dx, dy."""
    t = _inputs(3, 41, 520, 27)
    g = gen(28)
    dr, dh = bf(g, 3, 41, 520), bf(g, 3, 41, 520)
    out, grads = adaln.residual_adaln(**t), _gradients(adaln, t, ["x", "y"], dr, dh)
    for b in range(3):
        one = {k: None if v is None else v[b : b + 1] for k, v in t.items()}
        got = adaln.residual_adaln(**one), _gradients(adaln, one, ["x", "y"], dr[b : b + 1], dh[b : b + 1])
        assert all(torch.equal(a[b : b + 1], c) for a, c in zip((*out, *grads), (*got[0], *got[1])))
