"""kernels.int8 against its oracle: codes bit for bit, the product to one rounding."""

from __future__ import annotations

import importlib

import pytest
import torch

from block_cases import BF, U16, U32, bf, gen, within
from oracle import block_oracle as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="session")
def int8(pkg):
    return importlib.import_module("anima_flat_amd.kernels.int8")


@pytest.mark.parametrize("B,S,K", [
    (1, 1, 8), (2, 33, 2048), (1, 9, 1000), (3, 5, 4096), (1, 7, 3000), (1, 5, 8192), (1, 3, 8184), (1, 4, 4104),
])
@pytest.mark.parametrize("spread", [False, True])
def test_rowquant_bit_exact(int8, B, S, K, spread):
    g = gen(B + S + K)
    x = torch.randn(B, S, K, generator=g)
    if spread:  # magnitudes over 2^-90 .. 2^60 from row to row, and 2^-8 .. 1 in a row
        x = x * torch.exp2(torch.randint(-90, 61, (B, S, 1), generator=g).float())
        x = x * torch.exp2(torch.randint(-8, 1, (B, S, K), generator=g).float())
    x = x.to(BF)
    x[0, 0, 1:] = 0
    x[-1, -1] = 0  # an all-zero token
    q, s = int8.rowquant_int8(x.cuda())
    eq, es = ref.int8_rows(x.float())
    assert q.shape == x.shape and s.shape == (B * S, 1)
    assert torch.equal(s[:, 0].cpu(), es)
    assert torch.equal(q.cpu(), eq.view_as(q))


def test_rowquant_ties(int8):
    """Every half step of codes, from both sides: 127 in the row makes the scale 1."""
    half = torch.arange(-126.5, 127, 1.0)
    vals = torch.cat([half, torch.arange(-127.0, 128)])
    x = torch.cat([vals, torch.full((-len(vals) % 8,), 127.0)])[None, None].to(BF)
    assert torch.equal(x.float().flatten()[: len(vals)], vals)
    q, s = int8.rowquant_int8(x.cuda())
    assert s.item() == 1.0
    assert torch.equal(q.cpu().float(), torch.round(x.float()))


def test_rowquant_gelu(int8):
    """GELU's float32 error (under 3.1e-5 with a few roundings, relative) moves the scale by as much and a code by
    one step where the quotient is that near a tie."""
    g = gen(3)
    x = bf(g, 2, 40, 1032, scale=3.0)
    q, s = int8.rowquant_int8(x, gelu=True)
    y = ref.gelu(x.double())
    want = y.abs().amax(-1, keepdim=True) / 127
    sd = s.view(2, 40, 1).double()
    assert ((sd - want).abs() <= 3.3e-5 * want).all()
    within(q.double() * sd, y, sd * (0.5 + 2e-5) + 3.3e-5 * y.abs(), "q s")


def test_rowquant_gelu_tails(int8):
    """Far negative values (GELU's tail, -0 at -inf) and rows of nothing else; +inf and NaN."""
    x = torch.linspace(-13, 13, 512, device="cuda").repeat(6, 1)
    x[0, ::7] = -float("inf")
    x[1] = -12.0
    x[2] = torch.linspace(-9.5, -6, 512)
    x[3, 5] = float("inf")
    x[4, 6] = float("nan")
    x = x.to(BF)[None]
    q, s = int8.rowquant_int8(x, gelu=True)
    assert torch.isnan(s[:, 0]).tolist() == [False, False, False, True, True, False]
    assert (q[0, [1, 3, 4]] == 0).all() and (q[0, 0, ::7] == 0).all()
    keep = [0, 1, 2, 5]
    y = ref.gelu(x.double().clamp(min=-1e3))[0, keep]  # the formula has 0 * inf at -inf
    want = y.abs().amax(-1, keepdim=True).clamp(min=1e-12) / 127
    sd = s[keep].double()
    assert ((sd - want).abs() <= 3.3e-5 * want).all()
    within(q[0, keep].double() * sd, y, sd * (0.5 + 2e-5) + 3.3e-5 * y.abs(), "q s")


def test_rowquant_not_finite(int8):
    x = bf(gen(4), 1, 5, 512)
    clean, cs = int8.rowquant_int8(x)
    x = x.clone()
    x[0, 1, 3], x[0, 3, 500] = float("inf"), float("nan")
    q, s = int8.rowquant_int8(x)
    assert torch.isnan(s[:, 0]).tolist() == [False, True, False, True, False]
    assert (q[0, [1, 3]] == 0).all() and torch.equal(q[0, [0, 2, 4]], clean[0, [0, 2, 4]])
    assert torch.equal(s[[0, 2, 4]], cs[[0, 2, 4]])
    w = torch.ones(16, 512, dtype=torch.int8, device="cuda")
    y = int8.int8_linear(q, s, w, torch.ones(16, device="cuda"))
    assert torch.isnan(y[0, [1, 3]]).all() and torch.isfinite(y[0, [0, 2, 4]]).all()


def test_quantize_weight(int8):
    w = bf(gen(5), 24, 272)
    q, s = int8.quantize_weight(w)
    eq, es = ref.int8_rows(w.float().cpu())
    assert torch.equal(q.cpu(), eq) and torch.equal(s.cpu(), es)


def _product(int8, M, K, N, seed, B=1, full=False):
    g = gen(seed)
    lo, hi = (-128, 128) if full else (-127, 128)
    q = torch.randint(lo, hi, (B, M // B, K), generator=g, dtype=torch.int8).cuda()
    w = torch.randint(lo, hi, (N, K), generator=g, dtype=torch.int8).cuda()
    s = (torch.rand(M, 1, generator=g) + 0.01).cuda()
    ws = (torch.rand(N, generator=g) + 0.01).cuda()
    return q, s, w, ws


def _check_product(q, s, w, ws, y):
    """The sum is exact; conversion, two products and the rounding to bf16 are the error."""
    want = (q.double().flatten(0, 1) @ w.double().t()) * s.double().view(-1, 1) * ws.double()
    within(y.flatten(0, 1), want, (U16 + 4 * U32) * want.abs(), "y")


# Few tokens (1 to 64: 16-token tiles and their edges), then tiles of 128 and 256 with rests in
# every direction; K below a stage, with rests of every parity of 16-byte chunks.
@pytest.mark.parametrize("M,K,N", [
    (1, 16, 8), (2, 2048, 6144), (3, 272, 24), (15, 64, 16), (16, 1024, 136), (17, 80, 40), (32, 4096, 64),
    (33, 2048, 2048), (63, 144, 8), (64, 8192, 72), (65, 16, 8), (66, 112, 136), (128, 128, 128), (129, 1040, 264),
    (200, 144, 128), (256, 256, 256), (257, 2064, 520), (333, 1024, 4096), (1000, 2048, 2048), (2049, 528, 2056),
    (4096, 1152, 2048), (3952, 2048, 6144),
])
def test_product(int8, M, K, N):
    args = _product(int8, M, K, N, M + K + N)
    _check_product(*args, int8.int8_linear(*args))


# Whole rounds of the 256 x 256 tiles (256 of them on 256 CUs), partial ones in both directions,
# one to four stages of K with rests, and tokens left over for the small tiles.
@pytest.mark.parametrize("M,K,N", [
    (8192, 16, 2048), (8100, 112, 2040), (8192, 128, 2048), (8100, 144, 2040), (8192, 256, 2048), (8065, 400, 1800),
    (8192, 512, 2048), (18000, 528, 2040), (16385, 2048, 2048), (260, 1040, 65544),
    # Several tiles in turn, whole ones (whose stores the next tile's waits count) and partial ones.
    (16384, 272, 2048), (24576, 384, 2048), (33000, 400, 1000), (24576, 528, 2056),
])
def test_large_product(int8, M, K, N):
    args = _product(int8, M, K, N, M + K + N, full=True)
    _check_product(*args, int8.int8_linear(*args))


# 64 x 64 tiles with K split over the waves: one to five steps (some waves without any), rests of
# K, partial tiles both ways, one and two workgroups a CU; and rests of the large tiles.
@pytest.mark.parametrize("M,K,N", [
    (65, 16, 8), (65, 128, 64), (70, 144, 72), (128, 256, 128), (100, 400, 200), (333, 512, 520), (200, 640, 6144),
    (333, 4112, 2040), (666, 8192, 2048), (1000, 65536, 64), (8193, 512, 2048), (8192 + 100, 512, 2048),
])
def test_middle_product(int8, M, K, N):
    args = _product(int8, M, K, N, M + K + N, full=True)
    _check_product(*args, int8.int8_linear(*args))


def test_largest_sums(int8):
    """All codes at -128 or 127, K at its most: 65536 products of up to 2^14."""
    for M in (3, 130):
        q = torch.full((1, M, 65536), -128, dtype=torch.int8, device="cuda")
        w = torch.full((16, 65536), -128, dtype=torch.int8, device="cuda")
        w[1::2] = 127
        s, ws = torch.ones(M, 1, device="cuda"), torch.ones(16, device="cuda")
        _check_product(q, s, w, ws, int8.int8_linear(q, s, w, ws))


def test_layouts(int8):
    q, s, w, ws = _product(int8, 150, 160, 136, 8, B=2, full=True)
    want = int8.int8_linear(q, s, w, ws)
    _check_product(q, s, w, ws, want)

    def off(v):
        return torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v)

    def strided(v):
        return torch.stack((v, v), -1)[..., 0]

    for form in (off, strided):
        got = int8.int8_linear(form(q), form(s), form(w), form(ws))
        assert torch.equal(got, want)
    assert torch.equal(int8.int8_linear(q, s.view(2, 75), w, ws), want)


def test_rows_do_not_depend_on_their_neighbours(int8):
    """A token's outputs have the same bits in any batch: sums are exact, one epilogue."""
    q, s, w, ws = _product(int8, 300, 528, 264, 9)
    want = int8.int8_linear(q, s, w, ws)
    for a, b in ((0, 1), (5, 40), (17, 81), (100, 230)):
        assert torch.equal(int8.int8_linear(q[:, a:b], s[a:b], w, ws), want[:, a:b])


def test_no_tokens(int8):
    q, s = int8.rowquant_int8(torch.empty(2, 0, 64, dtype=BF, device="cuda"))
    assert q.shape == (2, 0, 64) and s.shape == (0, 1)
    y = int8.int8_linear(q, s, torch.ones(8, 64, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda"))
    assert y.shape == (2, 0, 8)
