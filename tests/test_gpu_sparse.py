"""Attention over selected blocks against its formula in 64 bits: values, gradients, lists,
lengths, views, special values."""

from __future__ import annotations

import importlib
import math

import pytest
import torch

from block_cases import gen, within
from conftest import REL_L2
from sparse_cases import BF, attend, heads, random_blocks, selected

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sp(pkg):
    return importlib.import_module("anima_flat_amd.kernels.sparse")


def _lens(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def _close(name, got, ref, err):
    within(got, ref, err, name)
    if ref.norm() > 0:
        assert (got.double() - ref).norm() <= REL_L2 * ref.norm(), name


def _check_forward(sp, q, k, v, blocks, lens=None):
    ref, err = attend(q, k, v, blocks, lens)
    out, lse = sp._sparse_fwd(q, k, v, blocks, lens, True)
    _close("out", out, ref["out"], err["out"])
    none = ref["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, none) and not out[none.transpose(1, 2)].any()
    within(torch.where(none, 0.0, lse), torch.where(none, 0.0, ref["lse"]), err["lse"], "lse")
    assert torch.equal(sp.sparse_attention(q, k, v, blocks, lens), out.flatten(2))


SIZES = [  # B, Sq, Sk, H, Hk, count, lengths
    (1, 1, 1, 1, 1, 1, None), (1, 64, 64, 2, 2, 1, None), (2, 65, 63, 2, 1, 3, None), (1, 130, 200, 3, 1, 2, None),
    (2, 100, 321, 4, 2, 6, [321, 130]), (3, 70, 150, 2, 2, 2, [0, 1, 97]), (1, 1, 1000, 4, 4, 9, None),
    (2, 33, 500, 6, 3, 8, [500, 448]), (1, 192, 640, 2, 2, 10, None), (1, 700, 96, 1, 1, 2, None), (2, 64, 129, 2, 2, 40, [-5, 999]),
]


@pytest.mark.parametrize("size", SIZES)
def test_forward(sp, size):
    B, Sq, Sk, H, Hk, count, lens = size
    g = gen(11)
    q, k, v = heads(g, B, Sq, H), heads(g, B, Sk, Hk), heads(g, B, Sk, Hk)
    lens = _lens(lens)
    _check_forward(sp, q, k, v, random_blocks(g, B, H, Sq, Sk, count, lens), lens)


# Lists of few blocks of keys, split over workgroups: tiles of three heads, and more words of
# tiles than a wave has lanes.
LONG = [(1, 4500, 150, 6, 2, 2, None), (1, 33000, 70, 8, 1, 1, [65]), (2, 40, 4000, 3, 3, 30, [4000, 900])]


@pytest.mark.parametrize("size", SIZES + LONG)
def test_gradients(sp, size):
    B, Sq, Sk, H, Hk, count, lens = size
    g = gen(12)
    q, k, v = (heads(g, B, s, h).requires_grad_(True) for s, h in ((Sq, H), (Sk, Hk), (Sk, Hk)))
    dout, lens = heads(g, B, Sq, H), _lens(lens)
    blocks = random_blocks(g, B, H, Sq, Sk, count, lens)
    got = torch.autograd.grad(sp.sparse_attention(q, k, v, blocks, lens), [q, k, v], dout.flatten(2))
    ref, err = attend(q, k, v, blocks, lens, dout)
    for name, t in zip(("dq", "dk", "dv"), got):
        assert t.is_contiguous() and t.dtype == BF
        # One key has gradients of zero for q and k: only the bound holds there.
        (_close if Sk > 1 else lambda n, a, r, e: within(a, r, e, n))(name, t, ref[name], err[name])
    again = torch.autograd.grad(sp.sparse_attention(q, k, v, blocks, lens), [q, k, v], dout.flatten(2))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("size", [(1, 100, 500, 4, 2, 3, None), (2, 70, 700, 2, 2, 9, [700, 130]), (1, 40, 9000, 2, 1, 70, None),
                                  (3, 7, 30, 2, 2, 1, None), (1, 33000, 150, 8, 4, 2, None)])
def test_gradients_of_keys_in_common(sp, size):
    """Keys of 8 times what differs between them: dq is what differs times dz, the rest cancels.
    Two roundings of it are left, of dz and of dq, half a step of 2^-8 at most each."""
    B, Sq, Sk, H, Hk, count, lens = size
    g = gen(31)
    q, v, dout = heads(g, B, Sq, H), heads(g, B, Sk, Hk), heads(g, B, Sq, H)
    k = (8 * heads(g, 1, 1, Hk).float() + heads(g, B, Sk, Hk).float()).to(BF)
    lens = _lens(lens)
    blocks = random_blocks(g, B, H, Sq, Sk, count, lens)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(sp.sparse_attention(q, k, v, blocks, lens), [q], dout.flatten(2))
    ref, _ = attend(q, k, v, blocks, lens, dout)
    assert (dq.double() - ref["dq"]).norm() <= 2 * 2.0**-8 * ref["dq"].norm()


@pytest.mark.parametrize("scale", [2.0**-80, 2.0**75])
@pytest.mark.parametrize("sk", [150, 1500])
def test_gradients_of_any_scale(sp, scale, sk):
    """dz whose squares leave the range of float32: the mean key falls back to the plain one, in
    split lists to none."""
    g = gen(32)
    q, k, v, dout = heads(g, 1, 70, 2), heads(g, 1, sk, 1), heads(g, 1, sk, 1), heads(g, 1, 70, 2) * scale
    blocks = random_blocks(g, 1, 2, 70, sk, 20)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(sp.sparse_attention(q, k, v, blocks), [q], dout.flatten(2))
    ref, err = attend(q, k, v, blocks, None, dout)
    _close("dq", dq, ref["dq"], err["dq"])


def test_gradients_by_differences(sp):
    """Along a direction: the loss, in 64 bits from the kernel's inputs, moves as the gradients
    say. A step of 2^-6 leaves a relative error of its square, (2^-6)^2 / 6 times third
    derivatives of order 1, and the gradients' own 5e-3."""
    g = gen(13)
    B, Sq, Sk, H, Hk = 1, 70, 200, 2, 1
    q, k, v = (heads(g, B, s, h).requires_grad_(True) for s, h in ((Sq, H), (Sk, Hk), (Sk, Hk)))
    dout = heads(g, B, Sq, H)
    blocks = random_blocks(g, B, H, Sq, Sk, 2)
    got = torch.autograd.grad(sp.sparse_attention(q, k, v, blocks), [q, k, v], dout.flatten(2))
    tensors = [t.detach().double() for t in (q, k, v)]
    for i, grad in enumerate(got):
        step = torch.randn(grad.shape, generator=g).cuda().double()
        loss = []
        for sign in (1, -1):
            moved = [t + sign * 2.0**-6 * step if i == j else t for j, t in enumerate(tensors)]
            loss.append((attend(*moved, blocks)[0]["out"] * dout.double()).sum())
        along = (loss[0] - loss[1]) / 2.0**-5
        size = (grad.double().square().sum() * 1.0).sqrt()  # of a direction of unit variance
        assert ((grad.double() * step).sum() - along).abs() < (5e-3 + 2.0**-10) * size, i


@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1, 1, None), (1, 130, 700, 2, 2, 3, None), (2, 70, 513, 4, 2, 4, [513, 65]),
                                  (3, 64, 300, 2, 1, 5, [0, 64, 299]), (1, 1, 4500, 3, 3, 7, None), (1, 65, 300, 1, 1, 9, None)])
def test_selection(sp, size):
    B, Sq, Sk, H, Hk, count, lens = size
    g = gen(14)
    q, k, lens = heads(g, B, Sq, H), heads(g, B, Sk, Hk), _lens(lens)
    got = sp.select_blocks(q, k, count, lens)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), selected(q.cpu(), k.cpu(), count, lens))


@pytest.mark.parametrize("blocks", [5, 64, 65, 300, 1100])
def test_selection_ties(sp, blocks):
    """Equal scores go to the lower block, in every form of the search; -0 is 0."""
    q = torch.ones(1, 64, 1, 128, dtype=BF, device="cuda")
    k = torch.zeros(1, 64 * blocks, 1, 128, dtype=BF, device="cuda")
    k[:, 64 : 128] = -0.0
    k[:, 64 * (blocks // 2) :: 64 * 7] = 1.0
    got = sp.select_blocks(q, k, 4)[0, 0, 0].tolist()
    one = list(range(blocks // 2, blocks, 7))[:4]
    assert got == sorted(one + [i for i in range(blocks) if i not in set(range(blocks // 2, blocks, 7))][: 4 - len(one)])
    assert sp.select_blocks(q, k * 0, 4)[0, 0, 0].tolist() == [0, 1, 2, 3]
    neg = sp.select_blocks(q, -k, 4)[0, 0, 0].tolist()
    zeros = [i for i in range(blocks) if i not in set(range(blocks // 2, blocks, 7))]
    assert neg == sorted((zeros + one)[:4]) if len(zeros) < 4 else neg == zeros[:4]


def test_selection_of_special_values(sp):
    """NaN before all others (it shows in the output), infinities by their sign; rows past the
    length are not read."""
    q = torch.ones(1, 64, 1, 128, dtype=BF, device="cuda")
    k = torch.zeros(1, 64 * 6, 1, 128, dtype=BF, device="cuda")
    k[0, 64 * 4 + 3, 0, 7] = math.nan
    k[0, 64 * 2 + 1, 0, 0] = math.inf
    k[0, 64 * 1 + 1, 0, 0] = -math.inf
    assert sp.select_blocks(q, k, 1).flatten().tolist() == [4]
    assert sp.select_blocks(q, k, 2).flatten().tolist() == [2, 4]
    assert sp.select_blocks(q, k, 5).flatten().tolist() == [0, 2, 3, 4, 5]
    assert sp.select_blocks(q, k, 3, _lens([64 * 4 + 3])).flatten().tolist() == [0, 2, 3]


def test_longest(sp):
    """4096 blocks: the search reads its scores from LDS, lists fill it."""
    g = gen(15)
    q = heads(g, 1, 66, 1)
    k = torch.randn(1, 262144, 1, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(BF)
    got = sp.select_blocks(q, k, 300)
    km = k.double().view(4096, 64, 128).mean(1)
    qm = torch.stack([q[0, :64, 0].double().mean(0), q[0, 64:, 0].double().mean(0)])
    want = (qm @ km.t().contiguous()).sort(dim=-1, descending=True, stable=True)[1][:, :300].sort(-1)[0]
    assert torch.equal(got[0, 0].long(), want)
    v = heads(g, 1, 1, 1).expand(1, 262144, 1, 128)
    out = sp.sparse_attention(q, k, v, torch.arange(4096, dtype=torch.int32, device="cuda").expand(1, 1, 2, 4096))
    assert torch.equal(out, v[:, :66, 0])  # an average of equal values
    with pytest.raises(ValueError, match="at most 262144"):
        sp.select_blocks(q, k[:, :1].expand(1, 262145, 1, 128), 1)


def test_lists_of_any_kind(sp):
    """Unsorted, repeated and impossible entries, and blocks past the length: the lists' sets."""
    g = gen(16)
    B, Sq, Sk, H = 2, 130, 600, 2
    q, k, v = heads(g, B, Sq, H), heads(g, B, Sk, H), heads(g, B, Sk, H)
    lens = _lens([600, 130])
    blocks = torch.randint(-3, 14, (B, H, 3, 12), generator=g, dtype=torch.int32)
    blocks[0, 0, 1] = -1
    blocks[0, 1, 2] = torch.tensor([2**31 - 1, -(2**31), 10, 4096, 9, 9, 9, 9, 9, 9, 9, 9], dtype=torch.int32)
    blocks = blocks.cuda()
    _check_forward(sp, q, k, v, blocks, lens)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    dout = heads(g, B, Sq, H)
    got = torch.autograd.grad(sp.sparse_attention(*leaves, blocks, lens), leaves, dout.flatten(2))
    ref, err = attend(q, k, v, blocks, lens, dout)
    for name, t in zip(("dq", "dk", "dv"), got):
        _close(name, t, ref[name], err[name])


def test_rows_past_the_length_are_not_read(sp):
    g = gen(17)
    B, Sq, Sk, H = 3, 64, 200, 2
    q, k, v = heads(g, B, Sq, H), heads(g, B, Sk, H), heads(g, B, Sk, H)
    lens = _lens([130, 5, 0])
    dirty = [t.clone() for t in (k, v)]
    for b, n in enumerate((130, 5, 0)):
        for t in dirty:
            t[b, n:] = math.nan
    blocks = random_blocks(g, B, H, Sq, Sk, 3, lens)
    assert torch.equal(sp.select_blocks(q, k, 3, lens), sp.select_blocks(q, dirty[0], 3, lens))
    dout = heads(g, B, Sq, H).flatten(2)
    results = []
    for kk, vv in ((k, v), dirty):
        leaves = [t.clone().requires_grad_(True) for t in (q, kk, vv)]
        out = sp.sparse_attention(*leaves, blocks, lens)
        results.append([out, *torch.autograd.grad(out, leaves, dout)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    for grad in results[0][2:]:
        for b, n in enumerate((130, 5, 0)):
            assert not grad[b, n:].any()


@pytest.mark.parametrize("sq", [64, 40000])
def test_special_values_stay_in_their_rows(sp, sq):
    """A NaN or infinite query spoils its own row, a NaN key the rows that list its block; sq:
    lists split over workgroups, and not."""
    g = gen(18)
    q, k, v = heads(g, 1, sq, 1), heads(g, 1, 320, 1), heads(g, 1, 320, 1)
    nq = -(-sq // 64)
    blocks = torch.tensor([0, 2, 3, 4], dtype=torch.int32, device="cuda").expand(1, 1, nq, 4).contiguous()
    clean = sp._sparse_fwd(q, k, v, blocks, None, True)
    bad = q.clone()
    bad[0, 3, 0, 5], bad[0, 17, 0, 9], bad[0, 40, 0] = math.nan, math.inf, -math.inf
    out, lse = sp._sparse_fwd(bad, k, v, blocks, None, True)
    rows = [i for i in range(sq) if i not in (3, 17, 40)]
    # Another row's NaN in a sum on the matrix pipe sends the row to a sum in plain arithmetic:
    # the same rounded probabilities but where two scores differ in their last bit.
    assert ((out[0, rows].double() - clean[0][0, rows].double()).abs() <= 2.0**-7 * clean[0][0, rows].double().abs() + 2.0**-12).all()
    assert ((lse[0, 0, rows] - clean[1][0, 0, rows]).abs() <= 2.0**-18 * (1 + clean[1][0, 0, rows].abs())).all()
    assert torch.isnan(out[0, 3]).all()
    kk = k.clone()
    kk[0, 70, 0, 0] = math.nan  # block 1: no list names it
    assert torch.equal(sp._sparse_fwd(q, kk, v, blocks, None, True)[0], clean[0])
    kk[0, 130, 0, 0] = math.nan
    assert torch.isnan(sp._sparse_fwd(q, kk, v, blocks, None, True)[0]).all()


def test_masked_by_infinite_keys(sp):
    """Keys that score -inf have no weight, wherever they stand; a list of nothing else gives 0."""
    g = gen(19)
    q, k, v = heads(g, 1, 64, 1), heads(g, 1, 256, 1), heads(g, 1, 256, 1)
    q[..., 0] = 1.0
    for bad in ([0], [0, 1], [1, 2], [3]):
        kk = k.clone()
        for b in bad:
            kk[0, 64 * b : 64 * b + 64, 0, 0] = -math.inf
        some = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 1, 1, 4)
        rest = torch.tensor([b for b in range(4) if b not in bad], dtype=torch.int32, device="cuda").view(1, 1, 1, -1)
        ref, err = attend(q, k, v, rest)
        _close("out", sp._sparse_fwd(q, kk, v, some, None, True)[0], ref["out"], err["out"])
        out, lse = sp._sparse_fwd(q, kk, v, torch.tensor(bad, dtype=torch.int32, device="cuda").view(1, 1, 1, -1), None, True)
        assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("big", [30.0, 1000.0])
def test_scores_of_any_size(sp, big):
    """Maxima that grow from block to block by more than exp can hold from the first one's."""
    g = gen(20)
    q, k, v = heads(g, 1, 128, 1), heads(g, 1, 640, 1), heads(g, 1, 640, 1)
    k = (k.float() * torch.linspace(0.1, big, 640, device="cuda")[None, :, None, None]).to(BF)
    blocks = torch.arange(10, dtype=torch.int32, device="cuda").expand(1, 1, 2, 10).contiguous()
    for kk, vv in ((k, v), (k.flip(1), v.flip(1))):
        ref, err = attend(q, kk, vv, blocks)  # a score of 10^4 has an fp32 error of its own
        within(sp._sparse_fwd(q, kk, vv, blocks, None, True)[0], ref["out"], err["out"], "out")


@pytest.mark.parametrize("form", ["fused", "head_major", "misaligned", "last_dim_strided", "expanded"])
def test_views(sp, form):
    g = gen(21)
    B, S, H = 2, 130, 2
    q, k, v = (heads(g, B, S, H) for _ in range(3))
    blocks = random_blocks(g, B, H, S, S, 2)
    if form == "fused":
        views = torch.cat((q, k, v), 2).chunk(3, 2)
    elif form == "head_major":
        views = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    elif form == "misaligned":
        views = [torch.empty(t.numel() + 4, dtype=BF, device="cuda")[4:].view(t.shape).copy_(t) for t in (q, k, v)]
    elif form == "last_dim_strided":
        views = [torch.stack((t, t), -1)[..., 0] for t in (q, k, v)]
    else:
        q, k, v = (t[:1].expand(B, S, H, 128) for t in (q, k, v))
        views = q, k, v
    wide = torch.stack((blocks, blocks), -1)[..., 0]
    base, seen = [t.contiguous() for t in (q, k, v)], []
    for tensors, lists in ((base, blocks), (views, wide)):
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        out = sp.sparse_attention(*leaves, lists)
        dout = torch.cos(torch.arange(out.numel(), device="cuda")).view(out.shape).to(BF)
        seen.append([sp.select_blocks(tensors[0], tensors[1], 2), out, *torch.autograd.grad(out, leaves, dout)])
    assert all(torch.equal(a, b) for a, b in zip(*seen))


def test_strides_of_single_elements(sp):
    """Dimensions of size 1 have strides that address nothing, and that contiguous() keeps."""
    q, k = heads(gen(24), 1, 1, 1), heads(gen(25), 1, 90, 1)
    odd = q.as_strided(q.shape, (3, 5, 7, 1))
    blocks = torch.tensor([0, 1], dtype=torch.int32, device="cuda").view(1, 1, 1, 2)
    assert torch.equal(sp.sparse_attention(odd, k, k, blocks), sp.sparse_attention(q, k, k, blocks))
    assert torch.equal(sp.select_blocks(odd, k, 1), sp.select_blocks(q, k, 1))


def test_every_block_is_the_dense_attention(pkg, sp):
    g = gen(22)
    q, k, v = heads(g, 2, 300, 3), heads(g, 2, 500, 3), heads(g, 2, 500, 3)
    every = sp.select_blocks(q, k, 8)
    assert torch.equal(every, torch.arange(8, dtype=torch.int32, device="cuda").expand(2, 3, 5, 8))
    a, b = sp.sparse_attention(q, k, v, every).double(), pkg.attention(q, k, v).double()
    ref, err = attend(q, k, v, every)
    assert ((a - b).abs() <= 2 * err["out"].flatten(2)).all()


def test_empty(sp):
    e = lambda *s: torch.empty(*s, dtype=BF, device="cuda", requires_grad=True)
    blocks = torch.zeros(2, 3, 0, 4, dtype=torch.int32, device="cuda")
    assert sp.select_blocks(e(2, 0, 3, 128), e(2, 5, 3, 128), 4).shape == (2, 3, 0, 4)
    q, k = e(2, 0, 3, 128), e(2, 5, 3, 128)
    out = sp.sparse_attention(q, k, k, blocks)
    assert out.shape == (2, 0, 384)
    assert not torch.autograd.grad(out, k, torch.ones_like(out))[0].any()
    q, k = torch.ones(2, 5, 3, 128, dtype=BF, device="cuda", requires_grad=True), e(2, 0, 3, 128)
    blocks = sp.select_blocks(q, k, 4)
    assert (blocks == -1).all() and blocks.shape == (2, 3, 1, 4)
    out = sp.sparse_attention(q, k, k, blocks)
    assert not out.any() and not torch.autograd.grad(out, q, torch.ones_like(out))[0].any()


def test_offsets_past_32_bits(sp):
    """Keys and values in a cache of 80 heads of 262144 tokens: 5.4 GB each."""
    g = gen(23)
    q = heads(g, 1, 64, 2)
    cache = [torch.empty(1, 262144, 80, 128, dtype=BF, device="cuda") for _ in range(2)]
    small = [heads(g, 1, 128, 2) for _ in range(2)]
    for big, t in zip(cache, small):
        big[:, :64, 78:], big[:, -64:, 78:] = t[:, :64], t[:, 64:]
    far = torch.tensor([0, 4095], dtype=torch.int32, device="cuda").expand(1, 2, 1, 2).contiguous()
    near = torch.tensor([0, 1], dtype=torch.int32, device="cuda").expand(1, 2, 1, 2).contiguous()
    results = []
    for k, v, blocks in ((*small, near), (cache[0][:, :, 78:], cache[1][:, :, 78:], far)):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = sp.sparse_attention(*leaves, blocks)
        dq, dk, dv = torch.autograd.grad(out, leaves, torch.ones_like(out))
        results.append([out, dq, *(torch.cat((t[:, :64], t[:, -64:]), 1) for t in (dk, dv))])
    assert all(torch.equal(a, b) for a, b in zip(*results))
