"""Attention over selected blocks on MI355X, opt-in.

For images beyond the trained size, where attention over all pairs of tokens outgrows the rest
of the block: each block of 64 queries attends the blocks of 64 keys that a cheap score picks
for it (import `anima_flat_amd.kernels.sparse` to use it; its ops live in the
`anima_flat_amd::` namespace):

  select_blocks     for each block of queries the key blocks with the largest product of mean
                    query and mean key
  sparse_attention  attention over given lists of blocks, forward and backward
  tile_order        an order of an image's tokens in which 64 neighbours are 8 x 8 patches

The rest stands as for `attention`: bf16, head_dim 128, no causal mask, `[B, S, H, hd]` views
read in place. Keys and values may have fewer heads than queries, and each batch item its own
number of keys. Gradients are deterministic.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from .. import _lib
from ..attention import _prep
from .common import _check, custom_op, refuse_captured_training

BLOCK = 64
MAX_KEYS = 262144
MAX_COUNT = 4096
MAX_ROW_STRIDE = 1 << 24


def _check_heads(q, k, v, seqused_k, more=()) -> None:
    tensors = [t for t in (q, k, v, seqused_k, *more) if t is not None]
    if not q.is_meta:
        _check(*tensors)
    if any(t.device != q.device for t in tensors):
        raise ValueError("all tensors must be on one device")
    if q.ndim != 4 or k.ndim != 4 or (v is not None and v.shape != k.shape):
        raise ValueError("q must be [B, Sq, H, hd], k and v [B, Sk, Hk, hd]")
    if k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] or k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(
            f"q {tuple(q.shape)} and k {tuple(k.shape)} disagree on batch or head_dim, or q's heads are no multiple of k's"
        )
    if any(t is not None and t.dtype != torch.bfloat16 for t in (q, k, v)):
        raise ValueError("unsupported dtype: only bfloat16 is implemented")
    if q.shape[3] != 128:
        raise ValueError(f"head_dim {q.shape[3]} is not supported (128 only)")
    if k.shape[1] > MAX_KEYS:
        raise ValueError(f"at most {MAX_KEYS} keys")
    if seqused_k is not None and (
        seqused_k.shape != q.shape[:1] or seqused_k.dtype not in (torch.int32, torch.int64)
    ):
        raise ValueError(f"seqused_k must be [B]={q.shape[0]}, int32 or int64")


def _check_blocks(q, blocks) -> None:
    B, Sq, H, _ = q.shape
    if blocks.ndim != 4 or blocks.shape[:3] != (B, H, _blocks_of(Sq)) or not 1 <= blocks.shape[3] <= MAX_COUNT:
        raise ValueError(f"blocks must be [B, H, ceil(Sq / 64), count]={(B, H, _blocks_of(Sq))} + (1 to {MAX_COUNT},)")
    if blocks.dtype != torch.int32:
        raise ValueError("blocks must be int32")


def _blocks_of(rows: int) -> int:
    return -(-rows // BLOCK)


def _lengths(seqused_k):
    if seqused_k is None:
        return None
    if seqused_k.dtype != torch.int32:
        seqused_k = seqused_k.clamp(0, MAX_KEYS).to(torch.int32)
    return seqused_k.contiguous()


def _near(t: torch.Tensor) -> torch.Tensor:
    """`_prep`, and a copy where tokens are further apart than the backward's 32-bit row offsets
    reach."""
    t = _prep(t)
    return t if t.stride(1) < MAX_ROW_STRIDE else t.clone(memory_format=torch.contiguous_format)


def _workspace(nbytes: int, like: torch.Tensor):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


def _sizes(q, k, count) -> dict:
    return {"B": q.shape[0], "Sq": q.shape[1], "Sk": k.shape[1], "H": q.shape[2], "Hk": k.shape[2], "hd": q.shape[3], "count": count, "dtype": 0}


def _set_strides(args, **tensors) -> None:
    for name, t in tensors.items():
        setattr(args, name + "_stride", _lib.c_strides(_lib.bshd_strides(t)))


# --------------------------------------------------------------------- ops --


def _check_count(count) -> None:
    if not 1 <= count <= MAX_COUNT:
        raise ValueError(f"count must be 1 to {MAX_COUNT}")


@custom_op("anima_flat_amd::select_blocks", mutates_args=())
def _select_blocks(q: torch.Tensor, k: torch.Tensor, count: int, seqused_k: Optional[torch.Tensor]) -> torch.Tensor:
    _check_heads(q, k, None, seqused_k)
    _check_count(count)
    B, Sq, H, _ = q.shape
    blocks = torch.empty((B, H, _blocks_of(Sq), count), dtype=torch.int32, device=q.device)
    q, k, lengths = _prep(q), _prep(k), _lengths(seqused_k)
    a = _lib.BlockSelectArgs(
        q=q.data_ptr(), k=k.data_ptr(), seqused_k=_lib.ptr(lengths), blocks=blocks.data_ptr(), **_sizes(q, k, count)
    )
    _set_strides(a, q=q, k=k)
    with torch.cuda.device(q.device):
        n = _lib.lib().aa_block_select_workspace(B, Sq, k.shape[1], H, k.shape[2])
        ws = _workspace(n, q)
        _lib.check(_lib.lib().aa_block_select(ctypes.byref(a), _lib.ptr(ws), n, _lib.stream(q)), "select_blocks")
    return blocks


@_select_blocks.register_fake
def _(q, k, count, seqused_k):
    _check_heads(q, k, None, seqused_k)
    _check_count(count)
    return q.new_empty((q.shape[0], q.shape[2], _blocks_of(q.shape[1]), count), dtype=torch.int32)


@custom_op("anima_flat_amd::sparse_fwd", mutates_args=())
def _sparse_fwd(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, blocks: torch.Tensor, seqused_k: Optional[torch.Tensor],
    keep: bool,
) -> tuple[torch.Tensor, torch.Tensor]:
    _check_heads(q, k, v, seqused_k, (blocks,))
    _check_blocks(q, blocks)
    B, Sq, H, _ = q.shape
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Sq) if keep else 0, dtype=torch.float32, device=q.device)
    if out.numel() == 0:
        return out, lse
    q, k, v, lengths, blocks = _prep(q), _prep(k), _prep(v), _lengths(seqused_k), blocks.contiguous()
    a = _lib.SparseFwdArgs(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        lse=lse.data_ptr() if keep else None, seqused_k=_lib.ptr(lengths), blocks=blocks.data_ptr(), softmax_scale=1.0 / math.sqrt(q.shape[3]),
        **_sizes(q, k, blocks.shape[3]),
    )
    _set_strides(a, q=q, k=k, v=v, out=out)
    with torch.cuda.device(q.device):
        n = _lib.lib().aa_sparse_fwd_workspace(B, Sq, H, blocks.shape[3])
        ws = _workspace(n, q)
        _lib.check(_lib.lib().aa_sparse_fwd(ctypes.byref(a), _lib.ptr(ws), n, _lib.stream(q)), "sparse_attention")
    return out, lse


@_sparse_fwd.register_fake
def _(q, k, v, blocks, seqused_k, keep):
    _check_heads(q, k, v, seqused_k, (blocks,))
    _check_blocks(q, blocks)
    B, Sq, H, _ = q.shape
    return q.new_empty(q.shape), q.new_empty((B, H, Sq) if keep else (0,), dtype=torch.float32)


@custom_op("anima_flat_amd::sparse_bwd", mutates_args=())
def _sparse_bwd(
    dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
    blocks: torch.Tensor, seqused_k: Optional[torch.Tensor],
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_heads(q, k, v, seqused_k, (blocks, dout, out, lse))
    _check_blocks(q, blocks)
    B, Sq, H, _ = q.shape
    if any(t.shape != q.shape or t.dtype != q.dtype for t in (dout, out)):
        raise ValueError("dout and out must have q's shape and dtype")
    if lse.shape != (B, H, Sq) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be float32 [B, H, Sq]={(B, H, Sq)}")
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    if q.numel() == 0 or k.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    dout, q, k, v, out = _near(dout), _near(q), _prep(k), _prep(v), _prep(out)
    lse, lengths, blocks = lse.contiguous(), _lengths(seqused_k), blocks.contiguous()
    a = _lib.SparseBwdArgs(
        dout=dout.data_ptr(), q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        lse=lse.data_ptr(), seqused_k=_lib.ptr(lengths), blocks=blocks.data_ptr(), dq=dq.data_ptr(), dk=dk.data_ptr(), dv=dv.data_ptr(),
        softmax_scale=1.0 / math.sqrt(q.shape[3]), **_sizes(q, k, blocks.shape[3]),
    )
    _set_strides(a, dout=dout, q=q, k=k, v=v, out=out, dq=dq, dk=dk, dv=dv)
    with torch.cuda.device(q.device):
        n = _lib.lib().aa_sparse_bwd_workspace(B, Sq, k.shape[1], H, k.shape[2], blocks.shape[3])
        ws = _workspace(n, q)
        _lib.check(_lib.lib().aa_sparse_bwd(ctypes.byref(a), _lib.ptr(ws), n, _lib.stream(q)), "sparse_attention backward")
    return dq, dk, dv


@_sparse_bwd.register_fake
def _(dout, q, k, v, out, lse, blocks, seqused_k):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _sparse_setup(ctx, inputs, output):
    refuse_captured_training("sparse_attention")
    q, k, v, blocks, seqused_k, keep = inputs
    if not keep:
        raise RuntimeError("sparse_attention: a call that needs gradients keeps its statistics (keep)")
    out, lse = output
    ctx.mark_non_differentiable(lse)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(q, k, v, out, lse, blocks, seqused_k)


def _sparse_backward(ctx, dout, _):
    if dout is None:
        return (None,) * 6
    return *_sparse_bwd(dout, *ctx.saved_tensors), None, None, None


torch.library.register_autograd("anima_flat_amd::sparse_fwd", _sparse_backward, setup_context=_sparse_setup)


# -------------------------------------------------------------- public API --


def select_blocks(q, k, count, seqused_k=None):
    """For each block of 64 queries the `count` blocks of 64 keys that are most like it.

    The score of a pair of blocks is the product of the mean query and the mean key, formed in
    64 bits: equal scores go to the lower block, and a rounding does not decide. No gradient
    flows through the choice.

    Args:
        q: Queries, bfloat16 `[B, Sq, H, 128]`.
        k: Keys, bfloat16 `[B, Sk, Hk, 128]` (H a multiple of Hk; at most 262144 keys).
        count: Blocks of keys per block of queries, 1 to 4096.
        seqused_k: Number of keys of each batch item, int32 or int64 `[B]` (below 0 is 0, beyond Sk
            all of them), or None for all.

    Returns:
        int32 `[B, H, ceil(Sq / 64), count]`, each list in ascending order, -1 behind its
        blocks where fewer hold a key. Blocks with a NaN come before all others.

    Raises:
        ValueError: If a tensor is not on CUDA, or a shape, dtype or size is not supported.
    """
    return _select_blocks(q.detach(), k.detach(), count, seqused_k)


def sparse_attention(q, k, v, blocks, seqused_k=None):
    """Attention of each block of 64 queries over its listed blocks of 64 keys.

    Args:
        q: Queries, bfloat16 `[B, Sq, H, 128]`.
        k, v: Keys and values, bfloat16 `[B, Sk, Hk, 128]` (H a multiple of Hk; at most 262144
            keys, less than 2^24 values from one to the next). Rows at or past `seqused_k` are
            not read.
        blocks: int32 `[B, H, ceil(Sq / 64), count]`, as `select_blocks` gives them, or any
            other: in any order, a block named twice counts once, numbers that are no block
            with a key are passed over.
        seqused_k: Number of keys of each batch item, int32 or int64 `[B]` (below 0 is 0, beyond Sk
            all of them), or None for all.

    Returns:
        Attention output with heads merged, `[B, Sq, H * 128]`; 0 for queries whose list is
        empty. Differentiable in q, k and v, once.

    Raises:
        ValueError: If a tensor is not on CUDA, or a shape, dtype or size is not supported (blocks
            of queries beyond 33 million; with gradients B H ceil(Sq / 4096) + B Hk ceil(Sk / 64) / 4
            or B Hk ceil(Sk / 64) beyond 16 million).
    """
    keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _sparse_fwd(q, k, v, blocks, seqused_k, keep)[0].flatten(2)


def tile_order(h, w, device=None, tile=8):
    """An order of the `h x w` tokens of an image in which neighbours in the sequence are
    neighbours in the image: patches of `tile x tile` tokens, row by row, each row by row. The
    64 tokens of a block are then one patch (where h and w are multiples of 8), which is what
    a block's mean stands for best.

    Returns:
        `(order, back)`, int64 `[h * w]`: `x[:, order]` puts tokens that are row by row (and
        the rows of their rotary tables) in this order, `y[:, back]` puts them back.
    """
    y, x = torch.meshgrid(torch.arange(h, device=device), torch.arange(w, device=device), indexing="ij")
    place = ((y // tile * (-(-w // tile)) + x // tile) * tile + y % tile) * tile + x % tile
    order = place.flatten().argsort()
    return order, order.argsort()
