"""Rotary positions on MI355X, apart from any norm, opt-in.

`kernels.rope` turns the whole of each head in the half layout, fused with the QK-norm, by the
tables of an h x w grid. This module has the general forms (import
`anima_flat_amd.kernels.rotary` to use it; its ops live in the `anima_flat_amd::` namespace):

  rotary_tables  cos and sin of any positions on up to four axes, stretched for lengths
                 beyond the trained one (by NTK, linearly, or by YaRN's parts)
  rotary         one tensor of heads turned by such tables: pairs (i, i + part / 2) or
                 (2 i, 2 i + 1), the whole head or its first part
  rotary_qk      queries and keys in one launch, with different numbers of heads

Angles are formed in 64 bits (aa_rotary_tables), the turn in 32 (aa_rotary), rounded once to
the type of its input. The backward is the turn by minus the angles.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from .. import _lib
from .common import _check, aligned, custom_op, refuse_captured_training

MAX_HD = 512
MAX_AXES = 4
SCALINGS = {"ntk": 0, "linear": 1, "yarn": 2}
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


# ------------------------------------------------------------------ tables --


def _check_tables(positions, dims, theta, scale, scaling, original) -> None:
    if not positions.is_meta:
        _check(positions)
    if not 1 <= len(dims) <= MAX_AXES or len(theta) != len(dims) or len(scale) != len(dims):
        raise ValueError(f"dims must name 1 to {MAX_AXES} axes, theta and scale one value each")
    if any(d < 0 or d % 2 for d in dims) or not 2 <= sum(dims) <= MAX_HD:
        raise ValueError(f"dims must be even, 2 to {MAX_HD} together")
    if positions.ndim < 2 or positions.shape[-1] != len(dims):
        raise ValueError("positions must be [..., axes]")
    if positions.dtype not in _POSITIONS:
        raise ValueError("positions must be int32, int64, float32 or float64")
    if scaling not in SCALINGS.values():
        raise ValueError("unknown scaling")
    if not all(s >= 1 and s < float("inf") for s in scale) or not all(0 < t < float("inf") for t in theta):
        raise ValueError("scale must be at least 1 and theta positive")
    if scaling == SCALINGS["yarn"] and not 0 < original < float("inf"):
        raise ValueError("yarn needs the trained length: original")


@custom_op("anima_flat_amd::rotary_tables", mutates_args=())
def _rotary_tables(
    positions: torch.Tensor, dims: Sequence[int], theta: Sequence[float], scale: Sequence[float], scaling: int,
    original: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    _check_tables(positions, dims, theta, scale, scaling, original)
    positions = positions.contiguous()
    shape = (*positions.shape[:-1], sum(dims) // 2)
    cos, sin = (torch.empty(shape, dtype=torch.float32, device=positions.device) for _ in range(2))
    a = _lib.RotaryTablesArgs(
        positions=positions.data_ptr(), cos=cos.data_ptr(), sin=sin.data_ptr(),
        rows=positions.numel() // len(dims), axes=len(dims), original=original, scaling=scaling,
        position_type=_POSITIONS[positions.dtype],
    )
    for i, (d, t, s) in enumerate(zip(dims, theta, scale)):
        a.dims[i], a.theta[i], a.scale[i] = d, t, s
    with torch.cuda.device(positions.device):
        _lib.check(_lib.lib().aa_rotary_tables(ctypes.byref(a), _lib.stream(positions)), "rotary_tables")
    return cos, sin


@_rotary_tables.register_fake
def _(positions, dims, theta, scale, scaling, original):
    _check_tables(positions, dims, theta, scale, scaling, original)
    shape = (*positions.shape[:-1], sum(dims) // 2)
    return positions.new_empty(shape, dtype=torch.float32), positions.new_empty(shape, dtype=torch.float32)


# -------------------------------------------------------------------- turn --


def _check_turn(q, k, cos, sin) -> None:
    tensors = [t for t in (q, k, cos, sin) if t is not None]
    if not q.is_meta:
        _check(*tensors)
    if any(t.device != q.device for t in tensors):
        raise ValueError("all tensors must be on one device")
    if q.ndim != 4 or (k is not None and (k.ndim != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
        raise ValueError("q and k must be [B, S, H, hd] of one batch, length and head_dim")
    if q.dtype not in _DTYPES or (k is not None and k.dtype != q.dtype):
        raise ValueError("unsupported dtype: q and k must be bfloat16, float16 or float32, both the same")
    B, S, _, hd = q.shape
    if hd % 8 or not 8 <= hd <= MAX_HD:
        raise ValueError(f"head_dim must be a multiple of 8, at most {MAX_HD}")
    if cos.shape != sin.shape or cos.ndim not in (2, 3) or cos.shape[-2] != S or (cos.ndim == 3 and cos.shape[0] not in (1, B)):
        raise ValueError("cos and sin must be [S, part / 2] or [B, S, part / 2]")
    if not 2 <= 2 * cos.shape[-1] <= hd:
        raise ValueError("the tables turn 2 to head_dim values")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32")


def _ready(t: torch.Tensor) -> torch.Tensor:
    """A view the kernel reads in place (head-dim stride 1, the others and the address at 16
    bytes), or a copy."""
    unit = 16 // t.element_size()
    if t.stride(3) != 1 or any(s % unit for s in t.stride()[:3]):
        # (contiguous() keeps the strides of dimensions of size 1.)
        return t.clone(memory_format=torch.contiguous_format)
    return aligned(t)


def _turn(q, k, cos, sin, interleaved, inverse):
    _check_turn(q, k, cos, sin)
    B, S, H, hd = q.shape
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ko = torch.empty((0,) if k is None else k.shape, dtype=q.dtype, device=q.device)
    if qo.numel() + ko.numel() == 0:
        return qo, ko
    q, k = _ready(q), None if k is None else _ready(k)
    cos, sin = aligned(cos.contiguous()), aligned(sin.contiguous())
    a = _lib.RotaryArgs(
        q=q.data_ptr(), k=_lib.ptr(k), q_out=qo.data_ptr(), k_out=None if k is None else ko.data_ptr(),
        cos=cos.data_ptr(), sin=sin.data_ptr(), table_stride=cos.stride(0) if cos.ndim == 3 and cos.shape[0] > 1 else 0,
        B=B, S=S, H=H, Hk=0 if k is None else k.shape[2], hd=hd, part=2 * cos.shape[-1], interleaved=interleaved,
        inverse=inverse, dtype=_DTYPES[q.dtype],
    )
    for name, t in (("q_stride", q), ("k_stride", k), ("q_out_stride", qo), ("k_out_stride", None if k is None else ko)):
        if t is not None:
            setattr(a, name, _lib.c_strides(_lib.bshd_strides(t)))
    with torch.cuda.device(q.device):
        _lib.check(_lib.lib().aa_rotary(ctypes.byref(a), _lib.stream(q)), "rotary")
    return qo, ko


@custom_op("anima_flat_amd::rotary", mutates_args=())
def _rotary(
    q: torch.Tensor, k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, interleaved: bool, inverse: bool
) -> tuple[torch.Tensor, torch.Tensor]:
    return _turn(q, k, cos, sin, interleaved, inverse)


@_rotary.register_fake
def _(q, k, cos, sin, interleaved, inverse):
    _check_turn(q, k, cos, sin)
    return q.new_empty(q.shape), q.new_empty((0,) if k is None else k.shape)


def _rotary_setup(ctx, inputs, output):
    refuse_captured_training("rotary")
    _, k, cos, sin, ctx.interleaved, ctx.inverse = inputs
    if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
        raise RuntimeError("rotary: the tables have no gradient")
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(cos, sin)
    ctx.pair = k is not None


def _rotary_backward(ctx, dq, dk):
    cos, sin = ctx.saved_tensors
    if not ctx.pair:
        dk = None
    back = (cos, sin, ctx.interleaved, not ctx.inverse)
    if dq is None:
        if dk is not None:
            dk = _rotary(dk, None, *back)[0]
    else:
        dq, got = _rotary(dq, dk, *back)
        dk = None if dk is None else got
    return dq, dk, None, None, None, None


torch.library.register_autograd("anima_flat_amd::rotary", _rotary_backward, setup_context=_rotary_setup)


# -------------------------------------------------------------- public API --


def _per_axis(value, axes: int) -> list[float]:
    return [float(v) for v in value] if isinstance(value, (tuple, list)) else [float(value)] * axes


def rotary_tables(positions, dims, theta=10000.0, scale=1.0, scaling="ntk", original=None):
    """cos and sin of rotary positions, for `rotary`, `rotary_qk` or `qkv_norm_rope`.

    Pair i of the d values that turn with an axis has the angle `position * theta^(-2i/d)`,
    formed in 64 bits: positions up to 10^8 are told apart. `scale` stretches an axis to so
    many times the length it was trained on:

      "ntk"     theta grows to `theta * scale^(d / (d - 2))`, as the model's `rope_scale` does:
                the slowest pair is stretched by `scale`, the fastest not at all
      "linear"  every angle is divided by `scale`
      "yarn"    pairs that turn at most once in the trained length `original` are stretched,
                those that turn 32 times or more are not, a ramp between, and both tables are
                multiplied by `0.1 ln(scale) + 1` (arXiv 2309.00071; the largest scale, with
                several axes). The ramp is linear in the number of turns, as in the paper's
                section 3.2; a ramp in the pair's index between two rounded bounds, which
                other programs have under this name, has other angles on it

    Args:
        positions: `[..., axes]` int32, int64, float32 or float64, or, where `dims` is one
            number, `[...]`.
        dims: Values of a head that turn with each axis (even), one after the other: one
            number, or up to four (`(44, 42, 42)`: the model's time, height and width).
        theta: Base of the frequencies, one for all axes or one each.
        scale: At least 1, one for all axes or one each.
        scaling: "ntk", "linear" or "yarn".
        original: The trained length ("yarn" only).

    Returns:
        `(cos, sin)`, float32 `[..., sum(dims) / 2]`.

    Raises:
        ValueError: If `positions` is not on CUDA, or a shape, dtype or value is not supported.
    """
    if isinstance(dims, int):
        dims, positions = [dims], positions.unsqueeze(-1)
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {', '.join(SCALINGS)}")
    dims = list(dims)
    return _rotary_tables(
        positions, dims, _per_axis(theta, len(dims)), _per_axis(scale, len(dims)), SCALINGS[scaling],
        0.0 if original is None else float(original),
    )


def rotary_qk(q, k, cos, sin, interleaved=False):
    """Queries and keys turned by their positions, in one launch.

    Args:
        q: `[B, S, H, hd]` bfloat16, float16 or float32 (hd a multiple of 8, at most 512).
        k: `[B, S, Hk, hd]` of q's dtype; Hk may be another number of heads.
        cos, sin: float32 `[S, part / 2]`, or `[B, S, part / 2]` for positions of each batch
            item's own; the first `part` values of each head turn, the others are copied.
        interleaved: Pairs are (2i, 2i + 1) instead of (i, i + part / 2).

    Returns:
        `(q', k')`, contiguous, of the inputs' shapes and dtype: pair (a, b) becomes
        `(a cos - b sin, b cos + a sin)`, in fp32, rounded once. Differentiable in q and k
        (the backward turns by minus the angles). Strided views with head-dim stride 1 and
        other strides that are multiples of 16 bytes are read in place.

    Raises:
        ValueError: If a tensor is not on CUDA, or a shape or dtype is not supported.
        RuntimeError: If the tables require grad: they have none.
    """
    return _rotary(q, k, cos, sin, interleaved, False)


def rotary(x, cos, sin, interleaved=False):
    """`rotary_qk` of one tensor `[B, S, H, hd]`."""
    return _rotary(x, None, cos, sin, interleaved, False)[0]
