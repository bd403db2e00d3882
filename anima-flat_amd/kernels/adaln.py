"""Norms, gate, residual and modulation around a block's sublayers on MI355X, opt-in.

What stands between two sublayers of the block (src/kernels/adaln.py:298-314 in the
reference, whose ops this module does not register: import `anima_flat_amd.kernels.adaln`
to use it; its ops live in the `anima_flat_amd::` namespace):

  residual_adaln       r = x + branch_scale * gate * norm(y); h = LayerNorm(r) * (1 + scale) + shift
  adaln                h = LayerNorm(x) * (1 + scale) + shift (in front of the first sublayer)
  residual_adaln_int8  residual_adaln with h as int8 codes and a scale per token, for
                       kernels.int8.int8_linear (inference; src/kernels/fp8.py:56-97 in int8)

One kernel forward (aa_adaln_fwd), one backward and, where the modulation or the norm's
weight is trained, a second that adds up its partial sums (aa_adaln_bwd). All arithmetic is
fp32; r and h are rounded to bf16 once each, and the norm is taken of the unrounded r.
Gradients are deterministic.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .. import _lib
from .common import _check, aligned, custom_op, refuse_captured_training
from .rope import _f32

MAX_D = 8192


def _mod_code(t: torch.Tensor) -> int:
    return 2 if t.dtype == torch.float32 else 0


def _mod_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else 0


def _check_arguments(x, y, gate, scale, shift, weight) -> None:
    tensors = [t for t in (x, y, gate, scale, shift, weight) if t is not None]
    if not x.is_meta:
        _check(*tensors)
    if any(t.device != x.device for t in tensors):
        raise ValueError("all tensors must be on one device")
    if x.ndim != 3 or x.shape[2] == 0:
        raise ValueError("x must be [B, S, D]")
    B, _, D = x.shape
    if D % 8 or D > MAX_D:
        raise ValueError(f"D must be a multiple of 8 and at most {MAX_D}")
    if y is not None and y.shape != x.shape:
        raise ValueError("y must have x's shape")
    if any(t is not None and t.dtype != torch.bfloat16 for t in (x, y)):
        raise ValueError("unsupported dtype of x or y: only bfloat16 is implemented")
    for name, t in (("gate", gate), ("scale", scale), ("shift", shift)):
        if t is None:
            continue
        if t.ndim != 2 or t.shape[1] != D or t.shape[0] not in (1, B):
            raise ValueError(f"{name} must be [B, D], [B, 1, D], [1, D] or [D]")
        if t.dtype not in (torch.bfloat16, torch.float32) or t.dtype != scale.dtype:
            raise ValueError(f"{name} must be bfloat16 or float32, as the other modulations")
    if weight is not None and (weight.shape != x.shape[2:] or weight.dtype not in (torch.bfloat16, torch.float32)):
        raise ValueError("weight must be [D], bfloat16 or float32")


def _readable(t: torch.Tensor | None) -> torch.Tensor | None:
    """Modulation rows that the kernels read in place, or a copy."""
    if t is None:
        return None
    unit = 16 // t.element_size()
    if t.stride(1) != 1 or (t.shape[0] > 1 and (t.stride(0) % unit or t.stride(0) < t.shape[1])):
        t = t.contiguous()
    return aligned(t)


def _forward(x, y, gate, scale, shift, weight, eps, branch_scale, want_stats, int8):
    _check_arguments(x, y, gate, scale, shift, weight)
    B, S, D = x.shape
    x, y = (None if t is None else aligned(t.contiguous()) for t in (x, y))
    gate, scale, shift = (_readable(t) for t in (gate, scale, shift))
    r = torch.empty_like(x) if y is not None else None
    h = q = qs = None
    if int8:
        q = torch.empty(B, S, D, dtype=torch.int8, device=x.device)
        qs = torch.empty(B * S, 1, dtype=torch.float32, device=x.device)
    else:
        h = torch.empty_like(x)
    stats = torch.empty(B * S if want_stats else 0, 4, dtype=torch.float32, device=x.device)
    w = None if weight is None else aligned(_f32(weight))
    a = _lib.AdalnArgs(
        x=x.data_ptr(), y=_lib.ptr(y), gate=_lib.ptr(gate), scale=scale.data_ptr(), shift=shift.data_ptr(),
        gate_stride=0 if gate is None else _mod_stride(gate), scale_stride=_mod_stride(scale),
        shift_stride=_mod_stride(shift), weight=_lib.ptr(w), r=_lib.ptr(r), h=_lib.ptr(h), q=_lib.ptr(q),
        q_scale=_lib.ptr(qs), stats=stats.data_ptr() if want_stats else None, B=B, S=S, D=D, eps=eps,
        branch_scale=branch_scale, dtype=_lib.dtype_code(x), mod_dtype=_mod_code(scale),
    )
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().aa_adaln_fwd(ctypes.byref(a), _lib.stream(x)), "adaln")
    return r, h, q, qs, stats


def _backward(dr, dh, x, y, gate, scale, weight, stats, shift_rows, branch_scale, mods):
    """(dx, dy, dgate, dscale, dshift, dweight); what is not computed has no elements."""
    _check_arguments(x, y, gate, scale, None, weight)
    B, S, D = x.shape
    for t in (dr, dh):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype or t.device != x.device):
            raise ValueError("gradients must have the outputs' shape, dtype and device")
    if stats.shape != (B * S, 4) or stats.dtype != torch.float32 or stats.device != x.device or not stats.is_contiguous():
        raise ValueError("stats must be those of the forward")
    if (y is None) != (gate is None) or shift_rows not in (1, B):
        raise ValueError("y and gate belong together, and shift has 1 or B rows")
    dr, dh, x, y = (None if t is None else aligned(t.contiguous()) for t in (dr, dh, x, y))
    gate, scale = _readable(gate), _readable(scale)
    dx = torch.empty_like(x)
    dy = torch.empty_like(x) if y is not None else x.new_empty(0)
    dgate, dscale, dshift, dweight = (x.new_empty(0) for _ in range(4))
    if mods:
        dscale, dshift = torch.empty_like(scale, memory_format=torch.contiguous_format), scale.new_empty(shift_rows, D)
        if y is not None:
            dgate = torch.empty_like(gate, memory_format=torch.contiguous_format)
        if weight is not None:
            dweight = torch.empty(D, dtype=torch.float32, device=x.device)
    out = dx, dy, dgate, dscale, dshift, dweight
    if x.numel() == 0:
        for t in out:
            t.zero_()
        return out
    w = None if weight is None else aligned(_f32(weight))

    def p(t):
        return t.data_ptr() if t.numel() else None

    a = _lib.AdalnBwdArgs(
        dr=_lib.ptr(dr), dh=_lib.ptr(dh), x=x.data_ptr(), y=_lib.ptr(y), gate=_lib.ptr(gate),
        scale=scale.data_ptr(), gate_stride=0 if gate is None else _mod_stride(gate),
        scale_stride=_mod_stride(scale), weight=_lib.ptr(w), stats=stats.data_ptr(), dx=dx.data_ptr(),
        dy=p(dy), dgate=p(dgate), dscale=p(dscale), dshift=p(dshift), dweight=p(dweight),
        gate_rows=1 if gate is None else gate.shape[0], scale_rows=scale.shape[0], shift_rows=shift_rows,
        B=B, S=S, D=D, branch_scale=branch_scale, dtype=_lib.dtype_code(x), mod_dtype=_mod_code(scale),
    )
    with torch.cuda.device(x.device):
        ws_bytes = _lib.lib().aa_adaln_bwd_workspace(B, S, D, int(mods))
        ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=x.device) if ws_bytes else None
        _lib.check(
            _lib.lib().aa_adaln_bwd(ctypes.byref(a), _lib.ptr(ws), ws_bytes, _lib.stream(x)), "adaln_bwd"
        )
    return out


# --------------------------------------------------------------------- ops --


@custom_op("anima_flat_amd::residual_adaln", mutates_args=())
def _residual_adaln(
    x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor,
    weight: Optional[torch.Tensor], eps: float, branch_scale: float, want_stats: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    r, h, _, _, stats = _forward(x, y, gate, scale, shift, weight, eps, branch_scale, want_stats, False)
    return r, h, stats


@_residual_adaln.register_fake
def _(x, y, gate, scale, shift, weight, eps, branch_scale, want_stats):
    _check_arguments(x, y, gate, scale, shift, weight)
    rows = x.shape[0] * x.shape[1] if want_stats else 0
    return x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty((rows, 4), dtype=torch.float32)


@custom_op("anima_flat_amd::adaln", mutates_args=())
def _adaln(
    x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, eps: float, want_stats: bool
) -> tuple[torch.Tensor, torch.Tensor]:
    _, h, _, _, stats = _forward(x, None, None, scale, shift, None, eps, 1.0, want_stats, False)
    return h, stats


@_adaln.register_fake
def _(x, scale, shift, eps, want_stats):
    _check_arguments(x, None, None, scale, shift, None)
    rows = x.shape[0] * x.shape[1] if want_stats else 0
    return x.new_empty(x.shape), x.new_empty((rows, 4), dtype=torch.float32)


@custom_op("anima_flat_amd::residual_adaln_int8", mutates_args=())
def _residual_adaln_int8(
    x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor,
    weight: Optional[torch.Tensor], eps: float, branch_scale: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    r, _, q, qs, _ = _forward(x, y, gate, scale, shift, weight, eps, branch_scale, False, True)
    return r, q, qs


@_residual_adaln_int8.register_fake
def _(x, y, gate, scale, shift, weight, eps, branch_scale):
    _check_arguments(x, y, gate, scale, shift, weight)
    rows = x.shape[0] * x.shape[1]
    return x.new_empty(x.shape), x.new_empty(x.shape, dtype=torch.int8), x.new_empty((rows, 1), dtype=torch.float32)


@custom_op("anima_flat_amd::adaln_bwd", mutates_args=())
def _adaln_bwd(
    dr: Optional[torch.Tensor], dh: Optional[torch.Tensor], x: torch.Tensor, y: Optional[torch.Tensor],
    gate: Optional[torch.Tensor], scale: torch.Tensor, weight: Optional[torch.Tensor], stats: torch.Tensor,
    shift_rows: int, branch_scale: float, mods: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _backward(dr, dh, x, y, gate, scale, weight, stats, shift_rows, branch_scale, mods)


@_adaln_bwd.register_fake
def _(dr, dh, x, y, gate, scale, weight, stats, shift_rows, branch_scale, mods):
    D = x.shape[2]
    return (
        x.new_empty(x.shape),
        x.new_empty(x.shape) if y is not None else x.new_empty(0),
        gate.new_empty(gate.shape) if mods and y is not None else x.new_empty(0),
        scale.new_empty(scale.shape) if mods else x.new_empty(0),
        scale.new_empty((shift_rows, D)) if mods else x.new_empty(0),
        x.new_empty(D, dtype=torch.float32) if mods and weight is not None else x.new_empty(0),
    )


def _residual_adaln_setup(ctx, inputs, output):
    refuse_captured_training("residual_adaln")
    x, y, gate, scale, shift, weight, _, ctx.branch_scale, want_stats = inputs
    if not want_stats:
        raise RuntimeError("residual_adaln: a call that needs gradients keeps its statistics (want_stats)")
    ctx.set_materialize_grads(False)
    ctx.mods = any(ctx.needs_input_grad[2:6])
    ctx.shift_rows = shift.shape[0]
    ctx.save_for_backward(x, y, gate, scale, weight, output[2])


def _residual_adaln_backward(ctx, dr, dh, _):
    x, y, gate, scale, weight, stats = ctx.saved_tensors
    if dr is None and dh is None:
        return (None,) * 9
    dx, dy, dgate, dscale, dshift, dweight = _adaln_bwd(
        dr, dh, x, y, gate, scale, weight, stats, ctx.shift_rows, ctx.branch_scale, ctx.mods
    )
    if not ctx.mods:
        return (dx, dy) + (None,) * 7
    dw = None if weight is None else dweight.to(weight.dtype)
    return dx, dy, dgate, dscale, dshift, dw, None, None, None


torch.library.register_autograd(
    "anima_flat_amd::residual_adaln", _residual_adaln_backward, setup_context=_residual_adaln_setup
)


def _adaln_setup(ctx, inputs, output):
    refuse_captured_training("adaln")
    x, scale, shift, _, want_stats = inputs
    if not want_stats:
        raise RuntimeError("adaln: a call that needs gradients keeps its statistics (want_stats)")
    ctx.set_materialize_grads(False)
    ctx.mods = any(ctx.needs_input_grad[1:3])
    ctx.shift_rows = shift.shape[0]
    ctx.save_for_backward(x, scale, output[1])


def _adaln_backward(ctx, dh, _):
    x, scale, stats = ctx.saved_tensors
    if dh is None:
        return (None,) * 5
    dx, _, _, dscale, dshift, _ = _adaln_bwd(
        None, dh, x, None, None, scale, None, stats, ctx.shift_rows, 1.0, ctx.mods
    )
    return (dx, dscale, dshift, None, None) if ctx.mods else (dx,) + (None,) * 4


torch.library.register_autograd("anima_flat_amd::adaln", _adaln_backward, setup_context=_adaln_setup)


# -------------------------------------------------------------- public API --
#
# Checks are made once: by the native kernels, which hand what they do not take to the ops'
# Python functions, and by these and the fakes through _check_arguments.


def _rows2(t: torch.Tensor) -> torch.Tensor:
    """A modulation `[B, 1, D]` or `[D]` as rows; anything else as it is, for the checks."""
    if t.ndim == 3 and t.shape[1] == 1:
        return t[:, 0]
    return t[None] if t.ndim == 1 else t


def _modulation(*mods: torch.Tensor) -> list[torch.Tensor]:
    """Modulations as rows of one dtype. (The callers leave out what is so already: in a small
    call this and _wants_grad would be a tenth of the host's time.)"""
    mods = [t if t.ndim == 2 else _rows2(t) for t in mods]
    if any(t.dtype != mods[0].dtype for t in mods):
        if any(t.dtype not in (torch.bfloat16, torch.float32) for t in mods):
            raise ValueError("gate, scale and shift must be bfloat16 or float32")
        mods = [t.float() for t in mods]
    return mods


def _wants_grad(x, y, gate, scale, shift, weight) -> bool:
    return torch.is_grad_enabled() and (
        x.requires_grad or y.requires_grad or gate.requires_grad or scale.requires_grad or shift.requires_grad
        or (weight is not None and weight.requires_grad)
    )


def residual_adaln(x, y, gate, scale, shift, weight=None, eps=1e-6, branch_scale=1.0):
    """Add a sublayer's gated output to the residual stream and norm the sum for the next one.

    Args:
        x: Residual stream `[B, S, D]`, bfloat16 (D a multiple of 8, at most 8192).
        y: The sublayer's output, x's shape.
        gate, scale, shift: Modulation, one row per batch item or one for all: `[B, D]`,
            `[B, 1, D]`, `[1, D]` or `[D]`, bfloat16 or float32 (mixed ones are widened).
            Views such as `mod.chunk(3, -1)` are read in place.
        weight: RMSNorm weight `[D]` of a norm on y in front of the gate, or None.
        eps: Epsilon of both norms.
        branch_scale: Constant factor of the gated branch.

    Returns:
        `(r, h)`: `r = x + branch_scale * gate * y` (y normed with `weight`) and
        `h = LayerNorm(r) * (1 + scale) + shift`, both bfloat16 `[B, S, D]`. Differentiable
        in every tensor, once (no second derivatives); in modulations and weight for at most
        65535 batch items.

    Raises:
        ValueError: If a tensor is not on CUDA, or its shape or dtype is not supported.
    """
    if not (gate.ndim == scale.ndim == shift.ndim == 2 and gate.dtype == scale.dtype == shift.dtype):
        gate, scale, shift = _modulation(gate, scale, shift)
    stats = _wants_grad(x, y, gate, scale, shift, weight)
    r, h, _ = _residual_adaln(x, y, gate, scale, shift, weight, eps, branch_scale, stats)
    return r, h


def adaln(x, scale, shift, eps=1e-6):
    """`LayerNorm(x) * (1 + scale) + shift`, arguments as for `residual_adaln`."""
    if not (scale.ndim == shift.ndim == 2 and scale.dtype == shift.dtype):
        scale, shift = _modulation(scale, shift)
    stats = torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or shift.requires_grad)
    return _adaln(x, scale, shift, eps, stats)[0]


def residual_adaln_int8(x, y, gate, scale, shift, weight=None, eps=1e-6, branch_scale=1.0):
    """`residual_adaln` with h as int8 tokens for `int8_linear`. Inference only (no autograd).

    Returns:
        `(r, q, s)`: r bfloat16, q int8 `[B, S, D]` and float32 scales `[B * S, 1]` with
        `h ~ q * s`, rounded from the fp32 h. A token with a value that is not finite has
        the scale NaN.
    """
    if not (gate.ndim == scale.ndim == shift.ndim == 2 and gate.dtype == scale.dtype == shift.dtype):
        gate, scale, shift = _modulation(gate, scale, shift)
    if _wants_grad(x, y, gate, scale, shift, weight):
        raise RuntimeError("residual_adaln_int8 has no backward: use residual_adaln for training")
    return _residual_adaln_int8(x, y, gate, scale, shift, weight, eps, branch_scale)
