"""Activations kept in 8 bits for the backward pass on MI355X, opt-in.

LoRA training (src/lora.py:14-137 in the reference) without block checkpointing keeps, per
layer, the input of every adapted projection and the 4-times-wide input of the MLP's GELU.
These operators compute their result from the bf16 input and keep an 8-bit copy of it:

  gelu8        GELU; backward dx = dy * GELU'(kept x)
  lora_down8   t = x @ a.T (a LoRA adapter's first product); backward dx = dt @ a,
               da = dt.T @ kept x

A kept value is an int8 code times a power of two that 32 neighbouring channels share: at
most 2^-7 of the group's largest magnitude away, exact in bf16, 33/32 bytes. Groups with a
value that is not finite read back as NaN. Import `anima_flat_amd.kernels.ckpt8` to use it;
its ops live in the `anima_flat_amd::` namespace.
"""

from __future__ import annotations

import torch

from .. import _lib
from .common import _check, aligned, custom_op, refuse_captured_training

GROUP = 32
MAX_RANK = 64
MAX_K = 65536


# Checks are made once: by the native kernels, which hand what they do not take to the ops'
# Python functions, and by these and the fakes through _check_tokens and _check_adapter.


def _check_tokens(x: torch.Tensor) -> None:
    if not x.is_meta:
        _check(x)
    if x.ndim != 3 or x.shape[2] == 0:
        raise ValueError("x must be [B, S, K]")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"unsupported dtype {x.dtype}: only bfloat16 is implemented")
    if x.shape[2] % 8 or x.shape[2] > MAX_K:
        raise ValueError(f"K must be a multiple of 8 and at most {MAX_K}")


def _check_adapter(x: torch.Tensor, a: torch.Tensor) -> None:
    if not x.is_meta:
        _check(x, a)
    _check_tokens(x)
    if a.ndim != 2 or a.shape[1] != x.shape[2] or a.dtype != x.dtype or a.device != x.device:
        raise ValueError("a must be [R, K] of x's dtype and device")
    if a.shape[0] % 8 or not 0 < a.shape[0] <= MAX_RANK:
        raise ValueError(f"the rank must be a multiple of 8 and at most {MAX_RANK}")


def _groups(K: int) -> int:
    return -(-K // GROUP)


def _kept(x: torch.Tensor, keep: bool, exps_shape: tuple[int, int]) -> tuple[torch.Tensor, torch.Tensor]:
    rows = x.numel() // x.shape[-1] if keep else 0
    codes = torch.empty(rows, GROUP * _groups(x.shape[-1]), dtype=torch.int8, device=x.device)
    exps = torch.empty(exps_shape if keep else (0, 0), dtype=torch.uint8, device=x.device)
    return codes, exps


def _check_kept(g: torch.Tensor, codes: torch.Tensor, exps: torch.Tensor, K: int, exps_shape: tuple[int, int]) -> None:
    """The copy that the forward of [B, S, K] tokens made, for a gradient of [B, S, ...]."""
    rows = g.shape[0] * g.shape[1]
    for t, shape, dtype in ((codes, (rows, GROUP * _groups(K)), torch.int8), (exps, exps_shape, torch.uint8)):
        if t.shape != shape or t.dtype != dtype or t.device != g.device or not t.is_contiguous():
            raise ValueError("codes and exps must be those of the forward")


def _ptr(t: torch.Tensor):
    return t.data_ptr() if t.numel() else None


# -------------------------------------------------------------------- GELU --


@custom_op("anima_flat_amd::gelu8", mutates_args=())
def _gelu8(x: torch.Tensor, keep: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_tokens(x)
    B, S, K = x.shape
    x = aligned(x.contiguous())
    y = torch.empty_like(x)
    codes, exps = _kept(x, keep, (B * S, _groups(K)))
    with torch.cuda.device(x.device):
        _lib.check(
            _lib.lib().aa_gelu8_fwd(
                _ptr(x), _ptr(y), _ptr(codes), _ptr(exps), B * S, K, _lib.dtype_code(x), _lib.stream(x)
            ),
            "gelu8",
        )
    return y, codes, exps


@_gelu8.register_fake
def _(x, keep):
    _check_tokens(x)
    B, S, K = x.shape
    return x.new_empty(x.shape), *_kept(x, keep, (B * S, _groups(K)))


@custom_op("anima_flat_amd::gelu8_bwd", mutates_args=())
def _gelu8_bwd(dy: torch.Tensor, codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    _check_tokens(dy)
    B, S, K = dy.shape
    _check_kept(dy, codes, exps, K, (B * S, _groups(K)))
    dy = aligned(dy.contiguous())
    dx = torch.empty_like(dy)
    with torch.cuda.device(dy.device):
        _lib.check(
            _lib.lib().aa_gelu8_bwd(
                _ptr(dy), _ptr(codes), _ptr(exps), _ptr(dx), B * S, K, _lib.dtype_code(dy), _lib.stream(dy)
            ),
            "gelu8_bwd",
        )
    return dx


@_gelu8_bwd.register_fake
def _(dy, codes, exps):
    return torch.empty_like(dy, memory_format=torch.contiguous_format)


def _gelu8_setup(ctx, inputs, output):
    refuse_captured_training("gelu8")
    if not inputs[1]:
        raise RuntimeError("gelu8: a call that needs gradients keeps its input (keep)")
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(output[1], output[2])


def _gelu8_backward(ctx, dy, _, __):
    if dy is None:
        return None, None
    return _gelu8_bwd(dy, *ctx.saved_tensors), None


torch.library.register_autograd("anima_flat_amd::gelu8", _gelu8_backward, setup_context=_gelu8_setup)


# -------------------------------------------------------------------- LoRA --


@custom_op("anima_flat_amd::lora_down8", mutates_args=())
def _lora_down8(x: torch.Tensor, a: torch.Tensor, keep: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_adapter(x, a)
    B, S, K = x.shape
    R = a.shape[0]
    x, a = aligned(x.contiguous()), aligned(a.contiguous())
    t = x.new_empty((B, S, R))
    codes, exps = _kept(x, keep, (_groups(K), -(-B * S // 16) * 16))
    with torch.cuda.device(x.device):
        ws_bytes = _lib.lib().aa_lora8_fwd_workspace(B * S, K, R)
        ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=x.device) if ws_bytes else None
        _lib.check(
            _lib.lib().aa_lora8_fwd(
                _ptr(x), _ptr(a), _ptr(t), _ptr(codes), _ptr(exps), _lib.ptr(ws), ws_bytes, B * S, K, R,
                _lib.dtype_code(x), _lib.stream(x),
            ),
            "lora_down8",
        )
    return t, codes, exps


@_lora_down8.register_fake
def _(x, a, keep):
    _check_adapter(x, a)
    B, S, K = x.shape
    return x.new_empty((B, S, a.shape[0])), *_kept(x, keep, (_groups(K), -(-B * S // 16) * 16))


@custom_op("anima_flat_amd::lora_down8_bwd", mutates_args=())
def _lora_down8_bwd(
    dt: torch.Tensor, a: torch.Tensor, codes: torch.Tensor, exps: torch.Tensor, need_x: bool, need_a: bool
) -> tuple[torch.Tensor, torch.Tensor]:
    _check(dt, a)
    if dt.ndim != 3 or a.ndim != 2 or dt.shape[2] != a.shape[0] or any(t.dtype != torch.bfloat16 for t in (dt, a)):
        raise ValueError("dt must be bfloat16 [B, S, R] and a bfloat16 [R, K]")
    B, S, _ = dt.shape
    R, K = a.shape
    if need_a:
        _check_kept(dt, codes, exps, K, (_groups(K), -(-B * S // 16) * 16))
    dt, a = aligned(dt.contiguous()), aligned(a.contiguous())
    dx = dt.new_empty((B, S, K) if need_x else 0)
    da = dt.new_empty(a.shape if need_a else 0)
    if B * S == 0:
        return dx, da.zero_()
    with torch.cuda.device(dt.device):
        ws_bytes = _lib.lib().aa_lora8_bwd_workspace(B * S, K, R) if need_a else 0
        ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=dt.device) if ws_bytes else None
        _lib.check(
            _lib.lib().aa_lora8_bwd(
                dt.data_ptr(), a.data_ptr(), _ptr(codes), _ptr(exps), _ptr(dx), _ptr(da), _lib.ptr(ws), ws_bytes,
                B * S, K, R, _lib.dtype_code(dt), _lib.stream(dt),
            ),
            "lora_down8_bwd",
        )
    return dx, da


@_lora_down8_bwd.register_fake
def _(dt, a, codes, exps, need_x, need_a):
    B, S, _ = dt.shape
    return dt.new_empty((B, S, a.shape[1]) if need_x else 0), dt.new_empty(a.shape if need_a else 0)


def _lora_down8_setup(ctx, inputs, output):
    refuse_captured_training("lora_down8")
    _, a, keep = inputs
    if ctx.needs_input_grad[1] and not keep:
        raise RuntimeError("lora_down8: a call that needs a's gradient keeps its input (keep)")
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(a, output[1], output[2])


def _lora_down8_backward(ctx, dt, _, __):
    if dt is None:
        return None, None, None
    a, codes, exps = ctx.saved_tensors
    need_x, need_a = ctx.needs_input_grad[:2]
    dx, da = _lora_down8_bwd(dt, a, codes, exps, need_x, need_a)
    return dx if need_x else None, da if need_a else None, None


torch.library.register_autograd(
    "anima_flat_amd::lora_down8", _lora_down8_backward, setup_context=_lora_down8_setup
)


# -------------------------------------------------------------- public API --


def gelu8(x: torch.Tensor) -> torch.Tensor:
    """GELU (erf form) whose backward reads an 8-bit copy of its input.

    Args:
        x: `[B, S, K]` bfloat16 (K a multiple of 8, at most 65536).

    Returns:
        `GELU(x)`, bfloat16. Under autograd the graph keeps 33/32 bytes per value of x (a
        plain GELU keeps 2); without, nothing is kept.

    Raises:
        ValueError: If `x` is not on CUDA, or its shape or dtype is not supported.
    """
    return _gelu8(x, x.requires_grad and torch.is_grad_enabled())[0]


def lora_down8(x: torch.Tensor, a: torch.Tensor) -> torch.Tensor:
    """The first product of a LoRA adapter, `x @ a.T`, whose backward reads an 8-bit copy of x.

    Args:
        x: `[B, S, K]` bfloat16 (K a multiple of 8, at most 65536).
        a: `[R, K]` bfloat16 (R a multiple of 8, at most 64); cast a float32 adapter to x's
            dtype, its gradient then comes back through the cast.

    Returns:
        `[B, S, R]` bfloat16, accumulated in fp32 and rounded once. Under autograd the graph
        keeps 33/32 bytes per value of x where a requires grad, and nothing of x where not.

    Raises:
        ValueError: If a tensor is not on CUDA, or a shape or dtype is not supported.
    """
    return _lora_down8(x, a, a.requires_grad and torch.is_grad_enabled())[0]
