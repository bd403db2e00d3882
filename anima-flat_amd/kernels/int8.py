"""Int8 products with a scale per token and per output channel on MI355X, opt-in.

The block's projections with both operands in int8, beside the FP8 tokens of kernels.fp8
(the reference's FP8 path is src/kernels/fp8.py:41-53, 234-328). Inference only.

  rowquant_int8    tokens to int8 with a scale per token, optionally after GELU
  quantize_weight  an nn.Linear weight to int8 with a scale per output channel (once, at load)
  int8_linear      the product: bf16 out, sums exact in int32

Import `anima_flat_amd.kernels.int8` to use it; its ops live in the `anima_flat_amd::`
namespace. kernels.adaln.residual_adaln_int8 makes int8 tokens in the norm itself.
"""

from __future__ import annotations

import torch

from .. import _lib
from .common import _check, aligned, custom_op


# Checks are made once: by the native kernels, which hand what they do not take to the ops'
# Python functions, and by these and the fakes through _check_tokens and _check_product.


def _check_tokens(x: torch.Tensor) -> None:
    if not x.is_meta:
        _check(x)
    if x.ndim != 3:
        raise ValueError("x must be [B, S, K]")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"unsupported dtype {x.dtype}: only bfloat16 is implemented")


@custom_op("anima_flat_amd::rowquant_int8", mutates_args=())
def _rowquant_int8(x: torch.Tensor, gelu: bool) -> tuple[torch.Tensor, torch.Tensor]:
    _check_tokens(x)
    B, S, K = x.shape
    x = aligned(x.contiguous())
    q = torch.empty(B, S, K, dtype=torch.int8, device=x.device)
    s = torch.empty(B * S, 1, dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(
            _lib.lib().aa_rowquant_int8(
                x.data_ptr(), B * S, K, int(gelu), q.data_ptr(), s.data_ptr(), _lib.dtype_code(x), _lib.stream(x)
            ),
            "rowquant_int8",
        )
    return q, s


@_rowquant_int8.register_fake
def _(x, gelu):
    _check_tokens(x)
    B, S, _ = x.shape
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty((B * S, 1), dtype=torch.float32)


def rowquant_int8(x: torch.Tensor, gelu: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantize tokens to int8 with a scale per token, optionally applying GELU first.

    Args:
        x: Tokens, shape `[B, S, K]`, bfloat16 (K a multiple of 8, at most 8192).
        gelu: Apply GELU (erf form) before quantizing.

    Returns:
        `(q, s)`: int8 tokens `[B, S, K]`, `q = round(127 * y / m)` to nearest even with the
        token's `m = max(max|y|, 1e-12)`, and `s = m / 127` as float32 `[B * S, 1]`. A token with a
        value that is not finite has the scale NaN and codes 0.

    Raises:
        ValueError: If `x` is not on CUDA, or its dtype / K is not supported.
        RuntimeError: If `x` requires grad (there is no backward).
    """
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("rowquant_int8 has no backward")
    return _rowquant_int8(x, gelu)


def quantize_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """An nn.Linear weight `[N, K]` (bfloat16, K at most 8192) as int8 codes `[N, K]` and a
    float32 scale per output channel `[N]`, for `int8_linear`."""
    if weight.ndim != 2:
        raise ValueError("weight must be [N, K]")
    q, s = rowquant_int8(weight.detach()[None])
    return q[0], s[:, 0]


def _check_product(q, s, weight, weight_scale) -> None:
    if not q.is_meta:
        _check(q, s, weight, weight_scale)
    if q.ndim != 3 or q.dtype != torch.int8:
        raise ValueError("q must be int8 [B, S, K]")
    if weight.ndim != 2 or weight.dtype != torch.int8 or weight.shape[1] != q.shape[2]:
        raise ValueError("weight must be int8 [N, K]")
    if s.dtype != torch.float32 or s.numel() != q.shape[0] * q.shape[1]:
        raise ValueError("s must be float32 with one scale per token")
    if weight_scale.dtype != torch.float32 or weight_scale.numel() != weight.shape[0]:
        raise ValueError("weight_scale must be float32 with one scale per output channel")
    if any(t.device != q.device for t in (s, weight, weight_scale)):
        raise ValueError("all tensors must be on one device")


@custom_op("anima_flat_amd::int8_linear", mutates_args=())
def _int8_linear(
    q: torch.Tensor, s: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor
) -> torch.Tensor:
    _check_product(q, s, weight, weight_scale)
    B, S, K = q.shape
    N = weight.shape[0]
    q, weight = aligned(q.contiguous()), aligned(weight.contiguous())
    s, weight_scale = s.contiguous(), weight_scale.contiguous()
    y = torch.empty(B, S, N, dtype=torch.bfloat16, device=q.device)
    with torch.cuda.device(q.device):
        _lib.check(
            _lib.lib().aa_int8_linear(
                q.data_ptr(), s.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(), y.data_ptr(),
                B * S, N, K, _lib.dtype_code(y), _lib.stream(q),
            ),
            "int8_linear",
        )
    return y


@_int8_linear.register_fake
def _(q, s, weight, weight_scale):
    _check_product(q, s, weight, weight_scale)
    return q.new_empty((q.shape[0], q.shape[1], weight.shape[0]), dtype=torch.bfloat16)


def int8_linear(
    q: torch.Tensor, s: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor
) -> torch.Tensor:
    """`(q * s) @ (weight * weight_scale[:, None]).T` with the sums in int32. Inference only.

    Args:
        q: int8 tokens `[B, S, K]` (K a multiple of 16, at most 65536).
        s: Their scales, float32, `[B * S, 1]` (as `rowquant_int8` gives them) or any shape
            of B * S elements.
        weight: int8 `[N, K]` (N a multiple of 8).
        weight_scale: float32 `[N]`.

    Returns:
        bfloat16 `[B, S, N]`: the int32 sum converted to fp32, times both scales, rounded once.

    Raises:
        ValueError: If a tensor is not on CUDA, or a shape or dtype is not supported.
    """
    if (s.requires_grad or weight_scale.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("int8_linear has no backward")
    return _int8_linear(q, s, weight, weight_scale)
