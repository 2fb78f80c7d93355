"""Dense products around the expert layer: activation(x w^T + bias) + residual in one kernel, with gradients.

The router's projection (FP32 logits out of BF16 rows), shared experts and the projections of an attention block: what a model keeps in
BF16 or FP16 beside the quantised experts.  Operands are read where they lie, whichever way a product needs them; sums are FP32.  CUDA
kernels of the library throughout; CPU tensors are refused, and tensors with tangents of forward mode.  The reference project has the
grouped quantised product alone.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _C
from .tokens import _differentiable, _own_signs, _refuse_tangents


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation, out_dtype, device_status):
        want_x, want_w, want_bias, _ = ctx.needs_input_grad[:4]
        keep = activation != "none" and (want_x or want_w or want_bias)
        d, slopes = _C.linear(x, w, bias, residual, activation, out_dtype, keep, device_status)
        ctx.save_for_backward(x if want_w else None, w if want_x else None, slopes)
        ctx.form = (x.dtype, want_bias, device_status)
        return d

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dd):
        dx = dw = db = None
        if any(ctx.needs_input_grad[:3]):
            rows = _own_signs(dd)
            rows = rows if rows.stride(-1) == 1 and rows.stride(0) >= rows.shape[1] else rows.contiguous()
            dx, dw, db = _C.linear_backward(rows, *ctx.saved_tensors, *ctx.form)
        return dx, dw, db, dd if ctx.needs_input_grad[3] else None, None, None, None


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, *,
           activation: str = "none", out_dtype: Optional[torch.dtype] = None, device_status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """activation(x w^T + bias) + residual, (M, N).

    ``x`` (M, K) and ``w`` (N, K) BF16 or FP16, of one type, contiguous along K, starting on 16 bytes and with row strides that are multiples
    of 8 elements; K a multiple of 8, M and N any.  ``bias`` (N,) of that type.  ``residual`` (M, N) and the result have
    ``out_dtype``: the operands' type, or float32.  ``activation``: none, relu, gelu, gelu_tanh or silu.  Sums, bias, activation and residual
    are FP32, rounded once.  ``device_status``: int32 on the device that receives bit 0 should a bounded wait in the kernels expire.

    Differentiable in x, w, bias and residual.  The backward pass keeps the activation's slope in 16 bits, off by 2^-15 at most and in the
    negative tails of gelu and silu by 2^-11 of itself, and rounds the gradient in front of the activation to the operands' type: the
    tensor cores take no wider operands.  An FP32 gradient that FP16 operands cannot hold is brought into their range by a power of two
    for the products, whose sums are multiplied by its inverse."""
    if _C._binding is not None and device_status is None and activation in _C.ACTIVATION_CODES and (out_dtype is None or out_dtype is torch.float32 or out_dtype is x.dtype):
        result = _C._binding.linear(x, w, bias, residual, _C.ACTIVATION_CODES[activation], 1 if out_dtype is torch.float32 else 0)
        if result is not None:
            return result
    _refuse_tangents(x, w, bias, residual)
    x, w, bias, residual = (_own_signs(t) for t in (x, w, bias, residual))
    if not _differentiable(x, w, bias, residual):
        return _C.linear(x, w, bias, residual, activation, out_dtype, device_status=device_status)[0]
    return _Linear.apply(x, w, bias, residual, activation, out_dtype, device_status)
