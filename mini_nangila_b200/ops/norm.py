"""Root-mean-square norm of rows (sm_100a): with the residual's addition, with
a backward pass, and with an output in 8 bits with one scale a row.

Sums and the norm are in fp32.  Rows may have up to 32768 elements.  Tensors
must be CUDA tensors and the extension must be built: there is no PyTorch
fallback.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .._ext import cuda


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y, _, stream = cuda().rms_norm_forward(x, weight, eps, residual, False)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if residual is None else stream, weight)
        ctx.eps, ctx.x_type, ctx.has_residual = eps, x.dtype, residual is not None
        return y if residual is None else (y, stream)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds=None):
        if dy is None and ds is None:
            return None, None, None, None
        s, weight = ctx.saved_tensors
        nx, nw, _, nr = ctx.needs_input_grad
        dx, dres, dw = cuda().rms_norm_backward(dy, ds, s, weight, ctx.eps, ctx.x_type, ctx.has_residual, nw)
        return dx if nx else None, dw, None, dres if nr else None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *, residual: torch.Tensor | None = None):
    """``s * rsqrt(mean(s^2) + eps) * weight`` over the last dimension.

    ``s`` is x, or ``x + residual`` rounded to the residual's type; with a
    residual the call returns ``(y, s)``, s being the stream that goes on.
    x: float32, bfloat16 or float16; residual and weight of x's type or
    float32; y has x's type.  Gradients reach x, weight and residual, from
    either output.
    """
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return _RMSNorm.apply(x, weight, float(eps), residual)
    y, _, stream = cuda().rms_norm_forward(x, weight, eps, residual, False)
    return y if residual is None else (y, stream)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *, residual: torch.Tensor | None = None):
    """``rms_norm`` with its output in 8 bits: ``(codes, scale)``, or ``(codes,
    scale, s)`` with a residual.

    ``codes * scale[..., None]`` is the norm's output: scale (float32, one a
    row) is the row's largest magnitude / 448, at least 2^-126, and codes are
    float8_e4m3fn.  A NaN stays one in its place; an infinity makes its row
    NaN.  No gradient.
    """
    y, scale, stream = cuda().rms_norm_forward(x.detach(), weight.detach(), eps,
                                               None if residual is None else residual.detach(), True)
    return (y, scale) if residual is None else (y, scale, stream)


def quantize_rows(x: torch.Tensor):
    """``(codes, scale)`` of the rows of x as ``rms_norm_fp8`` makes them: the
    8-bit form of a weight [out_features, in_features] or of activations."""
    y, scale, _ = cuda().rms_norm_forward(x.detach(), None, 0.0, None, True)
    return y, scale
