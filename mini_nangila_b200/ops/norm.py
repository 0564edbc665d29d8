"""Root-mean-square norm of rows (sm_100a): with the residual's addition, with
a backward pass, and with an output in 8 bits with one scale a row.

Sums and the norm are in fp32.  Rows may have up to 32768 elements.  Tensors
must be CUDA tensors and the extension must be built: there is no PyTorch
fallback.  Forward-mode derivatives and ``torch.jit.trace`` are refused with a
``NotImplementedError``.
"""
from __future__ import annotations

import torch

from .._ext import cuda


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *, residual: torch.Tensor | None = None,
             out_dtype: torch.dtype | None = None):
    """``s * rsqrt(mean(s^2) + eps) * weight`` over the last dimension.

    ``s`` is x, or ``x + residual`` rounded to the residual's type; with a
    residual the call returns ``(y, s)``, s being the stream that goes on.
    x: float32, bfloat16 or float16; residual and weight of x's type or
    float32; y has x's type, or a 16-bit ``out_dtype`` where x is float32.
    Gradients reach x, weight and residual, from either output.
    """
    out = cuda().rms_norm(x, weight, eps, residual, out_dtype)
    return out[0] if residual is None else out


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *, residual: torch.Tensor | None = None):
    """``rms_norm`` with its output in 8 bits: ``(codes, scale)``, or ``(codes,
    scale, s)`` with a residual.

    ``codes * scale[..., None]`` is the norm's output: scale (float32, one a
    row) is the row's largest magnitude / 448, at least 2^-126, and codes are
    float8_e4m3fn.  A row with a NaN is NaN, one with an infinity NaN there and
    0 beside it, as in ``rms_norm``.  No gradient.
    """
    return cuda().rms_norm_fp8(x, weight, eps, residual)


def quantize_rows(x: torch.Tensor):
    """``(codes, scale)`` of the rows of x as ``rms_norm_fp8`` makes them: the
    8-bit form of a weight [out_features, in_features] or of activations.  A NaN
    stays one in its place; an infinity makes ``codes * scale`` of its row NaN."""
    return cuda().rms_norm_fp8(x, None, 0.0, None)
