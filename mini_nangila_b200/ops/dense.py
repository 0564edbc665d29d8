"""Dense layers of a decoder on the tensor cores (sm_100a).

``linear`` is a matrix product with bias, activation and residual in its
epilogue; ``gated_linear`` computes both projections of a gated feed-forward
block, the activation and their product in one kernel.  Both have a backward
pass, a form for few rows (decoding) and one for 8-bit operands with scales
(``ops.norm.rms_norm_fp8`` and ``ops.norm.quantize_rows`` make those).

Calls run on the current stream of x's device, allocate from PyTorch's
allocator and can be captured into CUDA graphs.  Under ``torch.autocast`` 16-bit
operands are made as ``torch.nn.functional.linear`` makes them.  The extension
must be built, and tensors must be CUDA tensors: there is no PyTorch fallback.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .._ext import cuda

ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


class DenseError(RuntimeError):
    """A product gave up waiting for its own copies; its output is incomplete."""


def _autocast(*ts):
    """The tensors in autocast's type (8-bit operands and None stay)."""
    dt = torch.get_autocast_dtype("cuda")
    return [t if t is None or t.dtype == torch.float8_e4m3fn or not t.is_floating_point() else t.to(dt) for t in ts]


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        keep_z = activation != "none"
        y, z = cuda().linear_forward(x, weight, bias, residual, activation, None, None, None, keep_z)
        ctx.save_for_backward(x, weight, z)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dx, dw, db = cuda().linear_backward(dy, x, weight, z, ctx.activation, nx, nw, nb)
        return dx, dw, db, dy if nr else None, None


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation):
        h, g, u = cuda().gated_forward(x, w_gate, w_up, activation, None, None, None, None, True)
        ctx.save_for_backward(x, w_gate, w_up, g, u)
        ctx.activation = activation
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, g, u = ctx.saved_tensors
        nx, ng, nu = ctx.needs_input_grad[:3]
        dx, dg, du = cuda().gated_backward(dh, x, w_gate, w_up, g, u, ctx.activation, nx, ng or nu)
        return dx, dg if ng else None, du if nu else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
           residual: torch.Tensor | None = None, x_scale: torch.Tensor | None = None,
           w_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` with sums in fp32.

    * ``x``: [..., in_features], bfloat16 or float16; ``weight``: [out_features,
      in_features] and ``bias``: [out_features] of the same type;
    * ``residual``: the output's shape, of x's type or float32; the output has
      its type;
    * 8 bits: ``x`` and ``weight`` float8_e4m3fn with ``x_scale`` (one float32 a
      row of x) and ``w_scale`` (one an output feature); bias and output are of
      ``out_dtype`` (bfloat16 by default).  No gradient.
    * ``out_dtype`` may also be float32.

    The backward pass gives gradients to x, weight, bias and residual.  It
    keeps the sums before an activation in 24 bits, and rounds their gradient
    to x's type before the two products.
    """
    if torch.is_autocast_enabled("cuda"):
        x, weight, bias = _autocast(x, weight, bias)
        if residual is not None and residual.dtype != torch.float32 and x.dtype != torch.float8_e4m3fn:
            residual = residual.to(x.dtype)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        if x_scale is not None or w_scale is not None or x.dtype == torch.float8_e4m3fn:
            raise ValueError("linear: 8-bit operands have no gradient; call it under torch.no_grad()")
        if out_dtype is not None and out_dtype != (x.dtype if residual is None else residual.dtype):
            raise ValueError("linear: out_dtype is fixed by x and residual where gradients are needed")
        return _Linear.apply(x, weight, bias, residual, activation)
    return cuda().linear_forward(x, weight, bias, residual, activation, x_scale, w_scale, out_dtype, False)[0]


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, activation: str = "silu",
                 x_scale: torch.Tensor | None = None, gate_scale: torch.Tensor | None = None,
                 up_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``activation(x @ w_gate.T) * (x @ w_up.T)`` in one kernel.

    Types and 8-bit operands as in ``linear``: ``x_scale`` one float32 a row,
    ``gate_scale`` and ``up_scale`` one an output feature.  The backward pass
    keeps both projections in 24 bits and gives gradients to x and both
    weights.
    """
    if torch.is_autocast_enabled("cuda"):
        x, w_gate, w_up = _autocast(x, w_gate, w_up)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        if x_scale is not None or x.dtype == torch.float8_e4m3fn:
            raise ValueError("gated_linear: 8-bit operands have no gradient; call it under torch.no_grad()")
        if out_dtype is not None and out_dtype != x.dtype:
            raise ValueError("gated_linear: out_dtype is x's type where gradients are needed")
        return _Gated.apply(x, w_gate, w_up, activation)
    return cuda().gated_forward(x, w_gate, w_up, activation, x_scale, gate_scale, up_scale, out_dtype, False)[0]


def check(device: int | torch.device | None = None) -> None:
    """Raise ``DenseError`` if a product on ``device`` gave up a wait since the
    last check (waits end after 4 s); synchronises its current stream."""
    if device is None:
        device = torch.cuda.current_device()
    idx = device.index if isinstance(device, torch.device) else int(device)
    st = cuda().dense_status(torch.cuda.current_device() if idx is None else idx, True)
    if st[0] != 0:
        raise DenseError(f"dense product failed: device status {st}")
