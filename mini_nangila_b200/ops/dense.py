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
Forward-mode derivatives and ``torch.jit.trace`` are refused with a
``NotImplementedError``.
"""
from __future__ import annotations

import torch

from .. import _ext
from .._ext import cuda

ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
_ACT = {a: i for i, a in enumerate(ACTIVATIONS)}


class DenseError(RuntimeError):
    """A product gave up waiting for its own copies; its output is incomplete.
    Raised by every product on that device from the first one whose call finds
    it, until ``check`` has reported it."""


def _act(activation: str) -> int:
    try:
        return _ACT[activation]
    except KeyError:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}; got {activation!r}") from None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
           residual: torch.Tensor | None = None, x_scale: torch.Tensor | None = None,
           w_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` with sums in fp32.

    * ``x``: [..., in_features], bfloat16 or float16, at least one feature;
      ``weight``: [out_features, in_features] and ``bias``: [out_features] of the same type;
    * ``residual``: the output's shape, of x's type or float32; the output has
      its type;
    * 8 bits: ``x`` and ``weight`` float8_e4m3fn with ``x_scale`` (one float32 a
      row of x) and ``w_scale`` (one an output feature); bias and output are of
      ``out_dtype`` (bfloat16 by default).  No gradient.
    * ``out_dtype`` may also be float32, where no gradient is needed.

    The backward pass gives gradients to x, weight, bias and residual.  It
    keeps the sums before an activation in 24 bits, and rounds their gradient
    to x's type before the two products.
    """
    return cuda().linear(x, weight, bias, _act(activation), residual, x_scale, w_scale, out_dtype)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, activation: str = "silu",
                 x_scale: torch.Tensor | None = None, gate_scale: torch.Tensor | None = None,
                 up_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``activation(x @ w_gate.T) * (x @ w_up.T)`` in one kernel.

    Types and 8-bit operands as in ``linear``: ``x_scale`` one float32 a row,
    ``gate_scale`` and ``up_scale`` one an output feature.  The backward pass
    keeps both projections in 24 bits and gives gradients to x and both
    weights.
    """
    return cuda().gated_linear(x, w_gate, w_up, _act(activation), x_scale, gate_scale, up_scale, out_dtype)


def _index(device: int | torch.device | None) -> int:
    idx = device.index if isinstance(device, torch.device) else device
    return torch.cuda.current_device() if idx is None else int(idx)


def check(device: int | torch.device | None = None) -> None:
    """Raise ``DenseError`` if a product on ``device`` gave up a wait since the
    last check (waits end after 4 s); synchronises its current stream."""
    idx = _index(device)
    st = cuda().dense_status(idx, True)
    if st[0] != 0:
        raise DenseError(f"a dense product on cuda:{idx} gave up a wait: status {st}")


def poll(device: int | torch.device | None = None) -> None:
    """``check`` without waiting: raise if a product that has ended, of those on
    ``device``, gave up.  ``check`` clears the status."""
    ext = _ext._cuda
    if ext is not None:  # else no product was started
        idx = _index(device)
        if code := ext.dense_gave_up(idx):
            raise DenseError(f"a dense product on cuda:{idx} gave up a wait (status {code})")
