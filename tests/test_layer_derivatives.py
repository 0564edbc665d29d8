"""Derivatives and traces that the dense and norm operators cannot give are
refused, not lost: forward-mode tangents and torch.jit.trace."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from mini_nangila_b200 import _ext
from mini_nangila_b200.ops import dense, norm

pytestmark = pytest.mark.skipif(not _ext.cuda_available(), reason="the CUDA extension is not built")
BF, F8, F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


X, W, B, R, S = z(2, 8), z(3, 8), z(3), z(2, 3), z(8)
X8, W8, SX, SW = z(2, 8).to(F8), z(3, 8).to(F8), z(2, dtype=F32), z(3, dtype=F32)
CALLS = [  # (call of one tensor, that tensor)
    ("linear", lambda t: dense.linear(t, W), X), ("linear", lambda t: dense.linear(X, t), W),
    ("linear", lambda t: dense.linear(X, W, t), B), ("linear", lambda t: dense.linear(X, W, residual=t), R),
    ("linear", lambda t: dense.linear(X8, W8, x_scale=t, w_scale=SW), SX),
    ("linear", lambda t: dense.linear(X8, W8, x_scale=SX, w_scale=t), SW),
    ("gated_linear", lambda t: dense.gated_linear(t, W, W), X),
    ("gated_linear", lambda t: dense.gated_linear(X, t, W), W),
    ("gated_linear", lambda t: dense.gated_linear(X, W, t), W),
    ("gated_linear", lambda t: dense.gated_linear(X8, W8, W8, x_scale=t, gate_scale=SW, up_scale=SW), SX),
    ("gated_linear", lambda t: dense.gated_linear(X8, W8, W8, x_scale=SX, gate_scale=t, up_scale=SW), SW),
    ("gated_linear", lambda t: dense.gated_linear(X8, W8, W8, x_scale=SX, gate_scale=SW, up_scale=t), SW),
    ("rms_norm", lambda t: norm.rms_norm(t, S), X), ("rms_norm", lambda t: norm.rms_norm(X, t), S),
    ("rms_norm", lambda t: norm.rms_norm(X, S, residual=t), X),
    ("rms_norm_fp8", lambda t: norm.rms_norm_fp8(t, S), X), ("rms_norm_fp8", lambda t: norm.rms_norm_fp8(X, t), S),
    ("rms_norm_fp8", lambda t: norm.rms_norm_fp8(X, S, residual=t), X),
    ("rms_norm_fp8", lambda t: norm.quantize_rows(t), X),
]


@pytest.mark.parametrize("name,call,t", CALLS)
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(name, call, t, leaf):
    with fw.dual_level():
        d = fw.make_dual(t.clone().requires_grad_(leaf), torch.ones_like(t))
        with pytest.raises(NotImplementedError, match=f"{name} has no forward-mode derivative"):
            call(d)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(d)
        # without its tangent the call goes as far as it goes for a plain tensor
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):
            call(fw.unpack_dual(d).primal)
        with torch.no_grad(), fw._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA tensor"):
            call(d)


@pytest.mark.parametrize("name,call,t", CALLS)
def test_traces_are_refused(name, call, t):
    with pytest.raises(NotImplementedError, match=f"{name} cannot be traced"):
        torch.jit.trace(call, (t,))


@pytest.mark.gpu
def test_forward_mode_through_the_backward_passes_is_refused():
    x, w, s = (torch.randn(*d, device="cuda").to(BF).requires_grad_() for d in ((40, 64), (24, 64), (64,)))
    for y, name in ((dense.linear(x, w, activation="silu"), "linear"), (dense.gated_linear(x, w, w), "gated_linear"),
                    (norm.rms_norm(x, s), "rms_norm"), (norm.rms_norm(x, s, residual=x)[1], "rms_norm")):
        with fw.dual_level():
            dy = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match=f"gradient of {name} has no forward-mode"):
                torch.autograd.grad(y, x, dy)


@pytest.mark.gpu
def test_transforms_raise():
    x, w = torch.randn(3, 40, 64, device="cuda").to(BF), torch.randn(24, 64, device="cuda").to(BF)
    for f in (lambda v: dense.linear(v, w), lambda v: dense.gated_linear(v, w, w), lambda v: norm.rms_norm(v, w[0])):
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: f(v).float().sum())(x)
    dense.check()
