"""Arguments that the dense and norm operators refuse (the checks come before
any GPU work, so they run here on CPU tensors)."""
import pytest
import torch

from mini_nangila_b200 import _ext
from mini_nangila_b200.ops import dense, norm

pytestmark = pytest.mark.skipif(not _ext.cuda_available(), reason="the CUDA extension is not built")
BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


LINEAR = [
    (dict(x=z(2, 8), weight=z(3, 8)), "CUDA tensor"),
    (dict(x=z(2, 8, dtype=torch.float32), weight=z(3, 8, dtype=torch.float32)), "bfloat16, float16"),
    (dict(x=z(2, 8), weight=z(3, 8, dtype=torch.float16)), "like x"),
    (dict(x=z(2, 8), weight=z(3, 9)), "out_features"),
    (dict(x=z(2, 8), weight=z(8)), "out_features"),
    (dict(x=z(2, 0), weight=z(3, 0)), "no features"),
    (dict(x=torch.zeros((), dtype=BF), weight=z(3, 1)), "dimension"),
    (dict(x=z(2, 8), weight=z(3, 8), bias=z(4)), "bias"),
    (dict(x=z(2, 8), weight=z(3, 8), bias=z(3, dtype=torch.float32)), "bias"),
    (dict(x=z(2, 8), weight=z(3, 8), residual=z(1, 3)), "residual"),
    (dict(x=z(2, 8), weight=z(3, 8), residual=z(2, 3, dtype=torch.float16)), "residual"),
    (dict(x=z(2, 8), weight=z(3, 8), residual=z(2, 3), out_dtype=torch.float32), "residual's type"),
    (dict(x=z(2, 8), weight=z(3, 8), out_dtype=torch.float16), "out_dtype"),
    (dict(x=z(2, 8), weight=z(3, 8), activation="tanh"), "activation"),
    (dict(x=z(2, 8), weight=z(3, 8), x_scale=z(2, dtype=torch.float32)), "8-bit"),
    (dict(x=z(2, 8), weight=z(3, 8), w_scale=z(3, dtype=torch.float32)), "8-bit"),
    (dict(x=z(2, 8).to(F8), weight=z(3, 8).to(F8)), "x_scale"),
    (dict(x=z(2, 8).to(F8), weight=z(3, 8).to(F8), x_scale=z(2, dtype=torch.float32)), "w_scale"),
    (dict(x=z(2, 8).to(F8), weight=z(3, 8).to(F8), x_scale=z(3, dtype=torch.float32),
          w_scale=z(3, dtype=torch.float32)), "x_scale"),
    (dict(x=z(2, 8).to(F8), weight=z(3, 8).to(F8), x_scale=z(2, dtype=torch.float32), w_scale=z(3)), "w_scale"),
    (dict(x=z(2, 8).to(F8), weight=z(3, 8), x_scale=z(2, dtype=torch.float32)), "like x"),
]


@pytest.mark.parametrize("kw,text", LINEAR)
def test_linear_refuses(kw, text):
    with pytest.raises(ValueError if text == "activation" else RuntimeError, match=text):
        dense.linear(**kw)


GATED = [
    (dict(x=z(2, 8), w_gate=z(3, 8), w_up=z(3, 8)), "CUDA tensor"),
    (dict(x=z(2, 8), w_gate=z(3, 8), w_up=z(4, 8)), "same out_features"),
    (dict(x=z(2, 8), w_gate=z(3, 8), w_up=z(3, 7)), "w_up"),
    (dict(x=z(2, 8), w_gate=z(3, 8, dtype=torch.float16), w_up=z(3, 8)), "w_gate"),
    (dict(x=z(2, 8), w_gate=z(3, 8), w_up=z(3, 8), activation="swish"), "activation"),
    (dict(x=z(2, 8), w_gate=z(3, 8), w_up=z(3, 8), out_dtype=torch.float16), "out_dtype"),
    (dict(x=z(2, 8).to(F8), w_gate=z(3, 8).to(F8), w_up=z(3, 8).to(F8), x_scale=z(2, dtype=torch.float32),
          gate_scale=z(3, dtype=torch.float32)), "up_scale"),
]


@pytest.mark.parametrize("kw,text", GATED)
def test_gated_refuses(kw, text):
    with pytest.raises(ValueError if text == "activation" else RuntimeError, match=text):
        dense.gated_linear(**kw)


def test_gradients_of_8_bit_operands_are_refused():
    x, w, s = z(2, 8).to(F8), z(3, 8).to(F8), z(2, dtype=torch.float32)
    b = z(3).requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        dense.linear(x, w, b, x_scale=s, w_scale=z(3, dtype=torch.float32))
    with pytest.raises(ValueError, match="out_dtype"):
        dense.linear(z(2, 8).requires_grad_(), z(3, 8), out_dtype=torch.float32)
    with pytest.raises(ValueError, match="out_dtype"):
        dense.gated_linear(z(2, 8).requires_grad_(), z(3, 8), z(3, 8), out_dtype=torch.float32)


NORM = [
    (dict(x=z(2, 8), weight=z(8)), "CUDA tensor"),
    (dict(x=z(2, 8), weight=z(7)), "weight"),
    (dict(x=z(2, 8), weight=z(1, 8)), "weight"),
    (dict(x=z(2, 8), weight=z(8, dtype=torch.float16)), "weight"),
    (dict(x=z(2, 8, dtype=torch.float64), weight=z(8, dtype=torch.float64)), "float32"),
    (dict(x=z(2, 8), weight=z(8), residual=z(1, 8)), "residual"),
    (dict(x=z(2, 8, dtype=torch.float32), weight=z(8, dtype=torch.float32), residual=z(2, 8)), "residual"),
    (dict(x=z(2, 8), weight=z(8), eps=-1.0), "eps"),
    (dict(x=z(2, 0), weight=z(0)), "1 to 32768"),
    (dict(x=z(1, 32769), weight=z(32769)), "1 to 32768"),
    (dict(x=torch.zeros((), dtype=BF), weight=z(1)), "dimension"),
]


@pytest.mark.parametrize("kw,text", NORM)
def test_norm_refuses(kw, text):
    for f in (norm.rms_norm, norm.rms_norm_fp8):
        with pytest.raises(RuntimeError, match=text):
            f(**kw)


def test_quantize_rows_refuses():
    for x, text in ((z(2, 8), "CUDA tensor"), (z(2, 8, dtype=torch.int32), "float32"), (z(2, 0), "1 to 32768")):
        with pytest.raises(RuntimeError, match=text):
            norm.quantize_rows(x)


def test_arguments_of_another_kind_are_refused():
    x, w = z(2, 8), z(3, 8)
    for call, text in ((lambda: dense.linear(x, 3), "weight must be a torch.Tensor, not int"),
                       (lambda: dense.linear(x, w, residual=[1]), "residual must be a torch.Tensor"),
                       (lambda: dense.linear(x, w, out_dtype="bf16"), "out_dtype must be a torch.dtype"),
                       (lambda: dense.gated_linear(x, w, None), "w_up must be a torch.Tensor"),
                       (lambda: norm.rms_norm(None, w), "x must be a torch.Tensor"),
                       (lambda: norm.rms_norm(x, w, residual=0), "residual must be a torch.Tensor"),
                       (lambda: norm.rms_norm(x, w, "a"), "real number"),
                       (lambda: norm.quantize_rows([1.0]), "x must be a torch.Tensor")):
        with pytest.raises(TypeError, match=text):
            call()
    with pytest.raises(RuntimeError, match="out_dtype"):
        norm.rms_norm(z(2, 8), z(8), out_dtype=torch.float32)


def test_plans_of_products():
    """The planner takes every tile shape somewhere, splits k only where tiles
    leave SMs idle, and never into pieces of fewer than 4 blocks of k."""
    plan = _ext.cuda().dense_plan
    seen = set()
    for m in (17, 64, 300, 777, 2048, 8192, 100_000):
        for n in (16, 768, 2048, 5632, 50_304):
            for k in (64, 771, 2048, 8192):
                for dual in range(4):
                    for fp8 in (False, True):
                        cg, nb, splits = plan(m, n, k, dual, fp8, 148)
                        assert cg in (1, 2) and nb in (128, 256) and 1 <= splits <= 32
                        seen.add((cg, nb, splits > 1))
                        blocks = -(-k // (128 if fp8 else 64)) * (2 if dual == 2 else 1)
                        tiles = -(-m // (128 * cg)) * -(-n // (nb // 2 if dual == 1 else nb)) * (2 if dual == 3 else 1)
                        assert splits == 1 or (blocks // splits >= 4 and tiles * splits <= 148 // cg)
    assert {(c, n) for c, n, _ in seen} == {(1, 128), (1, 256), (2, 128), (2, 256)}
    assert any(s for *_, s in seen)
    for bad in ((0, 1, 1, 0, False, 148), (1, 1, 1, 4, False, 148), (1, 1, 1, 0, False, 1)):
        with pytest.raises(RuntimeError, match="positive"):
            plan(*bad)
    for bad in ((3, 128, 1), (1, 64, 1), (1, 128, 0), (2, 256, 65)):
        with pytest.raises(RuntimeError, match="plan has"):
            _ext.cuda().dense_force_plan(*bad)
