"""rms_norm, rms_norm_fp8 and quantize_rows on the GPU against 64 bits."""
import pytest
import torch

from mini_nangila_b200.ops import norm
from tests import layer_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (FP16, FP16, FP16), (BF16, F32, F32), (FP16, F32, FP16),
         (BF16, BF16, F32)]  # x, stream, weight
SIZES = [(1, 1), (3, 7), (5, 64), (2, 256), (9, 257), (130, 512), (4, 1000), (33, 1024), (7, 2048), (5, 2051),
         (3, 4096), (2, 8192), (1, 8200), (2, 32768)]


def randn(*shape, seed, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


@pytest.mark.parametrize("xt,st,wt", TYPES)
@pytest.mark.parametrize("rows,width", SIZES)
def test_forward(rows, width, xt, st, wt):
    x, w = randn(rows, width, seed=1, dtype=xt), 1 + randn(width, seed=2, std=0.2)
    w = w.to(wt)
    y, u, _ = O.rms_norm(x, w, 1e-5)
    got = norm.rms_norm(x, w)
    assert got.dtype == xt
    O.close(got, y, u * y.abs() + O.half_step(y, xt) * 1.01 + 1e-30)
    r = randn(rows, width, seed=3, dtype=st, std=3.0)
    y, u, s = O.rms_norm(x, w, 1e-6, r)
    got, stream = norm.rms_norm(x, w, 1e-6, residual=r)
    assert torch.equal(stream, s) and got.dtype == xt
    O.close(got, y, u * y.abs() + O.half_step(y, xt) * 1.01 + 1e-30)


@pytest.mark.parametrize("xt,st,wt", TYPES)
@pytest.mark.parametrize("rows,width", SIZES + [(1500, 96), (700, 2048)])
def test_gradients(rows, width, xt, st, wt):
    x, r = randn(rows, width, seed=11, dtype=xt), randn(rows, width, seed=12, dtype=st, std=2.0)
    w = (1 + randn(width, seed=13, std=0.2)).to(wt)
    dy, ds = randn(rows, width, seed=14, dtype=xt), randn(rows, width, seed=15, dtype=st)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    y, s = norm.rms_norm(x, w, residual=r)
    dx, dw, dr = torch.autograd.grad([y, s], leaves, [dy, ds])
    with torch.no_grad():
        d, ed, v, ev = O.rms_norm_grads(dy, ds, s, w, 1e-5)
        O.close(dx, d, ed + O.half_step(d, xt) * 1.01)
        O.close(dr, d, ed + O.half_step(d, st) * 1.01)
        O.close(dw, v, ev + O.half_step(v, wt) * 1.01)
    # without a residual
    y = norm.rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, leaves[:2], dy)
    with torch.no_grad():
        d, ed, v, ev = O.rms_norm_grads(dy, None, x, w, 1e-5)
        O.close(dx, d, ed + O.half_step(d, xt) * 1.01)
        O.close(dw, v, ev + O.half_step(v, wt) * 1.01)


def test_gradient_through_either_output_alone():
    x, r = randn(20, 96, seed=21, dtype=BF16), randn(20, 96, seed=22, dtype=BF16)
    w = randn(96, seed=23, dtype=BF16)
    g = randn(20, 96, seed=24, dtype=BF16)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    y, s = norm.rms_norm(x, w, residual=r)
    dx, dw, dr = torch.autograd.grad(s, leaves, g, retain_graph=True, allow_unused=True)
    assert torch.equal(dx, g) and torch.equal(dr, g) and (dw is None or not dw.any())
    dx, dw, dr = torch.autograd.grad(y, leaves, g)
    with torch.no_grad():
        d, ed, v, ev = O.rms_norm_grads(g, None, s, w, 1e-5)
        O.close(dx, d, ed + O.half_step(d, BF16) * 1.01)
        O.close(dw, v, ev + O.half_step(v, BF16) * 1.01)


def test_gradient_against_differences():
    x, w = randn(6, 40, seed=31), randn(40, seed=32)
    g = randn(6, 40, seed=33)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    gx, gw = torch.autograd.grad(norm.rms_norm(x, w), leaves, g)
    with torch.no_grad():
        vx, vw, h = randn(6, 40, seed=34).double(), randn(40, seed=35).double(), 1e-5
        f = [(O.rms_norm(x.double() + s * h * vx, w.double() + s * h * vw, 1e-5)[0] * g.double()).sum()
             for s in (1, -1)]
        num = (f[0] - f[1]) / (2 * h)
        a, b = (gx.double() * vx).sum(), (gw.double() * vw).sum()
        # fp32 gradients: 80 units of 2^-24 of the terms; differences: h^2
        scale = (gx.double() * vx).abs().sum() + (gw.double() * vw).abs().sum()
        assert abs(num - a - b) <= 1e-5 * scale


@pytest.mark.parametrize("xt", [F32, BF16, FP16])
@pytest.mark.parametrize("rows,width", SIZES)
def test_fp8(rows, width, xt):
    x, r = randn(rows, width, seed=41, dtype=xt), randn(rows, width, seed=42, dtype=xt, std=3.0)
    w = (1 + randn(width, seed=43, std=0.2)).to(xt)
    y, u, s = O.rms_norm(x, w, 1e-5, r)
    codes, scale, stream = norm.rms_norm_fp8(x, w, residual=r)
    assert codes.dtype == torch.float8_e4m3fn and scale.shape == (rows,) and torch.equal(stream, s)
    sc = y.abs().amax(-1) / 448
    O.close(scale, sc, sc * (u + 2.0 ** -22))
    # e4m3: half a step is 2^-4 of the value, at least half of the smallest step, 2^-10
    back = codes.double() * scale.double()[:, None]
    O.close(back, y, y.abs() * (2.0 ** -4 + 2 * u + 2.0 ** -21) + sc[:, None] * 2.0 ** -10 * 1.001)
    q, qs = norm.quantize_rows(x)
    sc = x.double().abs().amax(-1) / 448
    O.close(qs, sc, sc * 2.0 ** -22)
    O.close(q.double() * qs.double()[:, None], x.double(),
            x.double().abs() * (2.0 ** -4 + 2.0 ** -21) + sc[:, None] * 2.0 ** -10 * 1.001)


def test_zero_tiny_and_special_rows():
    x = torch.zeros(5, 300, device="cuda")
    x[1, 7] = 1e-38
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    x[4] = 2.0
    w = torch.ones(300, device="cuda")
    y = norm.rms_norm(x, w)
    assert not y[0].any() and y[2].isnan().all() and torch.allclose(y[4], torch.ones(300, device="cuda"), atol=1e-5)
    codes, scale = norm.quantize_rows(x)
    assert not codes[0].float().any() and (scale[:2] == 2.0 ** -126).all()
    assert codes[2, 3].float().isnan() and not codes[2, :3].float().any()
    assert not (codes[3].float() * scale[3]).isfinite().any()
    assert (codes[4].float() == 448).all()


def test_strides_and_empty():
    base = randn(40, 3 * 130, seed=51, dtype=BF16)
    w = randn(130, seed=52, dtype=BF16)
    r = randn(40, 135, seed=53, dtype=BF16)[:, 1:131]
    for x in (base[:, :130], base[:, 1:131], base[:, ::3], base[:, :130].t().contiguous().t(),
              base[:1, :130].expand(40, 130)):
        y, u, s = O.rms_norm(x, w, 1e-5, r)
        got, stream = norm.rms_norm(x, w, residual=r)
        assert torch.equal(stream, s)
        O.close(got, y, u * y.abs() + O.half_step(y, BF16) * 1.01)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    norm.rms_norm(x, w).sum().backward()
    assert x.grad.shape == (0, 8) and not w.grad.any()
    assert norm.rms_norm_fp8(x, w)[0].shape == (0, 8)
    assert norm.rms_norm(randn(3, 4, 8, seed=1), w).shape == (3, 4, 8)
