"""linear and gated_linear on the GPU against 64 bits (tests/layer_oracle.py):
the few-row kernel, the tensor-core kernel at sizes no tile divides, splits of
k, strides and alignments, 8-bit operands, and both backward passes."""
import pytest
import torch

from mini_nangila_b200.ops import dense, norm
from tests import layer_oracle as O

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def randn(*shape, seed, dtype=torch.float32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def operands(m, k, n, dtype, seed=0):
    return randn(m, k, seed=seed, dtype=dtype), randn(n, k, seed=seed + 1, dtype=dtype, std=k ** -0.5)


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    dense.check()


SKINNY = [(1, 64, 16), (1, 768, 768), (3, 100, 33), (8, 2048, 128), (9, 77, 50), (17, 129, 65), (32, 1000, 200)]
TILED = [(33, 64, 64), (128, 64, 128), (200, 136, 72), (257, 192, 264), (300, 1024, 96), (64, 4096, 128),
         (777, 513, 385), (1, 33, 1), (1024, 768, 2304)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,k,n", SKINNY + TILED)
def test_linear_sizes(m, k, n, dtype):
    x, w = operands(m, k, n, DT[dtype])
    y, e, _, _ = O.linear(x, w)
    O.close(dense.linear(x, w), y, e)


@pytest.mark.parametrize("kind", dense.ACTIVATIONS)
@pytest.mark.parametrize("m,k,n,dtype", [(5, 96, 40, "bf16"), (150, 96, 200, "fp16"), (150, 96, 203, "bf16")])
def test_linear_epilogue(m, k, n, dtype, kind):
    x, w = operands(m, k, n, DT[dtype], seed=3)
    b, r = randn(n, seed=5, dtype=DT[dtype]), randn(m, n, seed=6, dtype=DT[dtype])
    for bias, res in ((b, None), (None, r), (b, r), (b, r.float())):
        y, e, _, _ = O.linear(x, w, bias, kind, res, out=x.dtype if res is None else res.dtype)
        got = dense.linear(x, w, bias, activation=kind, residual=res)
        assert got.dtype == (x.dtype if res is None else res.dtype)
        O.close(got, y, e, (kind, bias is not None, res is not None))


def test_linear_wide_range():
    """Activations far from zero, where an exponential overflows."""
    for kind in dense.ACTIVATIONS:
        x = torch.tensor([[1.0]], device="cuda").bfloat16()
        w = torch.tensor([[-200.0], [-90.0], [-20.0], [0.0], [20.0], [90.0], [200.0]], device="cuda").bfloat16()
        for rows in (1, 40):
            xx = x.expand(rows, 1).contiguous()
            y, e, z, _ = O.linear(xx, w, kind=kind)
            O.close(dense.linear(xx, w, activation=kind), y, e + 1e-30, kind)


@pytest.mark.parametrize("m", [4, 130])
def test_strides_alignment_and_shapes(m):
    k, n = 96, 72
    base = randn(m, 2 * k + 3, seed=1, dtype=torch.bfloat16)
    wbase = randn(n, k + 8, seed=2, dtype=torch.bfloat16)
    views = [base[:, :k], base[:, 1:k + 1], base[:, ::2][:, :k], base.t().contiguous().t()[:, :k],
             base[:1, :k].expand(m, k)]
    weights = [wbase[:, :k], wbase[:, 1:k + 1], wbase.t().contiguous().t()[:, :k]]
    rbase = randn(m, n + 5, seed=4, dtype=torch.bfloat16)
    for x in views:
        for w in weights:
            r = rbase[:, 3:n + 3]
            y, e, _, _ = O.linear(x, w, r=r)
            O.close(dense.linear(x, w, residual=r), y, e)
    x3 = randn(2, m, k, seed=9, dtype=torch.bfloat16)
    got = dense.linear(x3, weights[0])
    assert got.shape == (2, m, n)
    O.close(got.reshape(-1, n), *O.linear(x3.reshape(-1, k), weights[0])[:2])
    assert dense.linear(x3[0, 0], weights[0]).shape == (n,)


@pytest.mark.parametrize("m,n", [(0, 8), (5, 0), (0, 0)])
def test_empty(m, n):
    x = torch.zeros(m, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.zeros(n, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = dense.linear(x, w, activation="silu")
    h = dense.gated_linear(x, w, w)
    assert y.shape == h.shape == (m, n)
    (y.sum() + h.sum()).backward()
    assert not x.grad.any() and not w.grad.any()


def test_rows_are_independent_of_special_values():
    """An infinity or NaN in one row of x reaches that row alone."""
    for m in (6, 140):
        x, w = operands(m, 80, 48, torch.bfloat16, seed=11)
        want = dense.linear(x, w, activation="gelu_tanh")
        x[2, 5], x[4, 7] = float("inf"), float("nan")
        got = dense.linear(x, w, activation="gelu_tanh")
        keep = [i for i in range(m) if i not in (2, 4)]
        assert torch.equal(got[keep], want[keep])
        assert got[4].isnan().all() and not got[2].isfinite().all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", dense.ACTIVATIONS)
@pytest.mark.parametrize("m,k,n", [(1, 64, 32), (7, 40, 33), (200, 136, 72), (1024, 64, 200), (130, 77, 259)])
def test_linear_gradients(m, k, n, kind, dtype):
    x, w = operands(m, k, n, DT[dtype], seed=20)
    b, r, dy = (randn(n, seed=22, dtype=DT[dtype]), randn(m, n, seed=23, dtype=DT[dtype]),
                randn(m, n, seed=24, dtype=DT[dtype]))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = dense.linear(x, w, b, activation=kind, residual=r)
    got = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        _, _, z, ez = O.linear(x, w, b, kind, r)
        for g, (v, e), name in zip(got, O.linear_grads(dy, x, w, z, ez, kind, True), "xwb"):
            assert g.dtype == x.dtype
            O.close(g, v, e, name)
        assert torch.equal(got[3], dy)


def test_linear_gradients_fp32_stream_and_frozen_parts():
    m, k, n = 100, 64, 48
    x, w = operands(m, k, n, torch.bfloat16, seed=30)
    r, dy = randn(m, n, seed=31), randn(m, n, seed=32)
    for need in ("xw", "x", "w", "r"):
        leaves = {"x": x.detach().requires_grad_("x" in need), "w": w.detach().requires_grad_("w" in need),
                  "r": r.detach().requires_grad_("r" in need)}
        y = dense.linear(leaves["x"], leaves["w"], activation="none", residual=leaves["r"])
        assert y.dtype == torch.float32
        y.backward(dy)
        _, _, z, ez = O.linear(x, w)
        for name, (v, e) in zip("xw", O.linear_grads(dy, x, w, z, ez, "none", False)):
            assert (leaves[name].grad is not None) == (name in need)
            if name in need:
                O.close(leaves[name].grad, v, e, name)
        assert ("r" in need) == (leaves["r"].grad is not None)


def test_gradient_against_differences():
    """dL/dt along random directions, by differences of the 64-bit formula at the kernel's own gradient."""
    x, w = operands(40, 24, 16, torch.float16, seed=40)
    dy = randn(40, 16, seed=42, dtype=torch.float16)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    gx, gw = torch.autograd.grad(dense.linear(x, w, activation="gelu"), leaves, dy)
    with torch.no_grad():
        for i in range(3):
            vx, vw = randn(40, 24, seed=50 + i).double(), randn(16, 24, seed=60 + i).double()
            h = 1e-5
            f = [(O.act((x.double() + s * h * vx) @ (w.double() + s * h * vw).t(), "gelu")[0] * dy.double()).sum()
                 for s in (1, -1)]
            num = (f[0] - f[1]) / (2 * h)
            ana = (gx.double() * vx).sum() + (gw.double() * vw).sum()
            # each gradient entry is within a few half steps (2^-11) of its magnitudes
            scale = (gx.double() * vx).abs().sum() + (gw.double() * vw).abs().sum()
            assert abs(num - ana) <= 4 * 2.0 ** -11 * scale


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,k,n", [(1, 64, 16), (5, 100, 33), (32, 2048, 48), (33, 64, 64), (200, 136, 72),
                                   (300, 1024, 130), (777, 129, 385)])
def test_gated_sizes(m, k, n, dtype):
    x, wg = operands(m, k, n, DT[dtype], seed=70)
    wu = randn(n, k, seed=73, dtype=DT[dtype], std=k ** -0.5)
    for kind in ("silu", "gelu_tanh", "none"):
        h, e, _ = O.gated(x, wg, wu, kind)
        O.close(dense.gated_linear(x, wg, wu, activation=kind), h, e, kind)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", dense.ACTIVATIONS)
@pytest.mark.parametrize("m,k,n", [(1, 64, 32), (9, 40, 33), (200, 136, 72), (600, 64, 200)])
def test_gated_gradients(m, k, n, kind, dtype):
    x, wg = operands(m, k, n, DT[dtype], seed=80)
    wu, dh = randn(n, k, seed=83, dtype=DT[dtype], std=k ** -0.5), randn(m, n, seed=84, dtype=DT[dtype])
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(dense.gated_linear(x, wg, wu, activation=kind), leaves, dh)
    with torch.no_grad():
        _, _, pre = O.gated(x, wg, wu, kind)
        for g, (v, e), name in zip(got, O.gated_grads(dh, x, wg, wu, kind, pre), ("x", "gate", "up")):
            O.close(g, v, e, name)


@pytest.mark.parametrize("m,k,n", [(1, 64, 16), (5, 100, 33), (20, 2048, 48), (33, 128, 64), (200, 136, 72),
                                   (300, 1024, 130), (140, 77, 41)])
def test_fp8_operands(m, k, n):
    x, xs = norm.quantize_rows(randn(m, k, seed=90))
    w, ws = norm.quantize_rows(randn(n, k, seed=91, std=k ** -0.5))
    wu, us = norm.quantize_rows(randn(n, k, seed=92, std=k ** -0.5))
    b, r = randn(n, seed=93, dtype=torch.bfloat16), randn(m, n, seed=94, dtype=torch.bfloat16)
    y, e, _, _ = O.linear(x.float(), w.float(), b, "gelu", r, out=torch.bfloat16, xs=xs, ws=ws)
    O.close(dense.linear(x, w, b, activation="gelu", residual=r, x_scale=xs, w_scale=ws), y, e)
    y, e, _, _ = O.linear(x.float(), w.float(), out=torch.float32, xs=xs, ws=ws)
    O.close(dense.linear(x, w, x_scale=xs, w_scale=ws, out_dtype=torch.float32), y, e)
    h, e, _ = O.gated(x.float(), w.float(), wu.float(), "silu", out=torch.bfloat16, xs=xs, gs=ws, us=us)
    O.close(dense.gated_linear(x, w, wu, x_scale=xs, gate_scale=ws, up_scale=us), h, e)


def test_every_tile_shape_and_split():
    """Sizes that the planner maps to each tile and to splits of k give the
    same sums as one row at a time does."""
    for m, k, n in [(33, 8192, 64), (129, 4096, 256), (512, 64, 4096), (2048, 256, 2048), (40, 640, 9000)]:
        x, w = operands(m, k, n, torch.bfloat16, seed=100)
        y, e, _, _ = O.linear(x, w)
        O.close(dense.linear(x, w), y, e, (m, k, n))


def test_same_bits_again():
    """No atomics: a call repeated gives the same bits, weight gradients with split sums among them."""
    x, w = operands(4096, 96, 80, torch.bfloat16, seed=110)
    b = randn(80, seed=111, dtype=torch.bfloat16)
    dy = randn(4096, 80, seed=112, dtype=torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    first = None
    for _ in range(3):
        y = dense.linear(x, w, b, activation="silu")
        got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        if first is None:
            first = got
        assert all(torch.equal(a, c) for a, c in zip(first, got))


@pytest.mark.parametrize("m", [777, 785, 129, 144, 1033])
def test_last_rows_of_a_ragged_prompt(m):
    """A few rows behind whole tiles take the few-row kernel where that is
    quicker: one row's result does not depend on the kernel beyond the bound."""
    x, w = operands(m, 512, 5632, torch.bfloat16, seed=120)
    b, r = randn(5632, seed=122, dtype=torch.bfloat16), randn(m, 5632, seed=123, dtype=torch.bfloat16)
    y, e, z, ez = O.linear(x, w, b, "silu", r)
    O.close(dense.linear(x, w, b, activation="silu", residual=r), y, e)
    dy = randn(m, 5632, seed=124, dtype=torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(dense.linear(x, w, b, activation="silu"), leaves, dy)
    with torch.no_grad():
        for g, (v, e), name in zip(got, O.linear_grads(dy, x, w, z, ez, "silu", True), "xwb"):
            O.close(g, v, e, name)
        h, e, _ = O.gated(x, w, w, "silu")
        O.close(dense.gated_linear(x, w, w), h, e)
        x8, xs = norm.quantize_rows(x)
        w8, ws = norm.quantize_rows(w)
        y, e, _, _ = O.linear(x8.float(), w8.float(), b, "none", r, out=torch.bfloat16, xs=xs, ws=ws)
        O.close(dense.linear(x8, w8, b, residual=r, x_scale=xs, w_scale=ws), y, e)
