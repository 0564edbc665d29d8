"""Paths of the dense kernels that sizes alone reach: whole sums with their
epilogue at long k (8 epilogue warps, residual fetched piece by piece), the same
in 8 bits, and the training pass of a float32 stream under autocast."""
import pytest
import torch

from mini_nangila_b200 import _ext
from mini_nangila_b200.ops import dense, norm
from tests import layer_oracle as O

pytestmark = pytest.mark.gpu
BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
PLANS = [(1, 128), (1, 256), (2, 128), (2, 256)]


def randn(*shape, seed, dtype=BF16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    dense.check()


@pytest.fixture
def force():
    yield _ext.cuda().dense_force_plan
    _ext.cuda().dense_force_plan(0, 0, 0)


@pytest.mark.parametrize("cg,nb", PLANS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k,n", [(300, 2048, 520), (257, 5632, 264), (1200, 1096, 1032)])
def test_long_sums_with_their_epilogue(m, k, n, dtype, cg, nb, force):
    """Whole sums of more than 1024 products, aligned rows: bias, activation, kept
    pre-activations and a residual of either type behind them in the same kernel."""
    x, w = randn(m, k, seed=1, dtype=dtype), randn(n, k, seed=2, dtype=dtype, std=k ** -0.5)
    b, r = randn(n, seed=3, dtype=dtype), randn(m, n, seed=4, dtype=dtype)
    dy = randn(m, n, seed=5, dtype=dtype)
    force(cg, nb, 1)
    assert _ext.cuda().dense_plan(m, n, k, 0, False, 148) == [cg, nb, 1]
    for kind, bias, res in (("none", None, r), ("gelu", b, r), ("silu", b, r.float()), ("none", None, r.float()),
                            ("relu", b, None)):
        y, e, _, _ = O.linear(x, w, bias, kind, res, out=dtype if res is None else res.dtype)
        O.close(dense.linear(x, w, bias, activation=kind, residual=res), y, e, (kind, res is None))
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    y = dense.linear(*leaves[:3], activation="gelu_tanh", residual=leaves[3])
    got = torch.autograd.grad(y, leaves, dy)
    want, e, z, ez = O.linear(x, w, b, "gelu_tanh", r)
    O.close(y, want, e)
    for g, (v, e), name in zip(got, O.linear_grads(dy, x, w, z, ez, "gelu_tanh", True), "xwb"):
        O.close(g, v, e, name)


@pytest.mark.parametrize("m,k,n", [(2048, 2048, 5632), (2048, 5632, 2048)])
def test_long_sums_as_planned(m, k, n):
    """A prompt through a layer's projections: the planner leaves these whole."""
    assert _ext.cuda().dense_plan(m, n, k, 0, False, 148)[2] == 1
    x, w = randn(m, k, seed=11), randn(n, k, seed=12, std=k ** -0.5)
    b, r = randn(n, seed=13), randn(m, n, seed=14)
    y, e, _, _ = O.linear(x, w, b, "silu", r)
    O.close(dense.linear(x, w, b, activation="silu", residual=r), y, e)
    y, e, _, _ = O.linear(x, w, r=r.float(), out=F32)
    O.close(dense.linear(x, w, residual=r.float()), y, e)


@pytest.mark.parametrize("cg,nb", PLANS)
@pytest.mark.parametrize("m,k,n", [(300, 2176, 520), (1200, 5632, 264)])
def test_long_8bit_sums_with_their_epilogue(m, k, n, cg, nb, force):
    x8, xs = norm.quantize_rows(randn(m, k, seed=21))
    w8, ws = norm.quantize_rows(randn(n, k, seed=22, std=k ** -0.5))
    u8, us = norm.quantize_rows(randn(n, k, seed=23, std=k ** -0.5))
    b, r = randn(n, seed=24), randn(m, n, seed=25)
    force(cg, nb, 1)
    assert _ext.cuda().dense_plan(m, n, k, 0, True, 148) == [cg, nb, 1]
    for kind, bias, res in (("none", None, r), ("gelu", b, r), ("silu", b, r.float()), ("none", None, None)):
        out = BF16 if res is None else res.dtype
        y, e, _, _ = O.linear(x8.float(), w8.float(), bias, kind, res, out=out, xs=xs, ws=ws)
        O.close(dense.linear(x8, w8, bias, activation=kind, residual=res, x_scale=xs, w_scale=ws), y, e,
                (kind, res is None))
    h, e, _ = O.gated(x8.float(), w8.float(), u8.float(), "silu", out=BF16, xs=xs, gs=ws, us=us)
    O.close(dense.gated_linear(x8, w8, u8, x_scale=xs, gate_scale=ws, up_scale=us), h, e)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind", ["none", "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", [(5, 96, 40), (200, 136, 72), (600, 768, 768)])
def test_training_of_a_float32_stream_under_autocast(m, k, n, kind, dtype):
    """float32 weights and stream: operands are cast as stock layers cast them, the
    stream's gradient passes whole, and the gradients of the float32 leaves are
    those of the cast operands."""
    x, r = randn(m, k, seed=31, dtype=F32), randn(m, n, seed=32, dtype=F32)
    w, b = randn(n, k, seed=33, dtype=F32, std=k ** -0.5), randn(n, seed=34, dtype=F32)
    dy = randn(m, n, seed=35, dtype=F32)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    with torch.autocast("cuda", dtype=dtype):
        y = dense.linear(*leaves[:3], activation=kind, residual=leaves[3])
    assert y.dtype == F32
    got = torch.autograd.grad(y, leaves, dy)
    xh, wh, bh = x.to(dtype), w.to(dtype), b.to(dtype)
    want, e, z, ez = O.linear(xh, wh, bh, kind, r, out=F32)
    O.close(y, want, e)
    for g, (v, e), name in zip(got, O.linear_grads(dy, xh, wh, z, ez, kind, True), "xwb"):
        assert g.dtype == F32
        O.close(g, v, e, name)
    assert torch.equal(got[3], dy)


@pytest.mark.parametrize("m,k,n", [(40, 96, 40), (300, 136, 72)])
def test_a_layers_half_under_autocast(m, k, n):
    """Norm of a float32 stream in 16 bits, gated product, product back into the
    stream, as the models run them: gradients of the float32 weights against 64
    bits.  Six roundings to bf16 (norm's output, h, dz, dg or du, the gradients
    between the products and a weight's cast), 2^-8 of the value each at most."""
    a, x = randn(m, k, seed=41), randn(m, k, seed=42, dtype=F32)
    s = 1 + randn(k, seed=43, dtype=F32, std=0.1)
    wg, wu = randn(n, k, seed=44, dtype=F32, std=k ** -0.5), randn(n, k, seed=45, dtype=F32, std=k ** -0.5)
    wd, dy = randn(k, n, seed=46, dtype=F32, std=n ** -0.5), randn(m, k, seed=47, dtype=F32)
    leaves = [t.clone().requires_grad_() for t in (a, x, s, wg, wu, wd)]
    with torch.autocast("cuda", dtype=BF16):
        h, t = norm.rms_norm(leaves[0], leaves[2], residual=leaves[1])
        y = dense.linear(dense.gated_linear(h, leaves[3], leaves[4]), leaves[5], residual=t)
    assert y.dtype == F32 and h.dtype == BF16
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    l64 = [v.detach().double().requires_grad_() for v in leaves]
    t64 = l64[0] + l64[1]
    h64 = t64 / (t64.square().mean(-1, keepdim=True) + 1e-5).sqrt() * l64[2]
    y64 = (torch.nn.functional.silu(h64 @ l64[3].t()) * (h64 @ l64[4].t())) @ l64[5].t() + t64
    want = [y64, *torch.autograd.grad(y64, l64, dy.double())]
    for p, q in zip(got, want):
        assert (p.double() - q).norm() <= 6 * 2.0 ** -8 * q.norm()
