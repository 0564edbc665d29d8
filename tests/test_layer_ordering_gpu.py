"""Operators that read what the kernel directly in front of them has just
written: weights, scales, residuals and norms' weights, not activations alone.
Each chain gives the bits that it gives with the GPU waited for in between."""
import pytest
import torch

from mini_nangila_b200.ops import dense, norm

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def randn(*shape, seed, dtype=BF16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def same_without_waiting(step, inputs):
    """step(input, sync) for each input: outputs of an input's turn live in the
    memory that the turn before has just freed, so a value read too early is
    another input's."""
    want = [[t.clone() for t in step(v, torch.cuda.synchronize)] for v in inputs]
    torch.cuda.synchronize()
    for _ in range(10):
        for v, w in zip(inputs, want):
            assert all(torch.equal(p, q) for p, q in zip(step(v, lambda: None), w))
    dense.check()


@pytest.mark.parametrize("rows", [1, 8, 16, 24, 200])
def test_weights_quantised_in_front(rows):
    x8, xs = norm.quantize_rows(randn(rows, 512, seed=1))

    def step(w, sync):
        w8, ws = norm.quantize_rows(w)
        sync()
        y = dense.linear(x8, w8, x_scale=xs, w_scale=ws)
        sync()
        u8, us = norm.quantize_rows(w)
        sync()
        return y, dense.gated_linear(x8, u8, u8, x_scale=xs, gate_scale=us, up_scale=us)

    with torch.no_grad():
        same_without_waiting(step, [randn(2048, 512, seed=s, std=0.04) for s in range(2, 6)])


@pytest.mark.parametrize("rows,k", [(1, 512), (8, 509), (16, 512), (24, 512), (200, 509)])
def test_weights_made_by_a_product_in_front(rows, k):
    """k = 509: rows that 16 bytes do not divide, read word by word or copied."""
    x, a = randn(rows, k, seed=11), randn(k, 64, seed=12, std=0.1)

    def step(b, sync):
        w = dense.linear(b, a)
        sync()
        y = dense.linear(x, w)
        sync()
        v = dense.linear(b, a, activation="silu")
        sync()
        return y, dense.gated_linear(x, v, v)

    with torch.no_grad():
        same_without_waiting(step, [randn(1024, 64, seed=s) for s in range(13, 17)])


@pytest.mark.parametrize("rows", [4, 300])
def test_residuals_and_norm_weights_made_in_front(rows):
    x, w, one = randn(rows, 256, seed=21), randn(256, 256, seed=22, std=0.06), randn(256, seed=23)

    def step(a, sync):
        r = norm.rms_norm(a, one)
        sync()
        y = dense.linear(x, w, residual=r)
        sync()
        s = norm.rms_norm(y[0], one)
        sync()
        n, t = norm.rms_norm(x, s, residual=y)
        sync()
        b = norm.rms_norm(t[0], one)
        sync()
        return n, t, dense.linear(x, w, b, activation="gelu")

    with torch.no_grad():
        same_without_waiting(step, [randn(rows, 256, seed=s) for s in range(24, 28)])


@pytest.mark.parametrize("rows", [3, 300])
def test_an_optimizer_step_in_front(rows):
    """Forward, backward, update in place, forward: the product behind the update
    reads the new weights, and the norm behind it its new weight."""
    def run(seed, sync):
        w = randn(256, 256, seed=seed, std=0.06).requires_grad_()
        s = randn(256, seed=seed + 1).requires_grad_()
        x = randn(rows, 256, seed=31)
        opt = torch.optim.SGD([w, s], lr=0.1)
        out = []
        for _ in range(3):
            sync()
            n = norm.rms_norm(x, s)
            sync()
            y = dense.linear(n, w, activation="silu")
            sync()
            opt.zero_grad()
            y.float().square().mean().backward()
            sync()
            opt.step()
            out.append(y.detach())
        return [*out, w.detach(), s.detach()]

    same_without_waiting(run, [32, 42])
