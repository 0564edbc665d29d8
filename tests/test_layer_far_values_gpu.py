"""Values and gradients where pre-activations lie far from zero, as in a gate
that has diverged: beyond 12 an activation is z and its derivative 1, below -12
both are an exponential's tail."""
import pytest
import torch

from mini_nangila_b200.ops import dense
from tests import layer_oracle as O

pytestmark = pytest.mark.gpu
FAR = [12.0, 16.0, 20.0, 29.0, 31.0, 40.0, 60.0, 90.0, 110.0, 1e3, 1e5, 1e15, 1e30]


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh", "gelu", "relu"])
@pytest.mark.parametrize("m", [1, 40])
def test_far_gates(kind, m):
    """One feature of ones: g and u are the weights, dg and du the gradients' rows,
    each read off by itself.  act(g) and act'(g) are off by their own rounding to
    bf16, 2^-8, and on the tail by that of the exponential's argument, 2^-24 |g|
    of the value, and a few units of 2^-22 for the exponential, the reciprocal and
    two products (16 of them); 2^-20 is four times that.  Tails below 1e-30 (GELU's
    from -12 on, the others' from -70) may be 0."""
    z = torch.tensor([s * v for v in FAR for s in (1, -1)], device="cuda").bfloat16()
    x = torch.ones(m, 1, device="cuda").bfloat16()
    wg = z[:, None].clone().requires_grad_()
    wu = torch.full_like(wg, 2.0).requires_grad_()
    dh = torch.zeros(m, z.numel(), device="cuda").bfloat16()
    dh[0] = 1
    h = dense.gated_linear(x, wg, wu, activation=kind)
    dg, du = (t[:, 0].double() for t in torch.autograd.grad(h, [wg, wu], dh))
    z = z.double()
    pos = z > 0
    near = torch.where(z > -80, z, torch.full_like(z, -80.0))  # the oracle's own products stay finite
    v, d = O.act(torch.where(pos, torch.full_like(z, 12.0), near), kind)
    v, d = torch.where(pos, z, v), torch.where(pos, torch.ones_like(z), d)
    off = 2.0 ** -8 + torch.where(pos, 0.0, (near.abs() + 16) * 2.0 ** -20)
    O.close(h[0].double(), 2 * v, 2 * (off * v.abs() + 1e-30))
    O.close(du, v, off * v.abs() + 1e-30)
    O.close(dg, 2 * d, 2 * (off * d.abs() + 1e-30))
