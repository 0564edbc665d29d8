"""Dense layers and the root-mean-square norm in 64 bits, each value with a
bound on how far a right kernel may be from it.

Bounds count roundings: a value stored in type t is off by at most
``finfo(t).eps / 2`` of itself (half a step; half of fp16's smallest step
where it is subnormal), and an fp32 sum of n products by at most ``(n + 8) *
2^-23`` of the sum of their magnitudes (a product or a partial sum loses at
most one unit of the last place, also where a unit truncates)."""
import math

import torch

E4M3_MAX = 448.0
# largest |second derivative| of each activation: what an error of z costs in act'(z)
CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "gelu_tanh": 0.82, "silu": 0.5}
SLOPE = 1.13  # largest |first derivative|
KEPT = 2.0 ** -15  # pre-activations kept in 24 bits: one step of 16 significant bits, cut off
MATH = 2.0 ** -20  # the fast exponential and divide, relative, with room for their arguments


def act(z, kind):
    """(value, derivative) in 64 bits."""
    if kind == "relu":
        on = (z > 0).double()
        return z * on, on
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if kind == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * a * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * 2 * a * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def half_step(v, dtype):
    """Bound of one rounding of v to dtype."""
    return v.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def product(x, w):
    """x @ w.T and its fp32 bound."""
    x, w = x.double(), w.double()
    return x @ w.t(), (x.shape[-1] + 8) * 2.0 ** -23 * (x.abs() @ w.abs().t())


def close(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    d = (got.double() - want).abs()
    bad = ~(d <= bound)  # a NaN is bad
    assert not bad.any(), (what, int(bad.sum()), bad.numel(), float((d / bound)[bad].max()), bad.nonzero()[:4].tolist())


def linear(x, w, b=None, kind="none", r=None, out=None, xs=None, ws=None):
    """(y, bound, z, bound of z as computed)."""
    z, ez = product(x, w)
    if xs is not None:
        q = xs.double()[:, None] * ws.double()[None]
        z, ez = z * q, ez * q + (z * q).abs() * 2.0 ** -22
    if b is not None:
        z, ez = z + b.double(), ez + 2.0 ** -23 * (z.abs() + b.double().abs())
    y, _ = act(z, kind)
    ey = SLOPE * ez + MATH * (y.abs() + (z.abs() if kind != "none" else 0))
    if r is not None:
        y = y + r.double()
        ey = ey + 2.0 ** -23 * y.abs()
    return y, ey + half_step(y, out or x.dtype), z, ez


def linear_grads(dy, x, w, z, ez, kind, with_bias):
    """[(dx, bound), (dw, bound)(, (db, bound))]; z kept in 24 bits and dz rounded once, as documented."""
    t = x.dtype
    dy64 = dy.double()
    _, d = act(z, kind)
    dz = dy64 * d
    if kind == "none":
        e = torch.zeros_like(dz) if dy.dtype == t else half_step(dz, t)
        sum_e = torch.zeros_like(dz)
    else:
        off = ez + KEPT * z.abs()
        e = dy64.abs() * (CURVE[kind] * off + MATH * (1 + z.abs()))
        if kind == "relu":
            e = e + dy64.abs() * (z.abs() <= off)
        sum_e = e
        e = e + half_step(dz.abs() + e, t)
    dx, edx = product(dz, w.t())
    dw, edw = product(dz.t(), x.t())
    out = [(dx, edx + e @ w.double().abs() + half_step(dx, t) * 1.01),
           (dw, edw + e.t() @ x.double().abs() + half_step(dw, t) * 1.01)]
    if with_bias:
        db = dz.sum(0)
        out.append((db, (dz.shape[0] + 8) * 2.0 ** -23 * dz.abs().sum(0) + sum_e.sum(0) + half_step(db, t) * 1.01))
    return [(v, b + 1e-30) for v, b in out]


def gated(x, wg, wu, kind, out=None, xs=None, gs=None, us=None):
    """(h, bound, (g, bound, u, bound))."""
    _, _, g, eg = linear(x, wg, xs=xs, ws=gs, out=out or x.dtype)
    _, _, u, eu = linear(x, wu, xs=xs, ws=us, out=out or x.dtype)
    a, _ = act(g, kind)
    ea = SLOPE * eg + MATH * (a.abs() + g.abs())
    h = a * u
    return h, a.abs() * eu + u.abs() * ea + ea * eu + half_step(h, out or x.dtype) * 1.01 + 1e-30, (g, eg, u, eu)


def gated_grads(dh, x, wg, wu, kind, pre):
    g, eg, u, eu = pre
    t = x.dtype
    d64 = dh.double()
    a, s = act(g, kind)
    og, ou = eg + KEPT * g.abs(), eu + KEPT * u.abs()
    es = CURVE[kind] * og + MATH * (1 + g.abs())
    ea = SLOPE * og + MATH * (a.abs() + g.abs())
    if kind == "relu":
        es = es + (g.abs() <= og)
    dg, du = d64 * u * s, d64 * a
    edg = d64.abs() * (u.abs() * es + ou * s.abs() + ou * es)
    edu = d64.abs() * ea
    edg, edu = edg + half_step(dg.abs() + edg, t), edu + half_step(du.abs() + edu, t)
    dx1, e1 = product(dg, wg.t())
    dx2, e2 = product(du, wu.t())
    dx = dx1 + dx2
    ax = x.double().abs()
    dwg, e3 = product(dg.t(), x.t())
    dwu, e4 = product(du.t(), x.t())
    return [(dx, 2 * (e1 + e2) + edg @ wg.double().abs() + edu @ wu.double().abs() + half_step(dx, t) * 1.01 + 1e-30),
            (dwg, e3 + edg.t() @ ax + half_step(dwg, t) * 1.01 + 1e-30),
            (dwu, e4 + edu.t() @ ax + half_step(dwu, t) * 1.01 + 1e-30)]


def rms_norm(x, w, eps, r=None):
    """(y in 64 bits, relative bound before its rounding, the stream)."""
    s = x if r is None else (x.double() + r.double()).to(r.dtype)
    v = s.double()
    y = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    # the sum of squares (each term and partial sum one unit), its root, three products
    return y, (x.shape[-1] / 2 + 16) * 2.0 ** -24, s


def rms_norm_grads(dy, ds, s, w, eps):
    """(dstream, bound before rounding, dweight, bound before rounding)."""
    v, dy, w = s.double(), dy.double(), w.double()
    n = v.shape[-1]
    inv = 1 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    hat, g = v * inv, dy * w
    dot = (g * hat).mean(-1, keepdim=True)
    d = inv * (g - hat * dot)
    u = (n + 32) * 2.0 ** -23
    ed = u * inv * (g.abs() + hat.abs() * (g * hat).abs().mean(-1, keepdim=True))
    if ds is not None:
        d = d + ds.double()
        ed = ed + 2.0 ** -23 * d.abs()
    dw = (dy * hat).sum(0)
    return d, ed + 1e-30, dw, (n / 2 + 32 + dy.shape[0]) * 2.0 ** -23 * (dy * hat).abs().sum(0) + 1e-30
