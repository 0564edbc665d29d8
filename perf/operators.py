"""Cases for the operators of a decoder layer's dense half: the matrix product
with bias, activation and residual in its epilogue, the gated product of two
projections, and the root-mean-square norm with the residual's addition and an
output in 8 bits.

``own`` chooses between the plain form (elementary torch operations in 32 bits)
and the framework's entry points (``mini_nangila_b200.ops.dense`` and
``mini_nangila_b200.ops.norm``).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126  # the smallest scale of a row in 8 bits
EPS = 1e-5


def _case(op, **kw):
    c = dict(op=op, rows=1, k=0, n=0, dtype="bf16", act="none", bias=False, residual=False, train=False)
    c.update(kw)
    return c


def listed():
    return [
        # one token through a small model's attention output projection: latency
        _case("linear", name="linear 1 token", rows=1, k=768, n=768, bias=True, residual=True),
        # eight sequences decoded together, the down projection of a 1.1B decoder
        _case("linear", name="linear 8 tokens down", rows=8, k=5632, n=2048, residual=True),
        # a prompt through the same projection
        _case("linear", name="linear prompt down", rows=2048, k=5632, n=2048, residual=True),
        # a ragged batch and widths that no vector or tile divides
        _case("linear", name="linear odd sizes", rows=1117, k=771, n=2309, dtype="fp16", act="gelu", bias=True),
        # the encoder layer of a character model in training
        _case("linear", name="linear small train", rows=8192, k=256, n=2048, dtype="fp16", act="gelu_tanh", bias=True,
              train=True),
        # the same prompt with both operands in 8 bits
        _case("linear_fp8", name="linear fp8 prompt", rows=2048, k=2048, n=5632),
        # one token through the gated block of a 1.1B decoder: its weights are read once
        _case("gated", name="gated 1 token", rows=1, k=2048, n=5632, act="silu"),
        # a short ragged prompt
        _case("gated", name="gated ragged prompt", rows=777, k=2048, n=5632, act="silu"),
        # the training micro batch, 4 sequences of 2048 tokens, forward and backward
        _case("gated", name="gated train", rows=8192, k=2048, n=5632, act="silu", train=True),
        # eight tokens decoded: latency
        _case("norm", name="norm 8 tokens", rows=8, k=2048, residual=True),
        # the training micro batch, forward and backward
        _case("norm", name="norm train", rows=8192, k=2048, residual=True, train=True),
        # a long prompt on its way into a product in 8 bits
        _case("norm_fp8", name="norm fp8 prompt", rows=16384, k=2048, residual=True),
    ]


COST = 6.0 * 8192 * 2048 * 2 * 5632  # of the largest listed case


def _size(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice([1, 1, 8, 64])
    return max(lo, min(hi, (v + step - 1) // step * step))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_fp8", "gated", "gated", "norm", "norm", "norm_fp8"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("norm", "norm_fp8"):
        if op == "norm" and rng.random() < 0.25:
            dtype = "fp32"
        return _case(op, rows=_size(rng, 1, 16384), k=_size(rng, 64, 8192), dtype=dtype,
                     residual=rng.random() < 0.7, train=op == "norm" and rng.random() < 0.5)
    c = _case(op, rows=_size(rng, 1, 8192), k=_size(rng, 64, 5632), n=_size(rng, 64, 5632), dtype=dtype)
    if op == "linear_fp8":
        c.update(act=rng.choice(["none", "none", "gelu_tanh", "silu"]), bias=rng.random() < 0.5,
                 residual=rng.random() < 0.5)
    elif op == "linear":
        c.update(act=rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.5,
                 residual=rng.random() < 0.5, train=rng.random() < 0.5)
    else:
        c.update(act=rng.choice(["silu", "silu", "gelu_tanh"]), train=rng.random() < 0.5)
    while _flops(c) > COST:
        c["rows"] = max(1, c["rows"] // 2)
    return c


# ------------------------------------------------------------------ inputs
def _e4m3_rows(v):
    """Rows of ``v`` (fp32) in e4m3 with one scale a row."""
    s = (v.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)
    return (v / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    m, k, n, train = case["rows"], case["k"], case["n"], case["train"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    def leaf(t, to=dt):
        return t.to(to).requires_grad_(train)

    st = {"case": case}
    if case["op"] in ("norm", "norm_fp8"):
        # a residual stream with a few channels far above the others
        loud = torch.rand(k, generator=g, device="cuda") < 0.01
        st["x"] = leaf(normal(m, k))
        st["w"] = leaf(1.0 + normal(k, std=0.1))
        if case["residual"]:
            st["r"] = leaf(normal(m, k) * torch.where(loud, 20.0, 2.0))
        if train:
            st["dy"] = normal(m, k, std=1e-2).to(dt)
            if case["residual"]:
                st["ds"] = normal(m, k, std=1e-2).to(dt)
        return st
    if case["op"] == "linear_fp8":
        st["x"], st["xs"] = _e4m3_rows(normal(m, k))
        st["w"], st["ws"] = _e4m3_rows(normal(n, k, std=k ** -0.5))
    else:
        st["x"] = leaf(normal(m, k))
        st["w"] = leaf(normal(n, k, std=k ** -0.5))
    if case["op"] == "gated":
        st["w2"] = leaf(normal(n, k, std=k ** -0.5))
    if case["bias"]:
        st["b"] = leaf(normal(n, std=0.1))
    if case["residual"]:
        st["r"] = leaf(normal(m, n))
    if train:
        st["dy"] = normal(m, n, std=1e-2).to(dt)
    return st


# -------------------------------------------------------------- plain form
def _act(z, act):
    if act == "relu":
        return z * (z > 0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    return z


def _plain(st):
    c = st["case"]
    dt = DTYPES[c["dtype"]]
    x = st["x"].float()
    if c["op"] in ("norm", "norm_fp8"):
        s = (x + st["r"].float()).to(dt) if c["residual"] else st["x"]
        v = s.float()
        y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * st["w"].float()
        out = _e4m3_rows(y) if c["op"] == "norm_fp8" else (y.to(dt),)
        return (*out, s) if c["residual"] else out
    w = st["w"].float()
    if c["op"] == "linear_fp8":
        x, w = x * st["xs"][:, None], w * st["ws"][:, None]
    z = x @ w.t()
    if c["bias"]:
        z = z + st["b"].float()
    y = _act(z, c["act"])
    if c["op"] == "gated":
        y = y * (x @ st["w2"].float().t())
    if c["residual"]:
        y = y + st["r"].float()
    return (y.to(dt),)


# --------------------------------------------------- the framework's calls
def _own(st):
    from mini_nangila_b200.ops import dense, norm

    c = st["case"]
    if c["op"] == "norm":
        out = norm.rms_norm(st["x"], st["w"], EPS, residual=st.get("r"))
        return out if c["residual"] else (out,)
    if c["op"] == "norm_fp8":
        return norm.rms_norm_fp8(st["x"], st["w"], EPS, residual=st.get("r"))
    if c["op"] == "gated":
        return (dense.gated_linear(st["x"], st["w"], st["w2"], activation=c["act"]),)
    if c["op"] == "linear_fp8":
        return (dense.linear(st["x"], st["w"], st.get("b"), activation=c["act"], residual=st.get("r"),
                             x_scale=st["xs"], w_scale=st["ws"], out_dtype=DTYPES[c["dtype"]]),)
    return (dense.linear(st["x"], st["w"], st.get("b"), activation=c["act"], residual=st.get("r")),)


def run(state):
    out = _own(state) if own else _plain(state)
    if not state["case"]["train"]:
        return list(out)
    outs, cots = [out[0]], [state["dy"]]
    if "ds" in state:
        outs, cots = outs + [out[1]], cots + [state["ds"]]
    wrt = [state[k] for k in ("x", "w", "w2", "b", "r") if k in state]
    return [*(o.detach() for o in out), *torch.autograd.grad(outs, wrt, cots)]


# ---------------------------------------------------------------- work
def _flops(c):
    m, k, n = c["rows"], c["k"], c["n"]
    if c["op"] in ("norm", "norm_fp8"):
        return (14.0 if c["train"] else 5.0) * m * k
    return (6.0 if c["train"] else 2.0) * m * k * n * (2 if c["op"] == "gated" else 1)


def work(case):
    m, k, n = case["rows"], case["k"], case["n"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        # x, y and, with a residual, it and their sum; then dy, ds and the gradients of x and the residual (the same)
        per = 4 if case["residual"] else 2
        b = e * (per * m * k + k)
        if case["train"]:
            b += e * ((3 if case["residual"] else 2) * m * k + k)
    elif case["op"] == "norm_fp8":
        b = e * ((3 if case["residual"] else 1) * m * k + k) + m * k + 4 * m
    else:
        q = 1 if case["op"] == "linear_fp8" else e
        nw = (2 if case["op"] == "gated" else 1) * n * k
        b = q * (m * k + nw) + e * m * n * (2 if case["residual"] else 1) + (e * n if case["bias"] else 0)
        if case["op"] == "linear_fp8":
            b += 4 * (m + n)
        if case["train"]:
            b += e * (m * n + m * k + nw + (n if case["bias"] else 0))
    return {"bytes": float(b), "flops": _flops(case)}


# ---------------------------------------------------------------- exact
def _act64(z, act):
    """The activation and its derivative in 64 bits."""
    if act == "relu":
        on = (z > 0).double()
        return z * on, on
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        # 0.5 (1 + tanh u) is the logistic function of 2 u
        s = torch.sigmoid(2 * a * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * 2 * a * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        v = {k: (t.double() if torch.is_tensor(t) else t) for k, t in st.items()}
        x, w, r, dy = v["x"], v["w"], v.get("r"), v.get("dy")
        if case["op"] in ("norm", "norm_fp8"):
            s = x if r is None else (x + r).to(DTYPES[case["dtype"]]).double()
            inv = 1 / (s.square().mean(-1, keepdim=True) + EPS).sqrt()
            hat = s * inv
            y = hat * w
            if case["op"] == "norm_fp8":
                sc = (y.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)
                out = [y / sc[:, None], sc]
            else:
                out = [y]
            out += [] if r is None else [s]
            if case["train"]:
                gh = dy * w
                ds = inv * (gh - hat * (gh * hat).mean(-1, keepdim=True))
                if r is not None:
                    ds = ds + v["ds"]
                out += [ds, (dy * hat).sum(0)] + ([] if r is None else [ds])
            return out
        if case["op"] == "linear_fp8":
            x, w = x * v["xs"][:, None], w * v["ws"][:, None]
        z = x @ w.t()
        if case["bias"]:
            z += v["b"]
        a, da = _act64(z, case["act"])
        if case["op"] == "gated":
            u = x @ v["w2"].t()
            if not case["train"]:
                return [a * u]
            dg, du = dy * u * da, dy * a
            return [a * u, dg @ w + du @ v["w2"], dg.t() @ x, du.t() @ x]
        out = [a if r is None else a + r]
        if case["train"]:
            dz = dy * da
            out += [dz @ w, dz.t() @ x] + ([dz.sum(0)] if case["bias"] else []) + ([] if r is None else [dy])
        return out
