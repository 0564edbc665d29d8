"""The dense and norm operators together, as models and training loops use
them: fused models against stock ones, the trainer, 8-bit evaluation, CUDA
graphs, streams, autocast, and sizes past 32-bit offsets."""
import subprocess
import sys
import os

import pytest
import torch
import torch.utils.checkpoint

from mini_nangila_b200 import _ext
from mini_nangila_b200.models import GPT2, GPT2Config, Llama, LlamaConfig
from mini_nangila_b200.ops import dense, norm
from tests import layer_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16 = torch.bfloat16


def randn(*shape, seed, dtype=BF16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def model(kind, fused, dtype=torch.float32):
    cfg = GPT2Config.tiny() if kind == "gpt2" else LlamaConfig.tiny()
    cfg.fused_ops = fused
    torch.manual_seed(0)
    m = (GPT2 if kind == "gpt2" else Llama)(cfg)
    with torch.no_grad():  # norms and biases away from their initial ones and zeros
        for n, p in m.named_parameters():
            if p.dim() == 1:
                p.add_(torch.randn(p.shape) * 0.1)
    return m.to("cuda", dtype)


def tokens(rows=4, seq=48):
    g = torch.Generator(device="cuda").manual_seed(3)
    t = torch.randint(0, 512, (rows, seq + 1), generator=g, device="cuda")
    return t[:, :-1].contiguous(), t[:, 1:].contiguous()


def loss_and_grads(m, autocast):
    x, y = tokens()
    with torch.autocast("cuda", dtype=BF16, enabled=autocast):
        loss = m(x, y)
    loss.backward()
    return loss.detach().double(), {n: p.grad.double() for n, p in m.named_parameters()}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gpt2", "llama"])
@pytest.mark.parametrize("mode", ["autocast", "bf16"])
def test_fused_model_is_as_near_to_fp32_as_the_stock_one(kind, mode):
    """The fused layers round no more often than the stock ones (sums, norms and
    streams in fp32, 16-bit operands), so their distance from the fp32 model is
    of the same size: at most twice the stock model's, in the 2-norm of every
    parameter's gradient, plus one rounding of it to bf16 (2^-8)."""
    dt = torch.float32 if mode == "autocast" else BF16
    ref_m = model(kind, False, dt).float()  # the same (rounded) weights
    ref = loss_and_grads(ref_m, False)
    stock = loss_and_grads(model(kind, False, dt), mode == "autocast")
    fused = loss_and_grads(model(kind, True, dt), mode == "autocast")
    dense.check()
    assert abs(fused[0] - ref[0]) <= 2 * abs(stock[0] - ref[0]) + 2.0 ** -8 * ref[0]
    for n, g in ref[1].items():
        off = [(v[1][n] - g).norm() for v in (stock, fused)]
        assert off[1] <= 2 * off[0] + 2.0 ** -8 * g.norm(), n


@pytest.mark.skipif(not _ext.cuda_available(), reason="the CUDA extension is not built")
@pytest.mark.parametrize("kind", ["gpt2", "llama"])
def test_fused_model_needs_cuda(kind):
    cfg = GPT2Config.tiny() if kind == "gpt2" else LlamaConfig.tiny()
    cfg.fused_ops = True
    m = (GPT2 if kind == "gpt2" else Llama)(cfg).to(BF16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        m(torch.zeros(1, 4, dtype=torch.long))


def test_quantize_weights_needs_fused_ops():
    with pytest.raises(ValueError, match="fused_ops"):
        Llama(LlamaConfig.tiny()).quantize_weights()


@pytest.mark.gpu
def test_8bit_evaluation():
    """Every projection in e4m3: rounding errors of 2^-4 at most, about 0.026 of
    a value's size on average, add up over 7 projections in 2 layers to a tenth
    of the logits at most; the direction of the logits stays."""
    for dt in (BF16, torch.float32):
        m = model("llama", True, dt)
        x, _ = tokens()
        with torch.no_grad(), torch.autocast("cuda", dtype=BF16, enabled=dt == torch.float32):
            a = m(x).double().flatten()
            m.quantize_weights()
            b = m(x).double().flatten()
        assert not torch.equal(a, b)
        assert torch.nn.functional.cosine_similarity(a, b, dim=0) > 0.99
    dense.check()


@pytest.mark.gpu
def test_8bit_layer_against_its_formula():
    m = model("llama", True, BF16).quantize_weights()
    f, cfg = m.layers[0], m.cfg
    x, a = randn(37, cfg.d_model, seed=1), randn(37, cfg.d_model, seed=2)
    n, s, st = norm.rms_norm_fp8(a, f.n2.weight, cfg.eps, residual=x)
    (g, gs), (u, us), (d, ds) = f.w8["gate"], f.w8["up"], f.w8["down"]
    h = dense.gated_linear(n, g, u, x_scale=s, gate_scale=gs, up_scale=us)
    want, e, _ = O.gated(n.float(), g.float(), u.float(), "silu", out=BF16, xs=s, gs=gs, us=us)
    O.close(h, want, e)
    h8, hs = norm.quantize_rows(h)
    y = dense.linear(h8, d, residual=st, x_scale=hs, w_scale=ds)
    want, e, _, _ = O.linear(h8.float(), d.float(), r=st, out=BF16, xs=hs, ws=ds)
    O.close(y, want, e)


@pytest.mark.gpu
def test_layer_half_trains_as_its_formula():
    """norm with residual -> gated product -> product with residual, forward and
    backward through all three at once, against 64 bits.  Bound: five roundings
    to 16 bits lie between an input and an output or a gradient (half a step
    each, 2^-9 of the value on average, 2^-8 at most), so 5 * 2^-8 of the norm."""
    m, d, f = 150, 96, 264
    a, x = randn(m, d, seed=1), randn(m, d, seed=2)
    w = (1 + randn(d, seed=3, dtype=torch.float32, std=0.1)).to(BF16)
    wg, wu, wd = randn(f, d, seed=4, std=d ** -0.5), randn(f, d, seed=5, std=d ** -0.5), randn(d, f, seed=6, std=f ** -0.5)
    dy = randn(m, d, seed=7)
    leaves = [t.requires_grad_() for t in (a, x, w, wg, wu, wd)]
    n, s = norm.rms_norm(a, w, residual=x)
    y = dense.linear(dense.gated_linear(n, wg, wu), wd, residual=s)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    l64 = [t.detach().double().requires_grad_() for t in leaves]
    s64 = l64[0] + l64[1]
    n64 = s64 / (s64.square().mean(-1, keepdim=True) + 1e-5).sqrt() * l64[2]
    y64 = (torch.nn.functional.silu(n64 @ l64[3].t()) * (n64 @ l64[4].t())) @ l64[5].t() + s64
    want = [y64, *torch.autograd.grad(y64, l64, dy.double())]
    for p, q in zip(got, want):
        assert (p.double() - q).norm() <= 5 * 2.0 ** -8 * q.norm()


@pytest.mark.gpu
def test_trainer_steps_a_fused_model():
    code = """
import torch, torch.distributed as dist
from mini_nangila_b200.models import GPT2, GPT2Config, Llama, LlamaConfig
from mini_nangila_b200.train import DDPTrainer, init_distributed
from mini_nangila_b200.ops import dense
init_distributed("nccl")
for M, cfg in ((GPT2, GPT2Config.tiny()), (Llama, LlamaConfig.tiny())):
    cfg.fused_ops = True
    tr = DDPTrainer(M(cfg), hook="fused", overlap_optimizer=True)
    before = {n: p.detach().clone() for n, p in tr.model.named_parameters()}
    t = torch.randint(0, 512, (4, 49), device="cuda")
    for _ in range(3):
        loss = tr.step(t[:, :-1].contiguous(), t[:, 1:].contiguous())
    assert torch.isfinite(loss) and tr.kernel_launches() > 0
    assert all(torch.isfinite(p).all() for p in tr.model.parameters())
    assert all(not torch.equal(before[n], p) for n, p in tr.model.named_parameters())
    dense.check()
dist.destroy_process_group()
print("ok")
"""
    env = {k: v for k, v in os.environ.items() if k not in ("MASTER_PORT", "RANK", "WORLD_SIZE", "LOCAL_RANK")}
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


@pytest.mark.gpu
def test_captured_decode_replays_with_new_inputs():
    d, f = 256, 520
    w = randn(d, seed=1)
    wg, wu, wd = randn(f, d, seed=2, std=0.06), randn(f, d, seed=3, std=0.06), randn(d, f, seed=4, std=0.04)
    for rows in (1, 7, 40):
        a, x = randn(rows, d, seed=5), randn(rows, d, seed=6)

        def step():
            n, s = norm.rms_norm(a, w, residual=x)
            return dense.linear(dense.gated_linear(n, wg, wu), wd, residual=s)

        with torch.no_grad():
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            for seed in (10, 11):
                a.copy_(randn(rows, d, seed=seed))
                x.copy_(randn(rows, d, seed=seed + 5))
                graph.replay()
                assert torch.equal(out, step())
    dense.check()


CAPTURE = """
import sys, torch, torch.nn.functional as F
from mini_nangila_b200.ops import dense, norm
ours, where = sys.argv[1] == "ours", sys.argv[2]
torch.manual_seed(0)
bf = torch.bfloat16
leaves = [t.to("cuda", bf).requires_grad_() for t in
          (torch.randn(64, 96), torch.ones(96), torch.randn(200, 96) * .1, torch.randn(200, 96) * .1,
           torch.randn(96, 200) * .1, torch.randn(96) * .1)]
x, w, g, u, d, b = leaves
dy = torch.randn(64, 96, device="cuda").to(bf)
def fwd():
    if not ours:
        n = F.rms_norm(x + x, (96,), w)
        return F.linear(F.silu(F.linear(n, g)) * F.linear(n, u), d, b) + x
    n, s = norm.rms_norm(x, w, residual=x)
    return dense.linear(dense.gated_linear(n, g, u), d, b, activation="gelu", residual=s)
def grads():
    return torch.autograd.grad(fwd(), leaves, dy)
want = grads()
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    for _ in range(2): grads()
torch.cuda.current_stream().wait_stream(side)
alive = None
if where == "default":
    alive = fwd()
elif where == "side":
    with torch.cuda.stream(side):
        alive = fwd()
    torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        got = grads()
    graph.replay(); graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    print("captured")
except RuntimeError as e:
    print("raised")
torch.cuda.synchronize()
if alive is not None:
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(alive, leaves, dy), want))
assert all(torch.equal(p, q) for p, q in zip(grads(), want))
dense.check()
print("lives")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["none", "side", "default"])
def test_captured_training_beside_a_live_eager_graph(where):
    """A forward and backward pass captured while an eager graph of the same
    leaves is alive, each in a process of its own: what happens is what happens
    with stock layers (on the default stream the capture raises: its leaves'
    gradients belong to that stream), and the process goes on with right results."""
    said = []
    for kind in ("stock", "ours"):
        r = subprocess.run([sys.executable, "-c", CAPTURE, kind, where], cwd=ROOT, capture_output=True, text=True,
                           timeout=300)
        assert r.returncode == 0, (kind, r.stdout[-500:], r.stderr[-2000:])
        said.append(r.stdout.split())
    assert said[0] == said[1] and said[1][-1] == "lives"
    assert said[1][0] == "captured" or where == "default"


@pytest.mark.gpu
def test_two_streams_and_two_graphs_share_nothing():
    """Products whose k is split (they have workspaces) on two streams at once,
    and as two graphs replayed at once, give what they give alone."""
    sets = [(randn(8192, 64, seed=s).requires_grad_(), randn(72, 64, seed=s + 1).requires_grad_(),
             randn(8192, 72, seed=s + 2)) for s in (20, 30)]

    def grads(i):
        x, w, dy = sets[i]
        return torch.autograd.grad(dense.linear(x, w, activation="silu"), [x, w], dy)

    want = [grads(i) for i in (0, 1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = grads(i)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(p, q) for p, q in zip(got[i], want[i]))
    graphs, outs = [], []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(grads(i))
        graphs.append(g)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(p, q) for p, q in zip(outs[i], want[i]))


@pytest.mark.gpu
def test_outputs_are_ready_for_stock_kernels():
    """Kernels start before the one in front ends: what follows, stock or not,
    still sees whole results."""
    w = randn(128, 128, seed=1, std=0.09)

    def chain(x, wait):
        for _ in range(10):
            x = dense.linear(x, w, activation="relu")
            if wait:
                torch.cuda.synchronize()
            x = x + 0.5
            if wait:
                torch.cuda.synchronize()
            x = dense.linear(x, w)
            if wait:
                torch.cuda.synchronize()
        return x

    for rows in (3, 300):
        x = randn(rows, 128, seed=2)
        want = chain(x, True)
        for _ in range(20):
            assert torch.equal(chain(x, False), want)


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_work_that_forks_and_joins_over_streams(captured):
    """An operator behind an event of another stream waits for that stream's
    kernels, stock ones and its own kind, run as they come and from a graph."""
    w = randn(512, 512, seed=1, std=0.04)
    big = randn(4096, 512, seed=2)
    small = randn(4, 512, seed=3)
    s = randn(512, seed=4)
    side = torch.cuda.Stream()

    def work(fork):
        main = torch.cuda.current_stream()
        a = big
        for _ in range(4):  # long enough to be running when the other stream starts
            a = dense.linear(a, w, activation="relu") + 0.25
        e = torch.cuda.Event()
        e.record(main)
        with torch.cuda.stream(side if fork else main):
            torch.cuda.current_stream().wait_event(e)
            b = dense.linear(a[-4:], w, residual=small)
            b = norm.rms_norm(b, s)
            f = torch.cuda.Event()
            f.record(torch.cuda.current_stream())
        c = dense.gated_linear(a, w, w)
        main.wait_event(f)
        return dense.linear(b, w, residual=c[-4:]), b, c

    with torch.no_grad():
        torch.cuda.synchronize()
        want = work(False)
        torch.cuda.synchronize()
        if not captured:
            for _ in range(10):
                got = work(True)
                torch.cuda.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(got, want))
            return
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = work(True)
        for _ in range(10):
            for t in got:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
def test_autocast_types():
    x, w, b = randn(40, 64, seed=1, dtype=torch.float32), randn(24, 64, seed=2, dtype=torch.float32), \
        randn(24, seed=3, dtype=torch.float32)
    for t in (BF16, torch.float16):
        leaves = [v.clone().requires_grad_() for v in (x, w, b)]
        with torch.autocast("cuda", dtype=t):
            y = dense.linear(*leaves)
            h = dense.gated_linear(leaves[0], leaves[1], leaves[1])
            z = dense.linear(*leaves, residual=randn(40, 24, seed=4, dtype=torch.float32))
        assert y.dtype == h.dtype == t and z.dtype == torch.float32
        (y.float().sum() + h.float().sum() + z.sum()).backward()
        assert all(v.grad.dtype == torch.float32 and torch.isfinite(v.grad).all() for v in leaves)
        with torch.no_grad(), torch.autocast("cuda", dtype=t):
            assert torch.equal(dense.linear(*leaves), dense.linear(x.to(t), w.to(t), b.to(t)))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x, w = randn(40, 64, seed=1).requires_grad_(), randn(24, 64, seed=2).requires_grad_()
    s = randn(64, seed=3).requires_grad_()
    for y in (dense.linear(x, w, activation="silu"), dense.gated_linear(x, w, w), norm.rms_norm(x, s)):
        (g,) = torch.autograd.grad(y.float().square().sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            g.float().sum().backward()


@pytest.mark.gpu
def test_saved_inputs_may_not_change():
    x, w = randn(40, 64, seed=1).requires_grad_(), randn(24, 64, seed=2).requires_grad_()
    y = dense.linear(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_less_usual_calls():
    """Views of 8-bit rows, fp32 outputs, expanded and strided vectors, one
    dimension, inference mode, recomputation, one tensor in two places."""
    for rows in (5, 60):
        big, bs = norm.quantize_rows(randn(2 * rows, 160, seed=1))
        w8, ws = norm.quantize_rows(randn(48, 160, seed=2, std=0.08))
        for x8, xs, w in ((big[::2], bs[::2], w8), (big[:rows, 3:99], bs[:rows, None], w8[:, 3:99])):
            y, e, _, _ = O.linear(x8.float(), w.float(), xs=xs.flatten(), ws=ws, out=torch.float32)
            O.close(dense.linear(x8, w, x_scale=xs, w_scale=ws, out_dtype=torch.float32), y, e)
        x, w = randn(rows, 96, seed=3), randn(40, 96, seed=4, std=0.1)
        y, e, _, _ = O.linear(x, w, out=torch.float32)
        O.close(dense.linear(x, w, out_dtype=torch.float32), y, e)
        h, e, _ = O.gated(x, w, w, "silu", out=torch.float32)
        O.close(dense.gated_linear(x, w, w, out_dtype=torch.float32), h, e)
        b = randn(1, seed=5).expand(40)
        O.close(dense.linear(x, w, b), *O.linear(x, w, b)[:2])
        b = randn(80, seed=6)[::2]
        O.close(dense.linear(x, w, b), *O.linear(x, w, b)[:2])
        with torch.inference_mode():
            assert torch.equal(dense.linear(x, w, b), dense.linear(x.clone(), w, b))
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        plain = torch.autograd.grad(dense.gated_linear(xl, wl, wl).sum(), [xl, wl])
        again = torch.autograd.grad(
            torch.utils.checkpoint.checkpoint(dense.gated_linear, xl, wl, wl, use_reentrant=False).sum(), [xl, wl])
        assert all(torch.equal(p, q) for p, q in zip(plain, again))
        sq = randn(rows, rows, seed=7).requires_grad_()
        (g,) = torch.autograd.grad(dense.linear(sq, sq).sum(), [sq])
        v = sq.detach().double()
        want = v.sum(0)[None].expand(rows, rows)  # of the first operand, and the same of the second
        bound = 2 * ((rows + 8) * 2.0 ** -23 * v.abs().sum(0)[None] + 2.0 ** -9 * want.abs()) + 2.0 ** -8 * 2 * want.abs()
        O.close(g, 2 * want, bound.expand(rows, rows) + 1e-30)
    v = randn(96, seed=8)
    assert dense.linear(v, w).shape == (40,) and torch.equal(dense.linear(v, w), dense.linear(v[None], w)[0])
    codes, scale = norm.rms_norm_fp8(v, torch.ones_like(v))
    assert codes.shape == (96,) and scale.shape == ()
    assert norm.rms_norm(v, torch.ones_like(v)).shape == (96,)


@pytest.mark.gpu
@pytest.mark.parametrize("cg,nb,splits", [(c, n, s) for c in (1, 2) for n in (128, 256) for s in (1, 3)])
def test_every_plan(cg, nb, splits):
    """Each tile shape, with and without pieces of k, over all operand orders and
    epilogues, at sizes no tile divides."""
    m, k, n = 413, 840, 296
    x, w, b = randn(m, k, seed=1), randn(n, k, seed=2, std=k ** -0.5), randn(n, seed=3)
    wu, r, dy = randn(n, k, seed=4, std=k ** -0.5), randn(m, n, seed=5), randn(m, n, seed=6)
    _ext.cuda().dense_force_plan(cg, nb, splits)
    try:
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        y = dense.linear(*leaves[:3], activation="gelu", residual=leaves[3])
        g1 = torch.autograd.grad(y, leaves, dy)
        gl = [t.clone().requires_grad_() for t in (x, w, wu)]
        h = dense.gated_linear(*gl)
        g2 = torch.autograd.grad(h, gl, dy)
        wide = dense.linear(x[:, :839], w[:, :839], residual=r.float())  # rows that no 16 bytes divide
        x8, xs = norm.quantize_rows(x)
        w8, ws = norm.quantize_rows(w)
        y8 = dense.linear(x8, w8, b, x_scale=xs, w_scale=ws, activation="silu")
    finally:
        _ext.cuda().dense_force_plan(0, 0, 0)
    want, e, z, ez = O.linear(x, w, b, "gelu", r)
    O.close(y, want, e)
    for g, (v, e), name in zip(g1, O.linear_grads(dy, x, w, z, ez, "gelu", True), "xwb"):
        O.close(g, v, e, name)
    want, e, pre = O.gated(x, w, wu, "silu")
    O.close(h, want, e)
    for g, (v, e), name in zip(g2, O.gated_grads(dy, x, w, wu, "silu", pre), ("x", "gate", "up")):
        O.close(g, v, e, name)
    O.close(wide, *O.linear(x[:, :839], w[:, :839], r=r.float(), out=torch.float32)[:2])
    O.close(y8, *O.linear(x8.float(), w8.float(), b, "silu", out=BF16, xs=xs, ws=ws)[:2])
    dense.check()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Outputs and rows of more than 2^31 elements: first, middle and last rows."""
    m, k, n = 70001, 64, 32008
    x, w = randn(m, k, seed=1), randn(n, k, seed=2, std=0.1)
    rows = torch.tensor([0, 1, 33333, 67100, m - 2, m - 1], device="cuda")
    y = dense.linear(x, w)
    assert y.numel() > 2 ** 31
    O.close(y[rows], *O.linear(x[rows], w)[:2])
    del y
    dy = torch.empty(m, n, device="cuda", dtype=BF16)
    dy[:] = randn(1, n, seed=3)
    dx, dw = torch.autograd.grad(dense.linear(x.requires_grad_(), w.requires_grad_()), [x, w], dy)
    with torch.no_grad():
        want, e = O.product(dy[:1], w.t())
        O.close(dx[rows], want.expand(len(rows), k), (e + O.half_step(want, BF16)).expand(len(rows), k))
        want = dy[0].double()[:, None] * x.double().sum(0)[None]
        e = (m + 8) * 2.0 ** -23 * dy[0].double().abs()[:, None] * x.double().abs().sum(0)[None]
        O.close(dw, want, e + O.half_step(want, BF16) * 1.01)
    del dy, dx, dw
    torch.cuda.empty_cache()
    rows, width = 1_050_003, 2048
    a = torch.empty(rows, width, device="cuda", dtype=BF16)
    a[:] = randn(1, width, seed=4)
    a[-1] = randn(width, seed=5)
    s = randn(width, seed=6)
    at = torch.tensor([0, rows // 2, rows - 2, rows - 1], device="cuda")
    out = norm.rms_norm(a, s)
    y, u, _ = O.rms_norm(a[at], s, 1e-5)
    O.close(out[at], y, u * y.abs() + O.half_step(y, BF16) * 1.01)
