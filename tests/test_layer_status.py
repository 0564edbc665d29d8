"""A product that gave up a wait is reported without being asked: by the next
product, and by the trainer before its next step and with its last one."""
import os
import socket

import pytest
import torch

from mini_nangila_b200 import _ext, train
from mini_nangila_b200.models import GPT2, GPT2Config
from mini_nangila_b200.ops import dense


class FakeExtension:
    """An extension whose kernels on device 1 have given up with `code`."""

    def __init__(self, code):
        self.code = code

    def dense_gave_up(self, device):
        return self.code if device == 1 else 0


def test_poll_raises_for_its_device(monkeypatch):
    monkeypatch.setattr(_ext, "_cuda", FakeExtension(5))
    dense.poll(0)
    dense.poll(torch.device("cuda", 0))
    for device in (1, torch.device("cuda", 1)):
        with pytest.raises(dense.DenseError, match="cuda:1 .*status 5"):
            dense.poll(device)
    monkeypatch.setattr(_ext, "_cuda", None)  # nothing was loaded, so nothing ran
    dense.poll(1)


def test_trainer_notices(monkeypatch):
    import torch.distributed as dist

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(s.getsockname()[1]))
    dist.init_process_group("gloo", rank=0, world_size=1)
    try:
        cfg = GPT2Config.tiny()
        tr = train.DDPTrainer(GPT2(cfg), hook="nccl", device=torch.device("cpu"))
        t = torch.randint(0, cfg.vocab_size, (2, 17))
        batch = (t[:, :-1].contiguous(), t[:, 1:].contiguous())
        asked = []

        def poll(device):
            asked.append((device, tr.steps_done))
            if fail[0] is not None and tr.steps_done >= fail[0]:
                raise dense.DenseError("a product gave up")

        monkeypatch.setattr(train.dense, "poll", poll)
        fail = [None]
        tr.step_host(*batch)
        assert not asked  # no device, no products
        monkeypatch.setattr(tr, "_products_on", torch.device("cuda", 0))
        fail[0] = 1
        before = [p.detach().clone() for p in tr.model.parameters()]
        with pytest.raises(dense.DenseError):  # in front of the step's first launch
            tr.step(*batch)
        assert tr.steps_done == 1 and all(torch.equal(p, q) for p, q in zip(before, tr.model.parameters()))
        fail[0] = 2
        with pytest.raises(dense.DenseError):  # the step that failed itself, once its loss is here
            tr.step_host(*batch)
        assert tr.steps_done == 2
        fail[0] = 4
        with pytest.raises(dense.DenseError):
            tr.train_steps([batch] * 2)
        assert tr.steps_done == 4
        fail[0] = 5
        with pytest.raises(dense.DenseError):
            tr.fit(lambda i: batch, 1)
        assert tr.steps_done == 5 and asked[-1] == (torch.device("cuda", 0), 5)
    finally:
        dist.destroy_process_group()


@pytest.mark.gpu
def test_the_next_product_raises():
    """The status words' copy in host memory is written here as a kernel that
    gave up writes it."""
    x, w = torch.randn(40, 64, device="cuda").bfloat16(), torch.randn(24, 64, device="cuda").bfloat16()
    xl = x.clone().requires_grad_()
    y = dense.linear(xl, w)
    h = dense.gated_linear(xl, w, w)
    torch.cuda.synchronize()
    dense.poll()
    words = _ext.cuda().dense_status_words(torch.cuda.current_device())
    assert words.tolist() == [0, 0, 0, 0]
    words[0], words[1] = 5, 7
    try:
        for call in (lambda: dense.linear(x, w), lambda: dense.linear(x[:2], w), lambda: dense.gated_linear(x, w, w),
                     lambda: y.sum().backward(retain_graph=True), lambda: h.sum().backward(retain_graph=True),
                     dense.poll):
            with pytest.raises(dense.DenseError, match="gave up"):
                call()
        with pytest.raises(dense.DenseError, match="gave up"):
            dense.check()  # reports it for the last time
    finally:
        words.zero_()
    dense.check()
    dense.poll()
    assert torch.equal(dense.linear(x, w), y.detach())
    y.sum().backward()


@pytest.mark.gpu
def test_first_product_of_a_process_may_be_captured():
    code = """
import torch
from mini_nangila_b200.ops import dense
x, w = torch.randn(40, 64, device="cuda").bfloat16(), torch.randn(24, 64, device="cuda").bfloat16()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = dense.linear(x, w)
g.replay()
torch.cuda.synchronize()
assert torch.equal(y, dense.linear(x, w))
dense.check()
print("ok")
"""
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]
