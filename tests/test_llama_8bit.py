"""When a Llama layer takes its 8-bit weights: in evaluation mode without
gradients, and only while they are those of its present weights."""
import copy

import pytest
import torch
import torch.utils.checkpoint

from mini_nangila_b200.models import Llama, LlamaConfig
from mini_nangila_b200.models import llama as L
from mini_nangila_b200.train import BucketAdamW

BF16 = torch.bfloat16


@pytest.fixture
def model(monkeypatch):
    """A model on the CPU whose layers say which way they went."""
    monkeypatch.setattr(L.norm, "quantize_rows", lambda w: (w.detach().clone(), w.detach()[:, 0].float()))
    monkeypatch.setattr(L.Layer, "_forward_8bit", lambda self, x, cos, sin: "8 bits")
    monkeypatch.setattr(L.norm, "rms_norm", lambda *a, **k: (_ for _ in ()).throw(KeyError("16 bits")))
    torch.manual_seed(0)
    return Llama(LlamaConfig(vocab_size=32, n_layer=1, n_head=2, n_kv_head=1, d_model=16, d_ff=24, max_seq=8,
                             fused_ops=True)).to(BF16)


def way(m):
    try:
        return m.layers[0](torch.zeros(1, 4, 16, dtype=BF16), None, None)
    except KeyError as e:
        return e.args[0]


def test_8_bits_are_for_evaluation(model):
    with torch.no_grad():
        assert way(model) == "16 bits"
        assert model.quantize_weights() is model and not model.training  # ready for evaluation
        assert way(model) == "8 bits"
        model.train()  # a forward pass of training may run without gradients: recomputation does
        assert way(model) == "16 bits"
        model.eval()
        assert way(model) == "8 bits"
    assert way(model) == "16 bits"  # gradients
    with torch.inference_mode():
        assert way(model) == "8 bits"


def changes():
    def step(m):
        o = torch.optim.SGD(m.parameters(), lr=0.1)
        for p in m.parameters():
            p.grad = torch.ones_like(p)
        o.step()

    def bucket_kernel(m):  # the exchange kernel updates parameters through their addresses
        b = BucketAdamW(torch.optim.AdamW(m.parameters()))
        b._pending = {"t": 0, "steps": [torch.zeros(())], "params": list(m.parameters())}
        b.kernel_done(None)

    def other_parameter(m):
        m.layers[0].ffn.up.weight = torch.nn.Parameter(torch.zeros_like(m.layers[0].ffn.up.weight))

    def other_data(m):
        m.layers[0].attn.k.weight.data = torch.zeros_like(m.layers[0].attn.k.weight)

    return {"optimizer": step, "optimizer in the exchange kernel": bucket_kernel,
            "load_state_dict": lambda m: m.load_state_dict(copy.deepcopy(m.state_dict())),
            "load_state_dict, assigned": lambda m: m.load_state_dict(copy.deepcopy(m.state_dict()), assign=True),
            "in place": lambda m: m.layers[0].attn.o.weight.detach().mul_(2), "type": lambda m: m.half(),
            "parameter": other_parameter, "data": other_data}


@pytest.mark.parametrize("change", changes())
def test_weights_that_changed_are_noticed(model, change):
    model.quantize_weights()
    with torch.no_grad():
        assert way(model) == "8 bits"
    changes()[change](model)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="quantize_weights"):
            way(model)
        model.quantize_weights()
        assert way(model) == "8 bits"


def test_other_weights_may_change(model):
    """Norms and embeddings have no 8-bit form."""
    model.quantize_weights()
    with torch.no_grad():
        model.emb.weight.mul_(2)
        model.layers[0].n1.weight.mul_(2)
        assert way(model) == "8 bits"


@pytest.mark.gpu
def test_recomputation_in_training_is_of_16_bits():
    """Reentrant checkpointing runs a layer's forward pass without gradients: the
    loss and the gradients are those without checkpointing."""
    cfg = LlamaConfig.tiny()
    cfg.fused_ops = True
    torch.manual_seed(0)
    m = Llama(cfg).to("cuda", BF16).quantize_weights().train()
    t = torch.randint(0, cfg.vocab_size, (2, 33), device="cuda")

    def run():
        m.zero_grad()
        loss = m(t[:, :-1].contiguous(), t[:, 1:].contiguous())
        loss.backward()
        return [loss.detach(), *(p.grad.clone() for p in m.parameters())]

    want = run()
    for layer in m.layers:
        layer.forward = (lambda f: lambda x, cos, sin: torch.utils.checkpoint.checkpoint(
            f, x, cos, sin, use_reentrant=True))(layer.forward)
    assert all(torch.equal(p, q) for p, q in zip(run(), want))


@pytest.mark.gpu
def test_8bit_evaluation_follows_the_weights():
    cfg = LlamaConfig.tiny()
    cfg.fused_ops = True
    torch.manual_seed(0)
    m = Llama(cfg).to("cuda", BF16).quantize_weights()
    t = torch.randint(0, cfg.vocab_size, (2, 32), device="cuda")
    with torch.no_grad():
        before = m(t)
        for layer in m.layers:
            layer.ffn.down.weight.mul_(1.5)
        with pytest.raises(RuntimeError, match="quantize_weights"):
            m(t)
        assert not torch.equal(m.quantize_weights()(t), before)
