"""Llama-style decoder in stock PyTorch: RMSNorm, rotary position embedding,
grouped-query attention, SwiGLU FFN.  ``LlamaConfig.b1_1()`` is the 1.1B
configuration (22 layers, d_model 2048, 32 heads, 4 KV heads, FFN 5632,
vocab 32000, context 2048).

``LlamaConfig(fused_ops=True)`` runs each layer's norms, gated feed-forward
block and down projection on this framework's kernels (``ops.norm``,
``ops.dense``): 16-bit operands (a 16-bit model, or ``torch.autocast``), CUDA
only.  ``Llama.quantize_weights`` then adds an 8-bit form of every projection
for evaluation: in evaluation mode, under ``torch.no_grad``.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import dense, norm


@dataclass
class LlamaConfig:
    """Llama-style dimensions; ``b1_1()`` is the 1.1B model (22 layers, d 2048, 32 heads, 4 KV heads)."""
    vocab_size: int = 32000
    max_seq: int = 2048
    n_layer: int = 22
    n_head: int = 32
    n_kv_head: int = 4
    d_model: int = 2048
    d_ff: int = 5632
    rope_theta: float = 10000.0
    eps: float = 1e-5
    init_std: float = 0.02
    fused_ops: bool = False

    @staticmethod
    def b1_1() -> "LlamaConfig":
        return LlamaConfig()

    @staticmethod
    def tiny() -> "LlamaConfig":
        return LlamaConfig(vocab_size=512, max_seq=64, n_layer=2, n_head=4, n_kv_head=2, d_model=64, d_ff=172)


class RMSNorm(nn.Module):
    def __init__(self, d: int, eps: float):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(d))

    def forward(self, x):
        xf = x.float()
        return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)).to(x.dtype) * self.weight


def half_type(x: torch.Tensor) -> torch.dtype | None:
    """The 16-bit type that the fused ops compute in for a float32 stream
    (autocast's); None where the stream itself has 16 bits."""
    return torch.get_autocast_dtype("cuda") if x.dtype == torch.float32 and torch.is_autocast_enabled("cuda") else None


def _state(w: torch.Tensor) -> tuple[int, int]:
    """What an update in place or other memory changes (inference tensors count no updates)."""
    return w.data_ptr(), 0 if w.is_inference() else w._version


def rope_tables(seq: int, hd: int, theta: float, device) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 1.0 / (theta ** (torch.arange(0, hd, 2, device=device, dtype=torch.float32) / hd))
    t = torch.arange(seq, device=device, dtype=torch.float32)
    f = torch.outer(t, inv)
    return f.cos(), f.sin()


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    # x: (B, H, T, D); rotate pairs (even, odd) halves
    d = x.shape[-1] // 2
    x1, x2 = x[..., :d], x[..., d:]
    c = cos[None, None, : x.shape[2]].to(x.dtype)
    s = sin[None, None, : x.shape[2]].to(x.dtype)
    return torch.cat([x1 * c - x2 * s, x1 * s + x2 * c], dim=-1)


class Attention(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.h, self.kvh = cfg.n_head, cfg.n_kv_head
        self.hd = cfg.d_model // cfg.n_head
        self.q = nn.Linear(cfg.d_model, cfg.n_head * self.hd, bias=False)
        self.k = nn.Linear(cfg.d_model, cfg.n_kv_head * self.hd, bias=False)
        self.v = nn.Linear(cfg.d_model, cfg.n_kv_head * self.hd, bias=False)
        self.o = nn.Linear(cfg.n_head * self.hd, cfg.d_model, bias=False)

    def mix(self, q, k, v, cos, sin):
        """Attention of the projections [batch, tokens, heads * head_dim]."""
        B, T, _ = q.shape
        q = q.view(B, T, self.h, self.hd).transpose(1, 2)
        k = k.view(B, T, self.kvh, self.hd).transpose(1, 2)
        v = v.view(B, T, self.kvh, self.hd).transpose(1, 2)
        q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
        return y.transpose(1, 2).reshape(B, T, self.h * self.hd)

    def forward(self, x, cos, sin):
        return self.o(self.mix(self.q(x), self.k(x), self.v(x), cos, sin))


class SwiGLU(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.gate = nn.Linear(cfg.d_model, cfg.d_ff, bias=False)
        self.up = nn.Linear(cfg.d_model, cfg.d_ff, bias=False)
        self.down = nn.Linear(cfg.d_ff, cfg.d_model, bias=False)

    def forward(self, x):
        return self.down(F.silu(self.gate(x)) * self.up(x))


class Layer(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.n1 = RMSNorm(cfg.d_model, cfg.eps)
        self.attn = Attention(cfg)
        self.n2 = RMSNorm(cfg.d_model, cfg.eps)
        self.ffn = SwiGLU(cfg)
        self.fused_ops = cfg.fused_ops
        self.w8 = None  # 8-bit weights: {projection: (codes, scale)}
        self._w8_of = ()  # and the state of the weights that they were made from

    def forward(self, x, cos, sin):
        if not self.fused_ops:
            x = x + self.attn(self.n1(x), cos, sin)
            return x + self.ffn(self.n2(x))
        # Not in training, where a recomputed layer runs forward without gradients.
        if self.w8 is not None and not self.training and not torch.is_grad_enabled():
            if any(p.get("weight") is not w or _state(w) != was for p, w, was in self._w8_of):
                raise RuntimeError("weights have changed since quantize_weights(); call it again")
            return self._forward_8bit(x, cos, sin)
        a = self.attn(norm.rms_norm(x, self.n1.weight, self.n1.eps, out_dtype=half_type(x)), cos, sin)
        n, x = norm.rms_norm(a, self.n2.weight, self.n2.eps, residual=x)
        h = dense.gated_linear(n, self.ffn.gate.weight, self.ffn.up.weight)
        return dense.linear(h, self.ffn.down.weight, residual=x)

    def quantize_weights(self) -> None:
        a, f = self.attn, self.ffn
        of = dict(q=a.q, k=a.k, v=a.v, o=a.o, gate=f.gate, up=f.up, down=f.down)
        self.w8 = {n: norm.quantize_rows(m.weight) for n, m in of.items()}
        self._w8_of = [(m._parameters, m.weight, _state(m.weight)) for m in of.values()]

    def _forward_8bit(self, x, cos, sin):
        t = x.dtype if x.dtype != torch.float32 else half_type(x) or torch.bfloat16

        def project(name, codes, scale, **kw):
            w, ws = self.w8[name]
            return dense.linear(codes, w, x_scale=scale, w_scale=ws, **kw)

        n, s = norm.rms_norm_fp8(x, self.n1.weight, self.n1.eps)
        y = self.attn.mix(*(project(p, n, s, out_dtype=t) for p in "qkv"), cos, sin)
        a = project("o", *norm.quantize_rows(y), out_dtype=t)
        n, s, x = norm.rms_norm_fp8(a, self.n2.weight, self.n2.eps, residual=x)
        (g, gs), (u, us) = self.w8["gate"], self.w8["up"]
        h = dense.gated_linear(n, g, u, x_scale=s, gate_scale=gs, up_scale=us, out_dtype=t)
        return project("down", *norm.quantize_rows(h), residual=x)


class Llama(nn.Module):
    """Llama-style decoder (RMSNorm, RoPE, grouped-query attention, SwiGLU); ``forward(x, y)`` returns the loss."""
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.cfg = cfg
        self.emb = nn.Embedding(cfg.vocab_size, cfg.d_model)
        self.layers = nn.ModuleList([Layer(cfg) for _ in range(cfg.n_layer)])
        self.norm = RMSNorm(cfg.d_model, cfg.eps)
        self.head = nn.Linear(cfg.d_model, cfg.vocab_size, bias=False)
        for m in self.modules():
            if isinstance(m, (nn.Linear, nn.Embedding)):
                nn.init.normal_(m.weight, mean=0.0, std=cfg.init_std)
        self._rope = None

    def forward(self, idx, targets=None):
        B, T = idx.shape
        if self._rope is None or self._rope[0].device != idx.device or self._rope[0].shape[0] < T:
            self._rope = rope_tables(max(T, self.cfg.max_seq), self.cfg.d_model // self.cfg.n_head,
                                     self.cfg.rope_theta, idx.device)
        cos, sin = self._rope
        x = self.emb(idx)
        for layer in self.layers:
            x = layer(x, cos, sin)
        logits = self.head(norm.rms_norm(x, self.norm.weight, self.norm.eps, out_dtype=half_type(x))
                           if self.cfg.fused_ops else self.norm(x))
        if targets is None:
            return logits
        return F.cross_entropy(logits.reshape(-1, logits.size(-1)).float(), targets.reshape(-1))

    def quantize_weights(self) -> "Llama":
        """Lay every layer's projections out in 8 bits (e4m3, one scale an output
        feature) beside the 16-bit ones, and go into evaluation mode; needs
        ``fused_ops`` and a model on its GPU.  Calls in evaluation mode under
        ``torch.no_grad`` use them from then on.  Once a weight has changed
        (an optimizer's step, ``load_state_dict``, another device or type) such
        calls raise until this is called again."""
        if not self.cfg.fused_ops:
            raise ValueError("quantize_weights needs LlamaConfig(fused_ops=True)")
        with torch.no_grad():
            for layer in self.layers:
                layer.quantize_weights()
        return self.eval()

    def num_params(self) -> int:
        return sum(p.numel() for p in self.parameters())
