"""A decoder layer over packed prompts on 4-bit projections: the operators of the prompt path together.

A text context is made from prompts of different lengths. ``PromptLayer`` runs one layer of such an encoder on their
tokens packed one after another, without padding: RMSNorm -> 4-bit query/key/value projection -> rotary positions ->
causal attention with grouped heads -> 4-bit output projection + residual -> RMSNorm -> 4-bit SwiGLU feed-forward +
residual. Norms, SwiGLU and residuals are the kernels of the W8A8 path.

    layer = PromptLayer.random(hidden=4096, heads=32, kv_heads=8, inner=12288, device="cuda")
    x = embeddings                                    # bf16 [tokens of all prompts, hidden]
    plan = pack([len(p) for p in prompts], "cuda")    # offsets and positions, made once for all layers
    for layer in layers:
        x = layer(x, plan, inv_freq, factor)
"""
from __future__ import annotations

from types import SimpleNamespace
from typing import NamedTuple

import torch

from . import kernels as K
from .attention import attention_packed
from .fp4 import Fp4Linear
from .rotary import rope

__all__ = ["PackedPrompts", "pack", "PromptLayer"]


class PackedPrompts(NamedTuple):
    cu_seqlens: torch.Tensor  # int32 [prompts + 1]
    positions: torch.Tensor   # int32 [tokens], from 0 in each prompt


def pack(lengths, device="cuda") -> PackedPrompts:
    """Offsets and positions of prompts of these lengths, one after another."""
    if not lengths or min(lengths) < 0:
        raise ValueError("pack: expected the lengths of one or more prompts")
    n = torch.tensor(lengths, dtype=torch.int64)
    cu = torch.cat((torch.zeros(1, dtype=torch.int64), n.cumsum(0)))
    positions = torch.arange(int(cu[-1])) - torch.repeat_interleave(cu[:-1], n)
    return PackedPrompts(cu.to(device=device, dtype=torch.int32), positions.to(device=device, dtype=torch.int32))


class PromptLayer:
    """One layer. qkv, out, gate_up, down: ``Fp4Linear``; norm weights bf16 [hidden]; ``gate_up`` gives the SwiGLU's
    value and gate halves side by side as ``kernels._swiglu`` takes them."""

    def __init__(self, qkv: Fp4Linear, out: Fp4Linear, gate_up: Fp4Linear, down: Fp4Linear, norm1: torch.Tensor,
                 norm2: torch.Tensor, *, heads: int, kv_heads: int, eps: float = 1e-6):
        self.head_dim, rest = divmod(qkv.out_features, heads + 2 * kv_heads)
        if rest or out.in_features != heads * self.head_dim or down.in_features * 2 != gate_up.out_features:
            raise ValueError("PromptLayer: the projections' sizes do not fit the heads or each other")
        self.qkv, self.out, self.gate_up, self.down = qkv, out, gate_up, down
        self.norm1, self.norm2 = (SimpleNamespace(weight=w, eps=eps) for w in (norm1, norm2))
        self.heads, self.kv_heads = heads, kv_heads

    @classmethod
    def random(cls, *, hidden: int, heads: int, kv_heads: int, inner: int, head_dim: int = 128, format: str = "nvfp4",
               seed: int = 0, device="cuda") -> "PromptLayer":
        """Random-init weights, quantised to ``format``."""
        g = torch.Generator(device=device).manual_seed(seed)

        def linear(n, k):
            layer = torch.nn.Linear(k, n, bias=False, device=device, dtype=torch.bfloat16)
            with torch.no_grad():
                layer.weight.copy_(torch.randn(n, k, generator=g, device=device) * k ** -0.5)
            return Fp4Linear(layer, format=format)

        def norm():
            return (1 + 0.05 * torch.randn(hidden, generator=g, device=device)).to(torch.bfloat16)

        return cls(linear((heads + 2 * kv_heads) * head_dim, hidden), linear(hidden, heads * head_dim),
                   linear(2 * inner, hidden), linear(hidden, inner), norm(), norm(), heads=heads, kv_heads=kv_heads)

    def __call__(self, x: torch.Tensor, prompts: PackedPrompts, inv_freq: torch.Tensor, factor: float = 1.0) -> torch.Tensor:
        """bf16 [tokens, hidden] -> the same."""
        h, hk, d = self.heads, self.kv_heads, self.head_dim
        qkv = self.qkv(K._rms_adaln(x, self.norm1, None, None, 0, 0))
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], 1))
        q, k = rope(q, k, prompts.positions, inv_freq, factor=factor)
        context = attention_packed(q, k, v, prompts.cu_seqlens)
        x = K._gated_residual(x, self.out(context.flatten(1)), None, None, 0)
        inner = K._swiglu(self.gate_up(K._rms_adaln(x, self.norm2, None, None, 0, 0)))
        return K._gated_residual(x, self.down(inner), None, None, 0)
