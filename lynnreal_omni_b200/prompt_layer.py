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

Prompts that all continue one text (an instruction, a template) share its keys and values, and each request may have
low-rank adapters of its own on the projections (``AdaptedLinear`` in place of ``Fp4Linear``):

    prefixes = []
    for layer in layers:                              # once for all batches behind this text
        t, kv = layer.read_prefix(t, inv_freq, factor)  # index=: as the model with an adapter reads it
        prefixes.append(kv)
    plan = pack([len(p) for p in prompts], "cuda", start=len(text))
    index = token_adapters(adapter_of_each_prompt, [len(p) for p in prompts], "cuda")
    for layer, kv in zip(layers, prefixes):
        x = layer(x, plan, inv_freq, factor, prefix=kv, index=index)
"""
from __future__ import annotations

from types import SimpleNamespace
from typing import NamedTuple

import torch

from . import kernels as K
from .adapters import AdaptedLinear
from .attention import attention_packed, attention_shared
from .fp4 import Fp4Linear
from .rotary import rope

__all__ = ["PackedPrompts", "pack", "PromptLayer"]


class PackedPrompts(NamedTuple):
    cu_seqlens: torch.Tensor  # int32 [prompts + 1]
    positions: torch.Tensor   # int32 [tokens], from `start` in each prompt


def pack(lengths, device="cuda", *, start: int = 0) -> PackedPrompts:
    """Offsets and positions of prompts of these lengths, one after another; ``start``: the first token's position in
    each (the length of a shared prefix)."""
    if not lengths or min(lengths) < 0:
        raise ValueError("pack: expected the lengths of one or more prompts")
    if start < 0:
        raise ValueError("pack: start must not be negative")
    if start + max(lengths) > 2 ** 31:
        raise ValueError(f"pack: positions from {start} on do not fit 32 bits")
    n = torch.tensor(lengths, dtype=torch.int64)
    cu = torch.cat((torch.zeros(1, dtype=torch.int64), n.cumsum(0)))
    positions = torch.arange(int(cu[-1])) - torch.repeat_interleave(cu[:-1], n) + start
    return PackedPrompts(cu.to(device=device, dtype=torch.int32), positions.to(device=device, dtype=torch.int32))


class PromptLayer:
    """One layer. qkv, out, gate_up, down: ``Fp4Linear``, or ``AdaptedLinear`` on one; norm weights bf16 [hidden];
    ``gate_up`` gives the SwiGLU's value and gate halves side by side as ``kernels._swiglu`` takes them."""

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

    def __call__(self, x: torch.Tensor, prompts: PackedPrompts, inv_freq: torch.Tensor, factor: float = 1.0, *, prefix=None,
                 index: torch.Tensor | None = None) -> torch.Tensor:
        """bf16 [tokens, hidden] -> the same. prefix: the (keys, values) that ``read_prefix`` gave, in front of every prompt;
        index: int32 [tokens], each token's adapter on the ``AdaptedLinear`` projections (None: they go without)."""
        cu = prompts.cu_seqlens
        if prefix is None:
            return self._run(x, prompts.positions, inv_freq, factor, lambda q, k, v: attention_packed(q, k, v, cu), index)
        return self._run(x, prompts.positions, inv_freq, factor, lambda q, k, v: attention_shared(q, k, v, *prefix, cu), index)

    def read_prefix(self, x: torch.Tensor, inv_freq: torch.Tensor, factor: float = 1.0, *, index: torch.Tensor | None = None):
        """One text on its own: bf16 [tokens, hidden] -> (the same for the next layer, (keys, values) bf16 [tokens, kv_heads, D] for the
        prompts that continue it). index: int32 [tokens], the adapter that reads the text (None: it is read without one, and prompts
        with adapters of their own then see the keys and values of the model without them). A text that several adapters are to read is
        read once for each, and their prompts are called apart."""
        kept = []

        def attend(q, k, v):
            kept.extend((k, v.contiguous()))  # rope's keys are a tensor of their own; the values a view of the projection
            return attention_packed(q, k, v, prompts.cu_seqlens)

        prompts = pack([x.shape[0]], x.device)
        return self._run(x, prompts.positions, inv_freq, factor, attend, index), tuple(kept)

    def _run(self, x, positions, inv_freq, factor, attend, index):
        if index is not None and not any(isinstance(p, AdaptedLinear) for p in (self.qkv, self.out, self.gate_up, self.down)):
            raise ValueError("PromptLayer: adapters are given, but no projection has any")

        def project(linear, rows):
            return linear(rows, index) if isinstance(linear, AdaptedLinear) else linear(rows)

        h, hk, d = self.heads, self.kv_heads, self.head_dim
        qkv = project(self.qkv, K._rms_adaln(x, self.norm1, None, None, 0, 0))
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], 1))
        q, k = rope(q, k, positions, inv_freq, factor=factor)
        context = attend(q, k, v)
        x = K._gated_residual(x, project(self.out, context.flatten(1)), None, None, 0)
        inner = K._swiglu(project(self.gate_up, K._rms_adaln(x, self.norm2, None, None, 0, 0)))
        return K._gated_residual(x, project(self.down, inner), None, None, 0)
