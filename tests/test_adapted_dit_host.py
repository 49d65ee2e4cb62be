"""CPU tests: DiT blocks, which pass no adapter numbers, refuse projections that would then silently go without their adapters."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from torch import nn

from lynnreal_omni_b200 import elementwise_fusion, fusion
from lynnreal_omni_b200.adapters import AdaptedLinear

HIDDEN = 64


def linear(n, k):
    return nn.Linear(k, n, bias=False, dtype=torch.bfloat16)


class _Attn(nn.Module):
    def __init__(self, fused):
        super().__init__()
        self.heads, self.fused_projections = 1, fused
        if fused:
            self.to_qkv = linear(3 * HIDDEN, HIDDEN)
        else:
            self.to_qkv, self.to_q, self.to_k, self.to_v = None, *(linear(HIDDEN, HIDDEN) for _ in range(3))
        self.to_out = nn.ModuleList([linear(HIDDEN, HIDDEN), nn.Dropout(0.0)])

    def set_processor(self, processor):
        self.processor = processor

    def forward(self, hidden_states, rotary_emb=None, attention_mask=None):
        raise AssertionError("the block ran")


class _Up(nn.Module):
    def __init__(self):
        super().__init__()
        self.proj = linear(4 * HIDDEN, HIDDEN)


def block_of(fused):
    block = nn.Module()
    block.attn = _Attn(fused)
    block.ff = nn.Module()
    block.ff.net = nn.ModuleList([_Up(), nn.Dropout(0.0), linear(HIDDEN, 2 * HIDDEN)])
    block.norm1 = block.norm2 = lambda x: x
    return block


PLACES = {"attn.to_qkv": True, "attn.to_q": False, "attn.to_v": False, "attn.to_out.0": True, "ff.net.0.proj": True, "ff.net.2": True}


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("kind", ["fused", "fused_quant", "elementwise"])
def test_adapted_projections_are_refused(kind, place):
    block = block_of(PLACES[place])
    transformer = SimpleNamespace(transformer_blocks=[block], modules=block.modules, training=False)
    if kind == "elementwise":
        elementwise_fusion.enable_elementwise_fusion(transformer)
    else:
        fusion.enable_fusion(transformer, fused_quant=kind == "fused_quant")
    owner, name = block.get_submodule(place.rpartition(".")[0]), place.rpartition(".")[2]
    base = block.get_submodule(place)
    adapter = torch.zeros(8, base.in_features), torch.zeros(base.out_features, 8), 1.0
    owner._modules[name] = AdaptedLinear.stack(base, [adapter])
    x, table = torch.zeros(1, 3, HIDDEN, dtype=torch.bfloat16), torch.zeros(1, 6 * HIDDEN, dtype=torch.bfloat16)
    block._lynnreal_adaln_cache, block._lynnreal_cache_key = {0: table}, SimpleNamespace(current=0)
    rotary = (torch.zeros(3, HIDDEN), torch.zeros(3, HIDDEN))
    with pytest.raises(ValueError, match="adapter"):
        block.forward(x, None, torch.zeros(3, dtype=torch.int64), rotary)


def test_an_output_projection_without_a_list_runs():
    """The element-wise blocks keep their native attention, whatever it holds."""
    block = block_of(True)
    block.attn.to_out = linear(HIDDEN, HIDDEN)
    elementwise_fusion.enable_elementwise_fusion(SimpleNamespace(transformer_blocks=[block], training=False))
    table = torch.zeros(1, 6 * HIDDEN, dtype=torch.bfloat16)
    block._lynnreal_adaln_cache, block._lynnreal_cache_key = {0: table}, SimpleNamespace(current=0)
    args = torch.zeros(1, 3, HIDDEN, dtype=torch.bfloat16), None, torch.zeros(3, dtype=torch.int64), None
    with pytest.raises(AssertionError, match="the block ran"):
        block.forward(*args)
    block.attn.to_out = AdaptedLinear.stack(block.attn.to_out, [(torch.zeros(8, HIDDEN), torch.zeros(HIDDEN, 8), 1.0)])
    with pytest.raises(ValueError, match="adapter"):
        block.forward(*args)
