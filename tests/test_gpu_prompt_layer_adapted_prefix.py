"""GPU tests of PromptLayer.read_prefix with an adapter: the text as the adapted model reads it."""
from __future__ import annotations

import pytest
import torch

from lynnreal_omni_b200 import kernels as K
from lynnreal_omni_b200.adapters import token_adapters
from lynnreal_omni_b200.prompt_layer import PromptLayer, pack
from lynnreal_omni_b200.rotary import rope, rope_frequencies
from test_gpu_prompt_layer_shared import D, HEADS, HIDDEN, KV_HEADS, adapted_layer, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 300, 700])
def test_prefix_read_with_an_adapter(tokens):
    """Its keys and values are those of the adapted projections, and what it hands on is what the layer makes of the same text."""
    layer = adapted_layer([4, 16, 8])
    inv_freq, factor = rope_frequencies(D)
    text, index = rows(tokens, 5), token_adapters([1], [tokens])
    after, (key, value) = layer.read_prefix(text, inv_freq, factor, index=index)
    assert torch.equal(after, layer(text, pack([tokens]), inv_freq, factor, index=index))
    qkv = layer.qkv(K._rms_adaln(text, layer.norm1, None, None, 0, 0), index)
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([HEADS * D, KV_HEADS * D, KV_HEADS * D], 1))
    _, k = rope(q, k, pack([tokens]).positions, inv_freq, factor=factor)
    assert torch.equal(key, k) and torch.equal(value, v)
    _, (bare, _) = layer.read_prefix(text, inv_freq, factor)
    assert not torch.equal(bare, key)


def test_refusal():
    layer = PromptLayer.random(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, inner=512, head_dim=D)
    inv_freq, _ = rope_frequencies(D)
    with pytest.raises(ValueError, match="no projection has any"):
        layer.read_prefix(rows(5, 1), inv_freq, index=token_adapters([0], [5]))
