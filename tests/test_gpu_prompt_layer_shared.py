"""GPU tests of a prompt layer behind a shared prefix with adapters: the operators together, as a server runs them.

The layer is compared bit for bit with its stages called one by one (each operator has tests of its own against 64 bits), and
requests with themselves in other company.
"""
from __future__ import annotations

import pytest
import torch

from lynnreal_omni_b200 import kernels as K
from lynnreal_omni_b200.adapters import AdaptedLinear, add_adapters, token_adapters
from lynnreal_omni_b200.attention import attention_packed, attention_shared
from lynnreal_omni_b200.prompt_layer import PromptLayer, pack
from lynnreal_omni_b200.rotary import rope, rope_frequencies

DEV = "cuda"
HIDDEN, HEADS, KV_HEADS, D = 512, 8, 2, 64


def adapted_layer(ranks, seed=0, inner=512):
    layer = PromptLayer.random(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, inner=inner, head_dim=D, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    for name in ("qkv", "out", "gate_up", "down"):
        base = getattr(layer, name)
        parts = [(torch.randn(r, base.in_features, generator=g).bfloat16().to(DEV) * base.in_features ** -0.5,
                  torch.randn(base.out_features, r, generator=g).bfloat16().to(DEV) * r ** -0.5, 0.5) for r in ranks]
        setattr(layer, name, AdaptedLinear.stack(base, parts))
    return layer


def rows(count, seed):
    return torch.randn(count, HIDDEN, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)


def stage_by_stage(layer, x0, plan, inv_freq, factor, prefix, index):
    def project(linear, x):
        return add_adapters(linear.base(x), x, linear.down, linear.up, index, linear.scale)

    qkv = project(layer.qkv, K._rms_adaln(x0, layer.norm1, None, None, 0, 0))
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([HEADS * D, KV_HEADS * D, KV_HEADS * D], 1))
    q, k = rope(q, k, plan.positions, inv_freq, factor=factor)
    x1 = K._gated_residual(x0, project(layer.out, attention_shared(q, k, v, *prefix, plan.cu_seqlens).flatten(1)), None, None, 0)
    inner = K._swiglu(project(layer.gate_up, K._rms_adaln(x1, layer.norm2, None, None, 0, 0)))
    return K._gated_residual(x1, project(layer.down, inner), None, None, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1], [1] * 40, [3, 70, 1, 200], [0, 40], [700]], ids=str)
def test_layer_stage_by_stage(lengths):
    layer = adapted_layer([4, 16, 8])
    inv_freq, factor = rope_frequencies(D)
    text = rows(333, 5)
    after, prefix = layer.read_prefix(text, inv_freq, factor)
    assert torch.equal(after, layer(text, pack([333]), inv_freq, factor))
    assert [t.shape for t in prefix] == [(333, KV_HEADS, D)] * 2
    plan = pack(lengths, start=333)
    index = token_adapters([None if i % 4 == 3 else i % 4 for i in range(len(lengths))], lengths)
    x = rows(sum(lengths), 6)
    got = layer(x, plan, inv_freq, factor, prefix=prefix, index=index)
    assert torch.equal(got, stage_by_stage(layer, x, plan, inv_freq, factor, prefix, index))
    assert torch.isfinite(got).all()


@pytest.mark.gpu
def test_keys_of_the_prefix_are_those_of_its_own_run():
    """The last tokens of a text, once as a request behind the rest of it: the same keys, values and attention."""
    layer = PromptLayer.random(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, inner=512, head_dim=D)
    inv_freq, factor = rope_frequencies(D)
    text = rows(300, 7)
    _, whole = layer.read_prefix(text, inv_freq, factor)
    _, front = layer.read_prefix(text[:260], inv_freq, factor)
    assert all(torch.equal(f, w[:260]) for f, w in zip(front, whole))
    qkv = layer.qkv(K._rms_adaln(text, layer.norm1, None, None, 0, 0))
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([HEADS * D, KV_HEADS * D, KV_HEADS * D], 1))
    q, k = rope(q, k, pack([300]).positions, inv_freq, factor=factor)
    assert torch.equal(k, whole[0]) and torch.equal(v, whole[1])
    behind = attention_shared(q[260:], k[260:], v[260:], *front, pack([40]).cu_seqlens)
    alone = attention_packed(q, k, v, pack([300]).cu_seqlens)[260:]
    # two orders of the same sums over bf16 probabilities
    assert float((behind.double() - alone.double()).norm()) <= 2.0 ** -7 * float(alone.double().norm())


@pytest.mark.gpu
def test_requests_do_not_see_each_other():
    layer = adapted_layer([16, 16])
    inv_freq, _ = rope_frequencies(D)
    _, prefix = layer.read_prefix(rows(100, 8), inv_freq)
    plan, lengths = pack([140, 160], start=100), [140, 160]
    x = rows(300, 9)
    first = layer(x, plan, inv_freq, prefix=prefix, index=token_adapters([0, 1], lengths))
    y = x.clone()
    y[140:] = 1.0
    again = layer(y, plan, inv_freq, prefix=prefix, index=token_adapters([0, None], lengths))
    assert torch.equal(again[:140], first[:140])
    none = layer(x, plan, inv_freq, prefix=prefix, index=token_adapters([None, None], lengths))
    assert torch.equal(none, layer(x, plan, inv_freq, prefix=prefix)) and not torch.equal(none[:140], first[:140])


@pytest.mark.gpu
def test_captured_step():
    """One token a request, captured once: later steps bring other tokens, positions and adapters."""
    layer = adapted_layer([8, 8, 8])
    inv_freq, _ = rope_frequencies(D)
    _, prefix = layer.read_prefix(rows(200, 10), inv_freq)
    plan = pack([1] * 20, start=200)
    x, index = rows(20, 11), token_adapters([0] * 20, [1] * 20)
    layer(x, plan, inv_freq, prefix=prefix, index=index)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, plan, inv_freq, prefix=prefix, index=index)
    for seed in range(3):
        x.copy_(rows(20, 20 + seed))
        index.copy_(token_adapters([(i * seed + seed) % 3 if i % 5 else None for i in range(20)], [1] * 20))
        plan.positions.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(x, plan, inv_freq, prefix=prefix, index=index))


@pytest.mark.gpu
def test_refusals():
    layer = PromptLayer.random(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, inner=512, head_dim=D)
    inv_freq, _ = rope_frequencies(D)
    x, plan = rows(5, 1), pack([5])
    with pytest.raises(ValueError, match="no projection has any"):
        layer(x, plan, inv_freq, index=token_adapters([0], [5]))
    key = torch.zeros(9, KV_HEADS + 1, D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="disagree"):
        layer(x, plan, inv_freq, prefix=(key, key))


def test_pack_behind_a_prefix():
    cu, positions = pack([2, 0, 3], "cpu", start=7)
    assert cu.tolist() == [0, 2, 2, 5] and positions.tolist() == [7, 8, 7, 8, 9]
    with pytest.raises(ValueError):
        pack([2], "cpu", start=-1)
