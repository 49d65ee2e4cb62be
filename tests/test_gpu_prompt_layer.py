"""GPU tests of the prompt path's operators together: prompt_layer.PromptLayer.

Every stage of the layer against its plain form on the stage's own input (a 4-bit rounding turns differences of a bf16
step upstream into differences of a code, so comparing ends alone would say little), and the layer against its stages bit
for bit. Tolerance of a stage, relative in the 2-norm: each bf16 rounding inside it is at most 2^-8 of a value, in the
2-norm about 2^-9.2; norm, SwiGLU and residual round up to three times: 2^-7; rope, attention (two roundings, measured
against sums of magnitudes elsewhere) and products (one): 2^-7 as well.
"""
from __future__ import annotations

import pytest
import torch

from lynnreal_omni_b200 import kernels as K
from lynnreal_omni_b200.attention import attention_packed
from lynnreal_omni_b200.fp4 import dequantize_rows_fp4
from lynnreal_omni_b200.prompt_layer import PromptLayer, pack
from lynnreal_omni_b200.rotary import rope, rope_frequencies
from test_gpu_attention_packed import reference as attention_reference
from test_gpu_fp4 import definition, scale_values
from test_gpu_rope import reference as rope_reference

DEV = "cuda"


def fake_quantized(x, format):
    value, raw, row = definition(x.bfloat16().cpu(), format)
    s = scale_values(raw, format).float() * (row if row is not None else 1.0)
    return (value.float().unflatten(1, (s.shape[1], -1)) * s[..., None]).flatten(1).to(x.device)


def weight(layer):
    return dequantize_rows_fp4(layer.weight_codes, layer.weight_scales, layer.weight_scale, format=layer.format).float()


def near(got, want):
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    assert float((got.double() - want.double()).norm()) <= 2.0 ** -7 * float(want.double().norm())
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("lengths", [[1], [3, 70, 1, 200], [0, 40]])
def test_layer_stage_by_stage(lengths, format):
    h, hk, d = 4, 2, 64
    layer = PromptLayer.random(hidden=256, heads=h, kv_heads=hk, inner=512, head_dim=d, format=format)
    prompts = pack(lengths)
    inv_freq, factor = rope_frequencies(d, scaling="yarn", factor=2.0)
    x0 = torch.randn(sum(lengths), 256, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)

    def norm(x, n):
        f = x.float()
        want = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + n.eps) * n.weight.float()
        return near(K._rms_adaln(x, n, None, None, 0, 0), want)

    def project(linear, x):
        return near(linear(x), fake_quantized(x, format) @ weight(linear).t())

    qkv = project(layer.qkv, norm(x0, layer.norm1))
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], 1))
    turned = rope(q, k, prompts.positions, inv_freq, factor=factor)
    q, k = (near(got, rope_reference(t, prompts.positions, inv_freq, False, factor)[0].to(DEV)) for got, t in zip(turned, (q, k)))
    context = near(attention_packed(q, k, v, prompts.cu_seqlens),
                   attention_reference(q, k, v, lengths, lengths, True, d ** -0.5)[0])
    update = project(layer.out, context.flatten(1))
    x1 = near(K._gated_residual(x0, update, None, None, 0), x0.float() + update.float())
    up = project(layer.gate_up, norm(x1, layer.norm2))
    value, gate = up.float().chunk(2, 1)
    inner = near(K._swiglu(up), value * torch.nn.functional.silu(gate))
    update = project(layer.down, inner)
    x2 = near(K._gated_residual(x1, update, None, None, 0), x1.float() + update.float())
    assert torch.equal(layer(x0, prompts, inv_freq, factor), x2)


@pytest.mark.gpu
def test_prompts_do_not_see_each_other():
    layer = PromptLayer.random(hidden=512, heads=8, kv_heads=2, inner=1024)
    inv_freq, _ = rope_frequencies(128)
    x = torch.randn(300, 512, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    first = layer(x, pack([140, 160]), inv_freq)
    y = x.clone()
    y[140:] = 1.0
    assert torch.equal(layer(y, pack([140, 160]), inv_freq)[:140], first[:140])


def test_pack():
    cu, positions = pack([2, 0, 3], "cpu")
    assert cu.tolist() == [0, 2, 2, 5] and positions.tolist() == [0, 1, 0, 1, 2]
    assert cu.dtype == positions.dtype == torch.int32
    with pytest.raises(ValueError):
        pack([], "cpu")
