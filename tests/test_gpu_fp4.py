"""GPU tests of the 4-bit floating-point rows: quantisation, its inverse and the product.

Quantisation is compared bit for bit with its fp32 definition evaluated on the CPU, and with the values in 64 bits by
the half-step bound. The product's reference is the 64-bit product of the decoded values; the tolerance is the bf16
rounding (2^-8 |ref| covers it and its double-rounding) plus fp32 accumulation: 2^-20 of the sum of magnitudes (K / 64
partial sums, each off by a few units of 2^-24).
"""
from __future__ import annotations

import math

import pytest
import torch

from lynnreal_omni_b200.fp4 import Fp4Linear, dequantize_rows_fp4, fp4_matmul, quantize_rows_fp4, tile_scales

pytestmark = pytest.mark.gpu
DEV = "cuda"
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def activations(rows, width, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g)
    x[:, torch.rand(width, generator=g) < 0.01] *= 20
    return x.bfloat16()


def untile(scales, rows, blocks):
    out = torch.zeros(rows, blocks, dtype=torch.uint8)
    s = scales.cpu()
    for r in range(rows):
        for b in range(blocks):
            out[r, b] = s[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]
    return out


def scale_values(raw, format):
    """Scale bytes -> values in 64 bits."""
    raw = raw.int()
    if format == "mxfp4":
        v = torch.ldexp(torch.ones(raw.shape, dtype=torch.float64), raw - 127)
        return torch.where(raw == 255, math.nan, v)
    e, m = raw >> 3 & 15, (raw & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, torch.ldexp(8 + m, e - 10))
    return torch.where((raw & 127) == 127, math.nan, v)


def decode(codes, scales, format):
    """Packed rows -> (values without the row scale, block scales) in 64 bits."""
    c = codes.cpu()
    v = GRID[torch.stack((c & 15, c >> 4), -1).flatten(1).long()]
    block = BLOCK[format]
    s = scale_values(untile(scales, v.shape[0], v.shape[1] // block), format)
    return (v.unflatten(1, (-1, block)) * s[..., None]).flatten(1), s


def definition(x, format):
    """(code values, scale bytes, row scales) of the fp32 definition."""
    x = x.float()
    row = x.abs().amax(1, keepdim=True)
    row = torch.where(row < 1e-8, torch.tensor(1e-8), row)
    if format == "nvfp4":
        big = torch.where(row > 2.0 ** 110, 2.0 ** -20, 1.0)  # exact; keeps 448 max and e A finite
        x, row = x * big, row * big
        b = x.unflatten(1, (-1, 16))
        stored = (b.abs().amax(2) * 448 / row).to(torch.float8_e4m3fn)
        raw, e = stored.view(torch.uint8), stored.float()
        inv = torch.where(e == 0, torch.tensor(0.0), torch.tensor(2688.0) / (e * row))
        row_scale = (row / big) * torch.tensor(1 / 2688, dtype=torch.float32)
    else:
        b = x.unflatten(1, (-1, 32))
        ex = (b.abs().amax(2).view(torch.int32) >> 23).clamp(min=0)
        raw = (ex - 2).clamp(min=0).to(torch.uint8)
        inv, row_scale = torch.ldexp(torch.ones(raw.shape), 127 - raw.int()), None
    a = (b * inv[..., None]).double()
    m = a.abs().clamp(max=6.0)
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    return torch.copysign(torch.round(m / step) * step, a).flatten(1), raw, row_scale


@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,width", [(1, 32), (3, 96), (129, 544), (33, 1056), (5, 2048), (2, 4128), (7, 6144),
                                        (2, 8192), (1, 16384), (2, 24576), (3, 32800)])
def test_quantize_matches_the_definition(rows, width, format):
    x = activations(rows, width, rows + width)
    codes, scales, row_scale = quantize_rows_fp4(x.to(DEV), format=format)
    value, raw, row = definition(x, format)
    c = codes.cpu()
    got = GRID[torch.stack((c & 15, c >> 4), -1).flatten(1).long()]
    blocks = width // BLOCK[format]
    assert torch.equal(untile(scales, rows, blocks), raw)
    assert torch.equal(got, value) and torch.equal(torch.signbit(got), torch.signbit(value))
    assert (row_scale is None and row is None) or torch.equal(row_scale.cpu(), row)
    # blocks past the row are zeros
    if blocks % 4:
        assert not bool(scales.cpu()[0, -1, 0, 0, blocks % 4:].any())
    # half a step of e2m1 (1 between 4 and 6), or the saturation at 6 (mxfp4: up to 8; nvfp4: the scale's rounding)
    decoded, s = decode(codes, scales, format)
    if row is not None:
        decoded = decoded * row.double()
        s = s * row.double()
    most = 2.0 if format == "mxfp4" else 1.0
    floor = 0 if format == "mxfp4" else x.double().abs().amax(1, keepdim=True) * 2.0 ** -10 / 448 * 6
    assert bool(((x.double() - decoded).abs() <= (most * s.repeat_interleave(BLOCK[format], 1)) * 1.0001 + floor).all())
    # and back, rounded once to bf16
    back = dequantize_rows_fp4(codes, scales, row_scale, format=format)
    scale32 = scale_values(raw, format).float() * (row if row is not None else 1.0)
    expected = (value.float().unflatten(1, (blocks, -1)) * scale32[..., None]).flatten(1).bfloat16()
    assert torch.equal(back.cpu(), expected)


@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
def test_quantize_ties_extremes_and_zeros(format):
    ties = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -0.0] * 2)
    rows = torch.stack([ties, ties * 2.0 ** 100, ties * 2.0 ** -100, ties * 2.0 ** 125, torch.zeros(32),
                        torch.full((32,), 2.0 ** -133), torch.cat((ties[:16], ties[16:] * 2.0 ** -14))]).bfloat16()
    codes, scales, row_scale = quantize_rows_fp4(rows.to(DEV), format=format)
    value, raw, row = definition(rows, format)
    c = codes.cpu()
    assert torch.equal(GRID[torch.stack((c & 15, c >> 4), -1).flatten(1).long()], value)
    assert torch.equal(untile(scales, rows.shape[0], 32 // BLOCK[format]), raw)


@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_non_finite_rows_stay_visible_and_apart(format, bad):
    x = activations(5, 128, 3)
    clean = fp4_product(x, format)
    x[2, 70] = bad
    y = fp4_product(x, format)
    assert bool(torch.isnan(y[2]).all())
    keep = [0, 1, 3, 4]
    assert torch.equal(y[keep], clean[keep])


def fp4_product(x, format):
    w = activations(40, x.shape[1], 9)
    a, b = quantize_rows_fp4(x.to(DEV), format=format), quantize_rows_fp4(w.to(DEV), format=format)
    return fp4_matmul(a[0], a[1], b[0], b[1], a[2], b[2], format=format).cpu()


def test_quantize_strided_rows():
    x = activations(9, 256, 4).to(DEV)
    for view in (x[:, 32:160], x[::2, 64:], x.t().contiguous().t(), x[:, 1:129], x[3:4, 32:96]):
        for got, want in zip(quantize_rows_fp4(view), quantize_rows_fp4(view.contiguous().clone())):
            if got.ndim == 5:
                blocks = view.shape[1] // 16
                assert torch.equal(untile(got, view.shape[0], blocks), untile(want, view.shape[0], blocks))
            else:
                assert torch.equal(got, want)


def product_case(m, n, k, format, seed, scales=True, bias=True):
    g = torch.Generator().manual_seed(seed)
    block = BLOCK[format]
    ops = []
    for rows in (m, n):
        codes = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
        low, high = (40, 90) if format == "nvfp4" else (118, 128)
        raw = torch.randint(low, high, (rows, k // block), generator=g, dtype=torch.uint8)
        ops += [codes.to(DEV), tile_scales(raw.to(DEV))]
    rs = (torch.rand(m, generator=g) + 0.5).to(DEV) if scales else None
    cs = (torch.rand(n, generator=g) + 0.5).to(DEV) if scales else None
    b = torch.randn(n, generator=g).bfloat16().to(DEV) if bias else None
    return ops, rs, cs, b


def check_product(m, n, k, format, seed=0, scales=True, bias=True):
    ops, rs, cs, b = product_case(m, n, k, format, seed, scales, bias)
    got = fp4_matmul(*ops, rs, cs, b, format=format).double().cpu()
    va, vb = decode(ops[0], ops[1], format)[0], decode(ops[2], ops[3], format)[0]
    ref, size = va @ vb.t(), va.abs() @ vb.abs().t()
    if rs is not None:
        f = rs.double().cpu()[:, None] * cs.double().cpu()
        ref, size = ref * f, size * f
    if b is not None:
        ref = ref + b.double().cpu()
    assert got.shape == (m, n)
    bound = 2.0 ** -8 * ref.abs() + 2.0 ** -20 * size
    err = (got - ref).abs()
    assert bool((err <= bound).all()), (m, n, k, float((err / bound).max()), (err > bound).nonzero()[:4].tolist())


@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 200, 64), (3, 129, 96), (17, 192, 256), (64, 193, 288), (65, 384, 512),
                                   (127, 64, 1024), (128, 128, 128), (129, 576, 320), (200, 1000, 160), (257, 40, 2080),
                                   (300, 777, 544), (1, 4099, 1056), (33, 640, 4096), (513, 385, 256), (1500, 12000, 96),
                                   (1300, 12003, 544)])
def test_product(m, n, k, format):
    check_product(m, n, k, format, seed=m + n + k)


@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
def test_product_without_scales_or_bias(format):
    check_product(70, 300, 224, format, scales=False, bias=False)
    check_product(5, 300, 224, format, scales=False, bias=False)


@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
def test_every_code_and_scale_position(format):
    """One code and one scale at a time: identity-like operands show each value of B in its own place."""
    block, k, n = BLOCK[format], 512, 256
    g = torch.Generator().manual_seed(5)
    b_codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    one, low, high = (0x38, 8, 126) if format == "nvfp4" else (127, 64, 190)
    b_raw = torch.randint(low, high, (n, k // block), generator=g, dtype=torch.uint8)
    a_codes = torch.zeros(k, k // 2, dtype=torch.uint8)
    i = torch.arange(k)
    a_codes[i, i // 2] = torch.where(i % 2 == 0, 0x02, 0x20).to(torch.uint8)  # 1.0 at (i, i)
    a_raw = torch.full((k, k // block), one, dtype=torch.uint8)
    b_scales = tile_scales(b_raw.to(DEV))
    got = fp4_matmul(a_codes.to(DEV), tile_scales(a_raw.to(DEV)), b_codes.to(DEV), b_scales, format=format).cpu()
    assert torch.equal(got, decode(b_codes, b_scales, format)[0].t().bfloat16())
    few = fp4_matmul(a_codes[:5].to(DEV), tile_scales(a_raw[:5].to(DEV)), b_codes.to(DEV), b_scales, format=format).cpu()
    assert torch.equal(few, got[:5])


def test_product_ignores_what_lies_past_the_rows():
    """NaN scales in the tiles' unused rows reach no result."""
    ops, rs, cs, b = product_case(5, 70, 96, "nvfp4", 3)
    clean = fp4_matmul(*ops, rs, cs, b)
    for scales, rows in ((ops[1], 5), (ops[3], 70)):
        flat = scales.permute(0, 3, 2, 1, 4).reshape(128, -1).clone()
        flat[rows:] = 0x7F
        scales.copy_(flat.reshape(1, 4, 32, -1, 4).permute(0, 3, 2, 1, 4))
    assert torch.equal(fp4_matmul(*ops, rs, cs, b), clean)


def test_product_repeats_bit_for_bit():
    ops, rs, cs, b = product_case(3, 1024, 6144, "nvfp4", 8)
    first = fp4_matmul(*ops, rs, cs, b)
    assert all(torch.equal(fp4_matmul(*ops, rs, cs, b), first) for _ in range(5))


def test_empty_rows():
    q = quantize_rows_fp4(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16))
    w = quantize_rows_fp4(activations(8, 64, 1).to(DEV))
    assert fp4_matmul(q[0], q[1], w[0], w[1], q[2], w[2]).shape == (0, 8)
    assert dequantize_rows_fp4(*q).shape == (0, 64)


@pytest.mark.parametrize("format", ["nvfp4", "mxfp4"])
def test_linear_layer(format):
    """The layer against the same layer in 64 bits: the 4-bit rounding of both sides is within a step of 1/4 each."""
    torch.manual_seed(0)
    linear = torch.nn.Linear(256, 72).bfloat16().to(DEV)
    layer = Fp4Linear(linear, format=format)
    x = torch.randn(2, 11, 256, device=DEV).bfloat16()
    y, want = layer(x), linear.double()(x.double())
    assert y.shape == (2, 11, 72) and y.dtype == torch.bfloat16
    # each value is off by at most a sixth (nvfp4) or a quarter (mxfp4, saturation) and the errors are independent:
    # about 0.1 of each side's norm, 0.3 of the product's at the outside
    assert float((y.double() - want).norm() / want.norm()) < 0.3
    packed = Fp4Linear.from_packed(layer.weight_codes, layer.weight_scales, layer.weight_scale, layer.bias, format=format)
    assert torch.equal(packed(x), y)


def test_refusals():
    x = activations(4, 64, 0).to(DEV)
    codes, scales, rs = quantize_rows_fp4(x)
    with pytest.raises(ValueError, match="format"):
        quantize_rows_fp4(x, format="fp4")
    with pytest.raises(ValueError, match="multiple of 32"):
        quantize_rows_fp4(x[:, :48])
    with pytest.raises(ValueError, match="bf16"):
        quantize_rows_fp4(x.float())
    with pytest.raises(ValueError, match="CUDA"):
        quantize_rows_fp4(x.cpu())
    with pytest.raises(ValueError, match="scales must be"):
        fp4_matmul(codes, scales[:, :0], codes, scales)
    with pytest.raises(ValueError, match="alike"):
        fp4_matmul(codes, scales, *quantize_rows_fp4(activations(4, 128, 0).to(DEV))[:2])
    with pytest.raises(ValueError, match="row_scale"):
        fp4_matmul(codes, scales, codes, scales, rs[:3])
    with pytest.raises(ValueError, match="bias"):
        fp4_matmul(codes, scales, codes, scales, bias=rs)
    with pytest.raises(ValueError, match="uint8"):
        dequantize_rows_fp4(codes.int(), scales)
    with pytest.raises(ValueError, match="1-byte"):
        tile_scales(rs)
