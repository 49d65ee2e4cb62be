"""GPU tests of rotary.rope against the rotation in 64 bits.

Tolerance: one bf16 rounding of the result (eight significant bits: half a unit is up to 2^-8 of the
value) plus the angle's error (sincospi of turns within 2^-23, that is 2 pi 2^-23 < 1e-6 radians; 2e-6 is allowed for the fp32 products) times the pair's magnitude.
"""
from __future__ import annotations

import math
from decimal import Decimal, localcontext

import pytest
import torch

from lynnreal_omni_b200.rotary import rope, rope_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda"


PI2 = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def far_angles(positions, inv_freq):
    """p f less its whole turns, in 60 digits: 64 bits keep no 1e-6 of an angle of 1e10 radians."""
    with localcontext() as c:
        c.prec = 60
        return torch.tensor([[float((Decimal(p) * Decimal(f)) % PI2) for f in inv_freq.tolist()]
                             for p in positions.tolist()], dtype=torch.float64)


def reference(x, positions, inv_freq, interleaved, factor, angle=None):
    """(rotated values, magnitude of each value's pair) in 64 bits on the CPU."""
    x = x.double().cpu()
    if angle is None:
        angle = torch.outer(positions.double().cpu().reshape(-1), inv_freq.double().cpu())
    c, s = angle.cos() * factor, angle.sin() * factor
    r = 2 * inv_freq.numel()
    flat = x.reshape(-1, x.shape[-2], x.shape[-1])
    out, size = flat.clone(), flat.abs()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = flat[..., first], flat[..., second]
    out[..., first] = a * c[:, None] - b * s[:, None]
    out[..., second] = b * c[:, None] + a * s[:, None]
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * factor
    return out.reshape(x.shape), size.reshape(x.shape)


def close(got, ref):
    ref, size = ref
    err = (got.double().cpu() - ref).abs()
    bound = 2.0 ** -8 * ref.abs() * 1.001 + 2e-6 * size + 1e-38
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv_heads,d,rotary", [(32, 8, 128, 128), (4, 1, 128, 64), (3, 3, 96, 96), (2, 1, 64, 24),
                                                     (5, 1, 80, 20), (1, 1, 7, 6), (2, 2, 16, 2), (1, 1, 2050, 2050)])
@pytest.mark.parametrize("tokens", [1, 5, 1300])
def test_rope(tokens, heads, kv_heads, d, rotary, interleaved):
    if d > 1000 and tokens > 5:
        tokens = 1190  # one token a block at that width, enough blocks to fill the GPU
    g = torch.Generator().manual_seed(tokens + d)
    q = torch.randn(tokens, heads, d, generator=g).bfloat16().to(DEV)
    k = torch.randn(tokens, kv_heads, d, generator=g).bfloat16().to(DEV)
    positions = torch.randint(0, 200000, (tokens,), generator=g).to(DEV)
    inv, factor = rope_frequencies(rotary, scaling="yarn", factor=4.0)
    qo, ko = rope(q, k, positions, inv, interleaved=interleaved, factor=factor)
    close(qo, reference(q, positions, inv, interleaved, factor))
    close(ko, reference(k, positions, inv, interleaved, factor))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rope_far_and_negative_positions(dtype):
    """Positions past 24 and (int64) 31 bits, where p * f in fp32 has no digits left after the point."""
    far = [0, -1, -100001, 2 ** 24 + 1, 2 ** 31 - 1, -(2 ** 31)]
    if dtype == torch.int64:
        far += [2 ** 31 + 12345, 2 ** 35 + 7, -(2 ** 35) - 7]
    positions = torch.tensor(far, dtype=dtype, device=DEV)
    q = torch.randn(len(far), 2, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    inv, _ = rope_frequencies(128)
    got, none = rope(q, None, positions, inv)
    assert none is None
    close(got, reference(q, positions, inv, False, 1.0, far_angles(positions, inv)))


def test_rope_strided_views_and_shapes():
    """Views of a fused projection, a batch dimension, unaligned starts and gaps, and empty calls."""
    g = torch.Generator().manual_seed(2)
    inv, _ = rope_frequencies(64, scaling="ntk", factor=8.0)
    fused = torch.randn(2, 9, (4 + 2 * 2) * 128, generator=g).bfloat16().to(DEV)
    q, k = fused[..., :512].unflatten(-1, (4, 128)), fused[..., 512:768].unflatten(-1, (2, 128))
    positions = torch.arange(18, device=DEV).reshape(2, 9)
    qo, ko = rope(q, k, positions, inv)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.is_contiguous()
    close(qo, reference(q, positions, inv, False, 1.0))
    close(ko, reference(k, positions, inv, False, 1.0))
    odd = torch.randn(7, 3, 133, generator=g).bfloat16().to(DEV)[:, :, 3:131]  # 2-byte aligned rows
    close(rope(odd, None, positions.flatten()[:7], inv)[0], reference(odd, positions.flatten()[:7], inv, False, 1.0))
    wide = torch.randn(7, 128, 3, generator=g).bfloat16().to(DEV).transpose(1, 2)  # columns not contiguous
    close(rope(wide, None, positions.flatten()[:7], inv)[0], reference(wide, positions.flatten()[:7], inv, False, 1.0))
    every_other = torch.arange(14, device=DEV)[::2]
    close(rope(odd, None, every_other, inv)[0], reference(odd, every_other, inv, False, 1.0))
    assert rope(q[:0], k[:0], positions[:0], inv)[0].shape == (0, 9, 4, 128)
    nothing = torch.empty(0, device=DEV)
    assert torch.equal(rope(q, None, positions, nothing)[0], q)


def test_rope_keeps_non_finite_values_in_their_pairs():
    inv, _ = rope_frequencies(8)
    q = torch.ones(1, 1, 16, device=DEV, dtype=torch.bfloat16)
    q[0, 0, 1], q[0, 0, 12] = math.inf, math.nan
    out = rope(q, None, torch.tensor([3], device=DEV), inv)[0][0, 0]
    bad = ~torch.isfinite(out)
    assert bad.nonzero().flatten().tolist() == [1, 5, 12]


def test_rope_other_stream():
    q = torch.randn(64, 4, 128, device=DEV).bfloat16()
    inv, _ = rope_frequencies(128)
    positions = torch.arange(64, device=DEV)
    expected = rope(q, None, positions, inv)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rope(q, None, positions, inv)[0]
    side.synchronize()
    assert torch.equal(got, expected)


def test_rope_refusals():
    q = torch.zeros(4, 2, 64, device=DEV, dtype=torch.bfloat16)
    p, inv = torch.arange(4, device=DEV), torch.ones(32, device=DEV)
    with pytest.raises(ValueError, match="bf16"):
        rope(q.float(), None, p, inv)
    with pytest.raises(ValueError, match="positions for"):
        rope(q, None, p[:3], inv)
    with pytest.raises(ValueError, match="int32 or int64"):
        rope(q, None, p.float(), inv)
    with pytest.raises(ValueError, match="do not fit"):
        rope(q, None, p, torch.ones(33, device=DEV))
    with pytest.raises(ValueError, match="fp32 vector"):
        rope(q, None, p, inv.double())
    with pytest.raises(ValueError, match="tokens or head_dim"):
        rope(q, q[:3], p, inv)
    with pytest.raises(ValueError, match="CUDA"):
        rope(q.cpu(), None, p.cpu(), inv.cpu())
