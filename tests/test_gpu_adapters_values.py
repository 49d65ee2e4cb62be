"""GPU tests of adapters.add_adapters at values and places that the formula decides (tolerance: as in test_gpu_adapters)."""
from __future__ import annotations

import math

import pytest
import torch

from lynnreal_omni_b200 import _lib
from lynnreal_omni_b200.adapters import add_adapters
from test_gpu_adapters import compare, reference, tensors

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128])
@pytest.mark.parametrize("tokens,width", [(5, 128), (130, 1024), (700, 128), (700, 1024)])
@pytest.mark.parametrize("where", ["x", "scale"])
def test_an_infinity_gives_infinities(where, tokens, width, rank):
    """Positive weights: an infinite input value, or scale, gives its rows infinities of its sign and no NaN, whatever the rank is
    padded to on the way; other rows stay what they were."""
    base, x, down, up, index, scale = tensors(tokens, width, 72 if width == 128 else 71, rank, 3, seed=rank)
    x, down, up = x.abs() + 1, down.abs() + 2.0 ** -6, up.abs() + 2.0 ** -6
    index[0] = 1
    lost = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    if where == "x":
        lost[::3] = True
        x[lost, 5] = -math.inf
    else:
        lost = index == 1
        scale[1] = -math.inf
    lost &= index >= 0
    got = add_adapters(base, x, down, up, index, scale)
    assert _lib.device_status() == 0 and bool(lost.any())
    assert bool((got[lost] == -math.inf).all())
    rest = ~lost
    compare(got[rest], reference(base[rest], x[rest], down, up, index[rest], scale))


@pytest.mark.parametrize("tokens", [9, 640])
def test_adapters_off_16_byte_boundaries(tokens):
    """Contiguous weights that begin anywhere, as slices of one flat checkpoint do."""
    base, x, down, up, index, scale = tensors(tokens, 128, 192, 16, 3)
    expected = add_adapters(base, x, down, up, index, scale)
    for left in (1, 4):
        flat = torch.full((left + down.numel() + 3 + up.numel() + 5,), 7.0, device=DEV, dtype=torch.bfloat16)
        d = flat[left:left + down.numel()].view(down.shape)
        u = flat[left + down.numel() + 3:-5].view(up.shape)
        d.copy_(down), u.copy_(up)
        assert d.is_contiguous() and u.is_contiguous()
        assert torch.equal(add_adapters(base, x, d, u, index, scale), expected)
        assert torch.equal(add_adapters(base, x, d, up, index, scale), expected)
        assert torch.equal(add_adapters(base, x, down, u, index, scale), expected)
    odd = torch.cat((index[:1], index))[1:]
    assert torch.equal(add_adapters(base, x, down, up, odd, scale), expected)
