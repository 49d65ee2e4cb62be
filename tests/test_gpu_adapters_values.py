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
