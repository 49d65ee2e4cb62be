"""GPU tests of attention.attention_shared at the sizes where its layout changes (tolerance: as in test_gpu_attention_shared)."""
from __future__ import annotations

import pytest

from test_gpu_attention_shared import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hk", [593, 600, 4096])
@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1, 2, 1], [30, 0, 9]), ([10], [10]), ([17], [300])])
def test_many_key_heads(lq, lk, hk):
    """More key/value heads than the GPU has places for blocks."""
    check(100, lq, lk, hk, hk, 64, seed=hk)
