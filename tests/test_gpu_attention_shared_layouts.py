"""GPU tests of attention.attention_shared at the sizes where its layout changes (tolerance: as in test_gpu_attention_shared)."""
from __future__ import annotations

import pytest
import torch

from lynnreal_omni_b200 import _lib
from lynnreal_omni_b200.attention import attention_shared
from test_gpu_attention_packed import compare, offsets, tensors
from test_gpu_attention_shared import check, prefix_tensors, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hk", [593, 600, 4096])
@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1, 2, 1], [30, 0, 9]), ([10], [10]), ([17], [300])])
def test_many_key_heads(lq, lk, hk):
    """More key/value heads than the GPU has places for blocks."""
    check(100, lq, lk, hk, hk, 64, seed=hk)


def test_more_rows_of_a_sequence_than_a_grid_has():
    """One sequence whose rows, 16 a block, are more blocks than a grid's third dimension counts. A sample of them is compared."""
    tokens, prefix, h, hk, d = 132572, 131072, 8, 2, 64
    q, k, v = tensors([tokens], [0], h, hk, d, seed=4)
    pk, pv = prefix_tensors(prefix, hk, d)
    got = attention_shared(q, k, v, pk, pv, offsets([tokens]), offsets([0]))
    assert _lib.device_status() == 0
    some = torch.cat((torch.arange(40), torch.arange(65520, 65560), torch.arange(131050, 131090), torch.arange(tokens - 40, tokens))).to(q.device)
    compare(got[some], reference(q[some], k, v, pk, pv, [len(some)], [0], True, d ** -0.5))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([17], [9000]), ([40], [3001]), ([128], [5000]), ([20, 20, 20, 20], [30, 4000, 700, 0]), ([33] * 9, [400 * i for i in range(9)]),
                                   ([90, 17, 1, 0, 64], [9000, 40, 2000, 50, 64])])
def test_pieces_of_prompts(lq, lk, causal, d):
    """Queries against longer own keys: in one piece, and in parts with the own keys split and not."""
    for prefix in (40, 700, 12000):
        check(prefix, lq, lk, 8, 2, d, causal, seed=d)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,hk,queries", [(64, 8, 8), (32, 8, 8), (32, 8, 5), (64, 8, 3), (16, 16, 1)])
def test_single_tokens_with_a_warp_a_slot(h, hk, queries, d):
    """Many slots, whose keys are as many as their rows ask for."""
    check(300, [queries] * 40, [max(queries, 131 * i % 1201) for i in range(40)], h, hk, d, seed=queries)
    check(300, [queries] * 3, [30, 31000, 700], h, hk, d, seed=queries)


def test_fewer_queries_than_sequences():
    check(500, [0] * 30 + [1] + [0] * 30 + [1], [20] * 62, 130, 1, 64)
    check(500, [0] * 30 + [1], [300] * 31, 130, 1, 128, False)
