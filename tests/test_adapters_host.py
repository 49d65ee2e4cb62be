"""CPU tests of what the host decides: refusals before anything runs, and workspaces as functions of the sizes."""
from __future__ import annotations

import pytest
import torch

from lynnreal_omni_b200 import _lib
from lynnreal_omni_b200.adapters import AdaptedLinear, add_adapters, token_adapters
from lynnreal_omni_b200.attention import attention_shared


def test_tensors_off_the_gpu_are_refused():
    a = torch.zeros(4, 64, dtype=torch.bfloat16)
    down, up = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 64, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        add_adapters(a, a, down, up, torch.zeros(4, dtype=torch.int32))
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        attention_shared(q, q, q, q, q, torch.tensor([0, 4], dtype=torch.int32))


def test_token_adapters():
    assert token_adapters([2, None, 0], [1, 2, 0], "cpu").tolist() == [2, -1, -1]
    assert token_adapters([], [], "cpu").shape == (0,)
    with pytest.raises(ValueError):
        token_adapters([0, 1], [3], "cpu")
    with pytest.raises(ValueError):
        token_adapters([0], [-3], "cpu")


def test_stack_pads_ranks():
    base = torch.nn.Linear(64, 24, bias=False, dtype=torch.bfloat16)
    parts = [(torch.ones(r, 64, dtype=torch.bfloat16), torch.ones(24, r, dtype=torch.bfloat16), float(r)) for r in (3, 9)]
    layer = AdaptedLinear.stack(base, parts)
    assert layer.down.shape == (2, 16, 64) and layer.up.shape == (2, 24, 16) and layer.scale.tolist() == [3.0, 9.0]
    assert layer.down[0].sum() == 3 * 64 and layer.up[0].sum() == 3 * 24
    with pytest.raises(ValueError):
        AdaptedLinear.stack(base, [(parts[0][0], parts[1][1], 1.0)])


def test_workspaces():
    lib = _lib.load()
    need = lib.lr_adapters_workspace_bytes
    assert need(1, 6144, 18432, 16, 8) == 0 and need(0, 64, 64, 8, 1) == 0  # one kernel, nothing between
    assert need(600, 64, 64, 8, 3) == 600 * 16 * 2 and need(12240, 6144, 24576, 72, 2) == 12240 * 128 * 2
    assert need(10, 64, 64, 9, 3) == 0  # refused by the call
    need = lib.lr_attention_shared_workspace_bytes
    assert need(8, 10000, 10000, 8192, 32, 8, 128) == 0  # whole prompts: nothing between
    few, many = need(64, 64, 20000, 8192, 32, 8, 128), need(64, 64, 20000, 80000, 32, 8, 128)
    assert 0 < few <= many < 1 << 28
    assert need(64, 64, 20000, 0, 32, 8, 128) == 0  # refused by the call


@pytest.mark.parametrize("args,message", [
    ((4, 64, 64, 12, 2), b"rank"), ((4, 60, 64, 8, 2), b"width"), ((4, 0, 64, 8, 2), b"shape"), ((-1, 64, 64, 8, 2), b"shape")])
def test_adapters_refuses_sizes(args, message):
    lib = _lib.load()
    tokens, width, outputs, rank, count = args
    assert lib.lr_adapters(None, width, None, outputs, None, None, None, None, tokens, width, outputs, rank, count, None, outputs, None,
                           0, None) in (_lib.LR_ERR_INVALID_ARGUMENT, _lib.LR_ERR_UNSUPPORTED)
    assert message in lib.lr_last_error()


def test_attention_shared_refuses():
    lib = _lib.load()

    def call(prefix=8, d=64, q=None):
        return lib.lr_attention_shared(q, 128, 64, None, 128, 64, None, 128, 64, None, 128, 64, None, 128, 64, None, None, 1, 4, 4, prefix,
                                       2, 2, d, 1, 0.125, None, None, 0, None)

    assert call(prefix=0) == _lib.LR_ERR_INVALID_ARGUMENT and b"prefix" in lib.lr_last_error()
    assert call(d=32) == _lib.LR_ERR_UNSUPPORTED
    assert call() == _lib.LR_ERR_INVALID_ARGUMENT and b"null" in lib.lr_last_error()
