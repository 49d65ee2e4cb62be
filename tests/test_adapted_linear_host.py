"""CPU tests of AdaptedLinear: what it accepts, and where it stands in the way of a silent mistake."""
from __future__ import annotations

import pytest
import torch

from lynnreal_omni_b200.adapters import AdaptedLinear, add_adapters


def ones(*shape):
    return torch.ones(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("down,up", [((3, 1), (24, 3)), ((3, 64), (1, 3)), ((3, 32), (24, 3)), ((3, 64), (64, 3)), ((3,), (24, 3)), ((3, 64), (24,)),
                                     ((3, 64), (24, 1)), ((3, 64, 1), (24, 3)), ((), (24, 3))])
def test_stack_refuses_adapters_of_other_sizes(down, up):
    """Also those that would spread over the rows or columns when they are copied into place."""
    base = torch.nn.Linear(64, 24, bias=False, dtype=torch.bfloat16)
    assert AdaptedLinear.stack(base, [(ones(3, 64), ones(24, 3), 1.0)]).down.shape == (1, 8, 64)
    with pytest.raises(ValueError, match="AdaptedLinear"):
        AdaptedLinear.stack(base, [(ones(3, 64), ones(24, 3), 1.0), (ones(*down), ones(*up), 1.0)])


def test_no_update_behind_autograd():
    """A projection whose output belongs to a graph: the update would be missing from the gradients, so the call is refused."""
    x, index = ones(5, 64), torch.zeros(5, dtype=torch.int32)
    layer = AdaptedLinear.stack(torch.nn.Linear(64, 24, dtype=torch.bfloat16), [(ones(3, 64), ones(24, 3), 1.0)])
    with pytest.raises(ValueError, match="gradients"):
        layer(x, index)
    out = ones(5, 24).requires_grad_()
    with pytest.raises(ValueError, match="gradients"):
        add_adapters(ones(5, 24), x, layer.down, layer.up, index, out=out)
    assert layer(x).requires_grad  # the projection alone stays as it is
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # on to the next check
        layer(x, index)
