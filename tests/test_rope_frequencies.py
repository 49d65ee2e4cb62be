"""CPU tests of rotary.rope_frequencies against the formulas."""
import math

import pytest
import torch

from lynnreal_omni_b200.rotary import rope_frequencies


def test_unscaled_linear_and_ntk():
    plain, one = rope_frequencies(128, device="cpu")
    assert one == 1.0 and plain.dtype == torch.float32
    expected = torch.tensor([10000.0 ** (-2 * i / 128) for i in range(64)], dtype=torch.float64)
    assert torch.equal(plain, expected.float())
    assert torch.equal(rope_frequencies(128, scaling="linear", factor=4, device="cpu")[0], (expected / 4).float())
    ntk = rope_frequencies(128, scaling="ntk", factor=4, device="cpu")[0].double()
    assert ntk[0] == 1 and math.isclose(ntk[-1], expected[-1] / 4, rel_tol=1e-6)
    assert bool((ntk <= expected * 1.000001).all()) and bool((ntk >= expected / 4 * 0.999999).all())


def test_yarn_keeps_fast_and_divides_slow_frequencies():
    plain = rope_frequencies(128, device="cpu")[0].double()
    inv, output = rope_frequencies(128, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    inv = inv.double()
    assert output == 0.1 * math.log(8.0) + 1.0
    turns = 4096 * plain / (2 * math.pi)
    # the ramp's ends are rounded outwards to whole indices, so beyond them the rule is exact
    fast, slow = turns > 32 * 1.2, turns < 1 / 1.2
    assert torch.allclose(inv[fast], plain[fast], rtol=1e-6) and torch.allclose(inv[slow], plain[slow] / 8, rtol=1e-6)
    ratio = inv / plain
    assert bool((ratio[1:] <= ratio[:-1] * 1.000001).all())
    assert torch.equal(rope_frequencies(2, scaling="yarn", factor=1.0, device="cpu")[0], torch.ones(1))


@pytest.mark.parametrize("kwargs", [dict(rotary_dim=0), dict(rotary_dim=5), dict(rotary_dim=8, scaling="other"),
                                    dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, base=1.0),
                                    dict(rotary_dim=8, fast_turns=1.0, slow_turns=2.0)])
def test_refusals(kwargs):
    with pytest.raises(ValueError):
        rope_frequencies(device="cpu", **kwargs)


@pytest.mark.parametrize("length,dim,base", [(65536, 128, 10000.0), (131072, 128, 10000.0), (262144, 64, 500.0), (4096, 128, 10000.0),
                                             (100, 128, 10000.0), (131072, 2, 10000.0)])
def test_yarn_ramp_may_end_beyond_the_last_index(length, dim, base):
    """One index at a time: where even the slowest frequency makes more than one turn, it is divided in part only."""
    inv, _ = rope_frequencies(dim, base=base, scaling="yarn", factor=4.0, original_length=length, device="cpu")
    start, end = (dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (32.0, 1.0))
    start, end = max(math.floor(start), 0), min(math.ceil(end), dim - 1)
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        divided = min(max((i - start) / max(end - start, 1e-3), 0.0), 1.0)
        assert math.isclose(inv[i], plain * (1 - divided) + plain / 4 * divided, rel_tol=1e-6), i
    if length == 131072 and dim == 128:
        assert math.isclose(inv[-1] / 10000.0 ** (-126 / 128), 0.46, rel_tol=1e-6)  # 18 of the ramp's 25 indices
