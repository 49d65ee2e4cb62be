"""GPU tests of adapters.add_adapters and AdaptedLinear against the formula in 64 bits, token by token.

Tolerance per value: the inner values are rounded to bf16 for the second product (2^-8 each, so 2^-8 of sum |scale h up|), the
output once (2^-8 of it); the fp32 sums of n terms are off by n 2^-24 of the sum of magnitudes at most (the first over the
width, the second over the rank and the base).
"""
from __future__ import annotations

import math

import pytest
import torch

from lynnreal_omni_b200 import _lib
from lynnreal_omni_b200.adapters import AdaptedLinear, add_adapters, token_adapters
from lynnreal_omni_b200.fp4 import Fp4Linear
from lynnreal_omni_b200.int8 import Int8Linear

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tensors(tokens, width, outputs, rank, count, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    base, x = normal(tokens, outputs), normal(tokens, width)
    down, up = normal(count, rank, width) * width ** -0.5, normal(count, outputs, rank) * rank ** -0.5
    scale = torch.rand(count, generator=g) + 0.5
    index = torch.randint(-1, count, (tokens,), generator=g, dtype=torch.int32)
    return [t.bfloat16().to(DEV) for t in (base, x, down, up)] + [index.to(DEV), scale.to(DEV)]


def reference(base, x, down, up, index, scale):
    """(the result, the bound on its error) in 64 bits."""
    out, width, rank = base.double(), x.shape[1], down.shape[1]
    size, fine = torch.zeros_like(out), out.abs() * rank * 2.0 ** -24
    for e in range(down.shape[0]):
        rows = (index == e).nonzero()[:, 0]
        s = 1.0 if scale is None else float(scale[e])
        xs, d, u = x[rows].double(), down[e].double(), up[e].double()
        h = s * (xs @ d.t())
        out[rows] += h @ u.t()
        size[rows] = h.abs() @ u.abs().t()
        fine[rows] += (abs(s) * (xs.abs() @ d.abs().t()) @ u.abs().t()) * (width + rank) * 2.0 ** -24
    return out, 2.0 ** -8 * (size + out.abs()) * (1 + 2.0 ** -8) + 2 * fine + 1e-30


def compare(got, expected):
    ref, bound = expected
    assert got.dtype == torch.bfloat16 and got.shape == ref.shape
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), (float((err / bound).max()), (~(err <= bound)).nonzero()[:4].tolist())


def check(tokens, width, outputs, rank, count, seed=0, index=None, scaled=True):
    base, x, down, up, drawn, scale = tensors(tokens, width, outputs, rank, count, seed)
    index = drawn if index is None else torch.tensor(index, dtype=torch.int32, device=DEV)
    scale = scale if scaled else None
    got = add_adapters(base, x, down, up, index, scale)
    compare(got, reference(base, x, down, up, index, scale))
    assert torch.equal(got[index < 0], base[index < 0])
    assert _lib.device_status() == 0
    return got


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 104, 128])
@pytest.mark.parametrize("tokens", [1, 17, 600])
def test_ranks(tokens, rank):
    check(tokens, 264, 520, rank, 3, seed=rank)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 31, 33, 64, 65, 511, 512, 513, 575, 576, 577, 1000])
@pytest.mark.parametrize("count", [1, 5, 70])
def test_tokens_and_adapters_in_any_order(tokens, count):
    check(tokens, 512, 256, 16, count, seed=tokens)


@pytest.mark.parametrize("width", [8, 24, 32, 40, 504, 2048, 6144, 20000])
@pytest.mark.parametrize("tokens", [3, 700])
def test_widths(tokens, width):
    check(tokens, width, 72, 16, 2, seed=width)


@pytest.mark.parametrize("outputs", [1, 7, 8, 31, 33, 255, 256, 264, 1001, 4096])
@pytest.mark.parametrize("tokens,rank", [(5, 16), (530, 16), (20, 64), (530, 128)])
def test_outputs(tokens, outputs, rank):
    check(tokens, 128, outputs, rank, 4, seed=outputs)


@pytest.mark.parametrize("tokens", [40, 900])
def test_one_adapter_for_all_and_none_for_any(tokens):
    check(tokens, 256, 256, 32, 3, index=[2] * tokens)
    check(tokens, 256, 256, 32, 3, index=[-1] * tokens)
    check(tokens, 256, 256, 32, 3, index=[-7] * tokens, scaled=False)


@pytest.mark.parametrize("tokens,outputs,count", [(600, 25864, 3), (70, 77000, 1), (640, 256 * 100 + 8, 2)])
def test_rows_that_the_grid_does_not_divide(tokens, outputs, count):
    """Blocks whose columns change from tile to tile, some of them past the last."""
    check(tokens, 64, outputs, 16, count, seed=outputs)


def test_large():
    check(5000, 4096, 12288, 32, 3, index=[0] * 2000 + [-1] * 17 + [2] * 2983)


@pytest.mark.parametrize("tokens", [30, 800])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_neighbours_do_not_reach_a_token(tokens, bad):
    """Infinities and NaN in other tokens' rows, other adapters and unused ones leave a row as it was."""
    base, x, down, up, index, scale = tensors(tokens, 256, 264, 16, 4)
    clean = add_adapters(base, x, down, up, index, scale)
    mine = index == 1
    for t in (x, base):
        t[~mine] = bad
    for t in (down, up):
        t[torch.arange(4) != 1] = bad
    scale[torch.arange(4) != 1] = bad
    got = add_adapters(base, x, down, up, index, scale)
    assert torch.equal(got[mine], clean[mine]) and bool(mine.any())
    assert not bool(torch.isfinite(got[~mine]).any())


@pytest.mark.parametrize("tokens", [12, 700])
def test_numbers_past_the_last_adapter_count_as_none(tokens):
    base, x, down, up, index, scale = tensors(tokens, 128, 128, 16, 3)
    wrong = index.clone()
    wrong[5], wrong[7] = 3, 2 ** 31 - 1
    index[5] = index[7] = -1
    expected = add_adapters(base, x, down, up, index, scale)
    assert _lib.device_status() == 0
    assert torch.equal(add_adapters(base, x, down, up, wrong, scale), expected)
    assert _lib.device_status() == 16 and _lib.device_status() == 0


@pytest.mark.parametrize("tokens", [9, 640])
def test_strides_and_places(tokens):
    """Rows of wider tensors, unaligned ones, a broadcast base, columns that are not contiguous, and results in place."""
    base, x, down, up, index, scale = tensors(tokens, 128, 192, 16, 3)
    expected = add_adapters(base, x, down, up, index, scale)
    for left in (0, 1, 8):
        wide_x, wide_base, wide_out = (torch.full((tokens, 400), 7.0, device=DEV, dtype=torch.bfloat16) for _ in range(3))
        xs, bs, os = wide_x[:, left:left + 128], wide_base[:, left:left + 192], wide_out[:, left:left + 192]
        xs.copy_(x)
        bs.copy_(base)
        assert torch.equal(add_adapters(bs, xs, down, up, index, scale), expected)
        assert add_adapters(bs, xs, down, up, index, scale, out=os) is os
        assert torch.equal(os, expected)
        assert bool((wide_out[:, :left] == 7).all()) and bool((wide_out[:, left + 192:] == 7).all())
        add_adapters(bs, xs, down, up, index, scale, out=bs)
        assert torch.equal(bs, expected)
        assert bool((wide_base[:, :left] == 7).all()) and bool((wide_base[:, left + 192:] == 7).all())
    assert torch.equal(add_adapters(base.t().contiguous().t(), x.t().contiguous().t(), down, up, index, scale), expected)
    assert torch.equal(add_adapters(base, x, down.transpose(1, 2).contiguous().transpose(1, 2), up, index, scale), expected)
    row = base[:1].expand(tokens, -1)
    assert torch.equal(add_adapters(row, x, down, up, index, scale), add_adapters(row.contiguous(), x, down, up, index, scale))


@pytest.mark.parametrize("tokens", [50, 3000])
def test_results_repeat_and_streams(tokens):
    args = tensors(tokens, 1024, 512, 32, 6)
    expected = add_adapters(*args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(add_adapters(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, expected) for g in got)


@pytest.mark.parametrize("tokens", [24, 900])
def test_graph_replay_follows_new_numbers(tokens):
    base, x, down, up, index, scale = tensors(tokens, 256, 256, 16, 5)
    add_adapters(base, x, down, up, index, scale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = add_adapters(base, x, down, up, index, scale)
    for seed in range(3):
        for t, fresh in zip((base, x, down, up, index, scale), tensors(tokens, 256, 256, 16, 5, seed)):
            t.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        compare(out, reference(base, x, down, up, index, scale))


def test_adapted_linear():
    """Beside an int8 and a 4-bit projection: the projection's own output plus the update, in place of nothing else."""
    g = torch.Generator().manual_seed(5)
    linear = torch.nn.Linear(256, 320, device=DEV, dtype=torch.bfloat16)
    parts = [(torch.randn(r, 256, generator=g).bfloat16().to(DEV), torch.randn(320, r, generator=g).bfloat16().to(DEV), 0.01 * (r + 1))
             for r in (4, 16, 1)]
    x = torch.randn(2, 20, 256, generator=g).bfloat16().to(DEV)
    index = token_adapters([0, None, 2, 1], [3, 7, 0, 30])
    assert index.dtype == torch.int32 and index.tolist() == [0] * 3 + [-1] * 7 + [1] * 30
    with torch.no_grad():
        for base in (Fp4Linear(linear), Int8Linear(linear)):
            layer = AdaptedLinear.stack(base, parts)
            assert layer.down.shape == (3, 16, 256) and layer.up.shape == (3, 320, 16)
            assert torch.equal(layer(x), base(x))
            got = layer(x, index)
            assert got.shape == (2, 20, 320)
            expected = add_adapters(base(x).view(40, 320), x.view(40, 256), layer.down, layer.up, index, layer.scale)
            assert torch.equal(got.view(40, 320), expected) and not torch.equal(got, base(x))


def test_empty_and_refusals():
    base, x, down, up, index, scale = tensors(6, 64, 64, 16, 2)
    assert add_adapters(base[:0], x[:0], down, up, index[:0], scale).shape == (0, 64)

    def refused(match, *args, **more):
        with pytest.raises(ValueError, match=match):
            add_adapters(*args, **more)

    refused("bf16", base.float(), x, down, up, index)
    refused("bf16", base, x, down.float(), up, index)
    refused("disagree", base, x, down, up[:1], index)
    refused("disagree", base, x, down[:, :8], up, index)
    refused("rank", base, x, down[:, :4], up[..., :4], index)
    refused("rank", base, x, down.repeat(1, 9, 1), up.repeat(1, 1, 9), index)
    refused("width", base, x[:, :60], down[..., :60], up, index)
    refused("base must", base[:, :32], x, down, up, index)
    refused("x must", base, x[:, :32], down, up, index)
    refused("differ in tokens", base[:5], x, down, up, index)
    refused("int32", base, x, down, up, index.long())
    refused("int32", base, x, down, up, index[:5])
    refused("fp32", base, x, down, up, index, scale.bfloat16())
    refused("fp32", base, x, down, up, index, scale[:1])
    refused("empty|no adapters", base, x, down[:0], up[:0], index)
    refused("out must", base, x, down, up, index, out=base[:, :32])
    refused("out must", base, x, down, up, index, out=base[:1].expand(6, -1))
    refused("out must", base, x, down, up, index, out=base.t().contiguous().t())
    refused("adapters' device", base, x.cpu(), down, up, index)
    with pytest.raises(ValueError, match="beside a projection"):
        AdaptedLinear(torch.nn.Linear(64, 32), down, up)
    with pytest.raises(ValueError, match="no adapters"):
        AdaptedLinear.stack(torch.nn.Linear(64, 64), [])
    with pytest.raises(ValueError, match="one adapter"):
        token_adapters([0], [3, 4], "cpu")
    with pytest.raises(ValueError, match="numbered"):
        token_adapters([-2], [3], "cpu")
