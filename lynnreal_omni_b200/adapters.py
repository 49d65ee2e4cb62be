"""Low-rank adapters of many requests beside a shared projection.

``add_adapters`` adds every token's own low-rank update to the output of a projection that all tokens share:

    out[t] = base[t] + scale[e] * up[e] (down[e] x[t]),  e = index[t]        (index[t] < 0: out[t] = base[t])

``AdaptedLinear`` puts it behind an ``Int8Linear``, an ``Fp4Linear`` or any other layer that maps bf16 rows to bf16 rows:

    layer = AdaptedLinear.stack(Fp4Linear(linear), [(down0, up0, 2.0), (down1, up1, 0.5)])
    index = token_adapters([0, 1, None], [3, 70, 12], "cuda")  # prompts of 3, 70 and 12 tokens, the last without one
    y = layer(x, index)                                        # x bf16 [85, in_features]
"""
from __future__ import annotations

import functools

import torch
from torch import nn

from . import _lib
from ._lib import check, ptr, stream_of

__all__ = ["add_adapters", "token_adapters", "AdaptedLinear"]

MOST_RANK = 128


def token_adapters(adapters, lengths, device="cuda") -> torch.Tensor:
    """int32 [tokens]: the adapter of each token of requests of these lengths, one after another (None: no adapter)."""
    if len(adapters) != len(lengths) or (lengths and min(lengths) < 0):
        raise ValueError("token_adapters: expected one adapter, or None, for each request's length")
    if any(a is not None and a < 0 for a in adapters):
        raise ValueError("token_adapters: adapters are numbered from 0")
    numbers = torch.tensor([-1 if a is None else a for a in adapters], dtype=torch.int32)
    return numbers.repeat_interleave(torch.tensor(lengths, dtype=torch.int64)).to(device)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device: int, tokens: int, width: int, outputs: int, rank: int, count: int) -> int:
    """lr_adapters' need for these sizes on this device (a function of them alone)."""
    return _lib.load().lr_adapters_workspace_bytes(tokens, width, outputs, rank, count)


def _check_stack(name: str, down: torch.Tensor, up: torch.Tensor, scale: torch.Tensor | None):
    """(adapters, rank, width, outputs) of adapters that fit each other."""
    if down.dtype is not torch.bfloat16 or down.ndim != 3 or up.dtype is not torch.bfloat16 or up.ndim != 3:
        raise ValueError(f"{name}: down and up must be bf16 tensors of three dimensions, got {down.dtype} {tuple(down.shape)}, "
                         f"{up.dtype} {tuple(up.shape)}")
    count, rank, width = down.shape
    up_count, outputs, up_rank = up.shape
    if up_count != count or up_rank != rank or up.get_device() != down.get_device():
        raise ValueError(f"{name}: down [adapters, rank, in] and up [adapters, out, rank] disagree: {tuple(down.shape)}, {tuple(up.shape)}")
    if count == 0 or width == 0 or outputs == 0:
        raise ValueError(f"{name}: no adapters, or empty ones")
    if rank == 0 or rank % 8 or rank > MOST_RANK:
        raise ValueError(f"{name}: the rank must be a multiple of 8 up to {MOST_RANK} (pad with zeros), got {rank}")
    if width % 8:
        raise ValueError(f"{name}: the input width must be a multiple of 8, got {width}")
    if scale is not None and (scale.dtype is not torch.float32 or scale.numel() != count or scale.get_device() != down.get_device()):
        raise ValueError(f"{name}: scale must hold {count} fp32 values on the adapters' device")
    return count, rank, width, outputs


def _readable(weight: torch.Tensor) -> torch.Tensor:
    """The weight as the kernels read it: contiguous from a 16-byte boundary."""
    return weight if weight.is_contiguous() and weight.data_ptr() % 16 == 0 else weight.clone(memory_format=torch.contiguous_format)


def add_adapters(base: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, index: torch.Tensor,
                 scale: torch.Tensor | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 [tokens, out]: base plus every token's low-rank update.

    base bf16 [tokens, out] and x bf16 [tokens, in]: rows may be strided; down bf16 [adapters, rank, in], up bf16
    [adapters, out, rank], rank a multiple of 8 up to 128 (copied at each call where they are not contiguous from a 16-byte
    boundary); scale fp32 [adapters] (None: 1); index int32 [tokens] on the device, negative for no adapter (a number past the last
    adapter counts as none and raises bit 4 of the device status). The inner values down[e] x[t] are summed in fp32, scaled and
    rounded to bf16 for the second product; base and update are added in fp32 and rounded once. Any order will do, tokens of one adapter side by side are fastest. ``out`` may be ``base`` itself; it must not overlap
    x, nor base in any other way. There is no backward pass: an ``out`` that belongs to an autograd graph is refused."""
    if out is not None and out.requires_grad and torch.is_grad_enabled():
        raise ValueError("add_adapters: out belongs to an autograd graph, whose gradients would miss the update; call it under torch.no_grad()")
    count, rank, width, outputs = _check_stack("add_adapters", down, up, scale)
    device = down.get_device()
    if base.dtype is not torch.bfloat16 or base.ndim != 2 or base.shape[1] != outputs or base.get_device() != device:
        raise ValueError(f"add_adapters: base must be a bf16 [tokens, {outputs}] tensor on the adapters' device, got {base.dtype} "
                         f"{tuple(base.shape)}")
    if x.dtype is not torch.bfloat16 or x.ndim != 2 or x.shape[1] != width or x.get_device() != device:
        raise ValueError(f"add_adapters: x must be a bf16 [tokens, {width}] tensor on the adapters' device, got {x.dtype} "
                         f"{tuple(x.shape)}")
    tokens = x.shape[0]
    if base.shape[0] != tokens:
        raise ValueError(f"add_adapters: base and x differ in tokens: {base.shape[0]}, {tokens}")
    if index.dtype is not torch.int32 or index.ndim != 1 or index.shape[0] != tokens or index.get_device() != device:
        raise ValueError("add_adapters: index must be int32 [tokens] on the adapters' device")
    if device < 0:
        raise ValueError("add_adapters: expected CUDA tensors")
    if device != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return add_adapters(base, x, down, up, index, scale, out=out)
    if out is None:
        out = torch.empty_like(base, memory_format=torch.contiguous_format)
    elif (out.dtype != torch.bfloat16 or out.shape != base.shape or out.get_device() != device or out.stride(1) != 1
          or (tokens > 1 and out.stride(0) < outputs)):
        raise ValueError("add_adapters: out must be a bf16 tensor of base's shape with contiguous rows that do not overlap")
    down_at, up_at = down.data_ptr(), up.data_ptr()
    if (down_at | up_at) % 16 or not (down.is_contiguous() and up.is_contiguous() and index.is_contiguous()):
        down, up, index = _readable(down), _readable(up), index.contiguous()
        down_at, up_at = down.data_ptr(), up.data_ptr()
    if scale is not None:
        scale = scale.contiguous()
    base_stride, one = base.stride()
    if one != 1:
        base, base_stride = base.contiguous(), outputs
    x_stride, one = x.stride()
    if one != 1 or x_stride % 8 or x_stride < width or x.data_ptr() % 16:
        x, x_stride = x.clone(memory_format=torch.contiguous_format), width
    need = _workspace_bytes(device, tokens, width, outputs, rank, count)
    workspace = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    check(_lib.load().lr_adapters(x.data_ptr(), x_stride, base.data_ptr(), base_stride, down_at, up_at,
                                  ptr(scale), index.data_ptr(), tokens, width, outputs, rank, count, out.data_ptr(),
                                  max(out.stride(0), outputs), ptr(workspace), need, stream_of(x)), "add_adapters")
    return out


class AdaptedLinear(nn.Module):
    """A shared projection and the adapters of its requests, for inference. ``base``: a layer from bf16 [..., in] to a new bf16
    [..., out] tensor, in which the update is made."""

    def __init__(self, base: nn.Module, down: torch.Tensor, up: torch.Tensor, scale: torch.Tensor | None = None):
        super().__init__()
        _, _, width, outputs = _check_stack("AdaptedLinear", down, up, scale)
        if width != base.in_features or outputs != base.out_features:
            raise ValueError(f"AdaptedLinear: adapters of {width} to {outputs} beside a projection of {base.in_features} to "
                             f"{base.out_features}")
        self.base, self.in_features, self.out_features = base, width, outputs
        self.register_buffer("down", _readable(down))
        self.register_buffer("up", _readable(up))
        self.register_buffer("scale", scale)

    @classmethod
    def stack(cls, base: nn.Module, adapters) -> "AdaptedLinear":
        """From a list of (down [rank, in], up [out, rank], scale) of any ranks up to 128; ranks are padded with zeros."""
        if not adapters:
            raise ValueError("AdaptedLinear: no adapters")
        for d, u, _ in adapters:
            if (d.ndim != 2 or u.ndim != 2 or d.shape[0] != u.shape[1] or d.shape[1] != base.in_features
                    or u.shape[0] != base.out_features):
                raise ValueError(f"AdaptedLinear: expected (down [rank, {base.in_features}], up [{base.out_features}, rank], scale) for each "
                                 f"adapter, got {tuple(d.shape)}, {tuple(u.shape)}")
        ranks = [d.shape[0] for d, _, _ in adapters]
        rank = max(8, -(-max(ranks) // 8) * 8)
        device = adapters[0][0].device
        down = torch.zeros(len(ranks), rank, base.in_features, dtype=torch.bfloat16, device=device)
        up = torch.zeros(len(ranks), base.out_features, rank, dtype=torch.bfloat16, device=device)
        for i, (d, u, _) in enumerate(adapters):
            down[i, :ranks[i]], up[i, :, :ranks[i]] = d, u
        return cls(base, down, up, torch.tensor([s for _, _, s in adapters], dtype=torch.float32, device=device))

    def forward(self, x: torch.Tensor, index: torch.Tensor | None = None) -> torch.Tensor:
        """x bf16 [..., in], index int32 with a number for each row (None: the shared projection alone)."""
        y = self.base(x)
        if index is None:
            return y
        rows = y.view(-1, self.out_features)
        add_adapters(rows, x.reshape(-1, self.in_features), self.down, self.up, index.reshape(-1), self.scale, out=rows)
        return y
