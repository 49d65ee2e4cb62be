"""Rotary positions of queries and keys: half and interleaved layouts, part of the head, scaled for long contexts.

``rope_frequencies`` makes the frequencies once; ``rope`` turns the queries and keys of a batch of tokens at any
positions. Unlike ``kernels.qk_norm_rope`` there is no norm, no table per position, and queries and keys may differ
in their number of heads.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from ._lib import check, ptr, stream_of

__all__ = ["rope_frequencies", "rope"]


def rope_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                     original_length: int = 4096, fast_turns: float = 32.0, slow_turns: float = 1.0, device="cuda"):
    """(inv_freq fp32 [rotary_dim / 2] in radians per position, output factor).

    f_i = base^(-2 i / rotary_dim), for contexts ``factor`` times as long as the ``original_length``:
      * None: unscaled;
      * "linear": f_i / factor;
      * "ntk": the base grown to base * factor^(R / (R - 2)), so that the slowest frequency is divided by the factor
        and the fastest is kept;
      * "yarn": frequencies that make more than ``fast_turns`` turns over the original length are kept, those below
        ``slow_turns`` divided by the factor, a linear ramp over the index between (its ends rounded outwards to whole
        indices and held in [0, rotary_dim - 1]); outputs times 0.1 ln(factor) + 1.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rope_frequencies: rotary_dim must be positive and even, got {rotary_dim}")
    if not (base > 1 and factor >= 1 and original_length > 0 and fast_turns > slow_turns > 0):
        raise ValueError("rope_frequencies: base > 1, factor >= 1, original_length > 0, fast_turns > slow_turns > 0")
    half = rotary_dim // 2
    index = torch.arange(half, dtype=torch.float64)
    output = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = base ** (-index / half)
    if scaling == "linear" or (scaling == "ntk" and rotary_dim == 2):
        inv = inv / factor
    elif scaling == "yarn":
        def crossing(turns):  # the (real) index whose frequency makes that many turns over the original length
            return half * math.log(original_length / (2 * math.pi * turns)) / math.log(base)
        # the ramp may end beyond the last index, half - 1: no frequency is then divided in full
        low, high = max(math.floor(crossing(fast_turns)), 0), min(math.ceil(crossing(slow_turns)), rotary_dim - 1)
        divided = ((index - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv = inv * (1 - divided) + inv / factor * divided
        output = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"rope_frequencies: scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    return inv.to(device=device, dtype=torch.float32), output


def _tokens_view(t: torch.Tensor):
    """(t, token stride, head stride) of [tokens, heads, head_dim] with contiguous columns; a view wherever the strides
    allow."""
    if t.stride(-1) != 1:
        t = t.contiguous()
    if t.ndim != 3:
        t = t.reshape(-1, t.shape[-2], t.shape[-1])
    return t, *t.stride()[:2]


def rope(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
         interleaved: bool = False, factor: float = 1.0):
    """Rotated (query, key), contiguous, in the inputs' shapes.

    query [..., heads, D] and key [..., kv_heads, D] (or None): bf16, strided views of a fused projection are fine;
    positions: int32 or int64, one per token; inv_freq: fp32 [rotary_dim / 2]. The first rotary_dim columns of each
    head are turned, as pairs (i, i + rotary_dim / 2) or, ``interleaved``, (2i, 2i + 1); the others are copied.
    """
    device = query.device
    for name, t in (("query", query), ("key", key)):
        if t is not None and (t.dtype != torch.bfloat16 or t.ndim < 3 or t.device != device):
            raise ValueError(f"rope: {name} must be a bf16 [..., heads, head_dim] tensor on the query's device")
    q, q_ts, q_hs = _tokens_view(query)
    tokens, heads, d = q.shape
    rotary = 2 * inv_freq.numel()
    if inv_freq.dtype != torch.float32 or inv_freq.ndim != 1 or inv_freq.device != device:
        raise ValueError("rope: inv_freq must be an fp32 vector on the query's device")
    if rotary > d:
        raise ValueError(f"rope: {rotary} rotary columns do not fit head_dim {d}")
    wide = positions.dtype == torch.int64
    if not (wide or positions.dtype == torch.int32) or positions.device != device:
        raise ValueError("rope: positions must be int32 or int64 on the query's device")
    if positions.numel() != tokens:
        raise ValueError(f"rope: {positions.numel()} positions for {tokens} tokens")
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    q_out = torch.empty(*query.shape, dtype=torch.bfloat16, device=device)
    k_out, k_args = None, (None, 0, 0, 0)
    if key is not None:
        k, k_ts, k_hs = _tokens_view(key)
        if k.shape[0] != tokens or k.shape[2] != d:
            raise ValueError("rope: query and key differ in tokens or head_dim")
        k_out = torch.empty(*key.shape, dtype=torch.bfloat16, device=device)
        k_args = (k.data_ptr(), k_ts, k_hs, k.shape[1])
    check(_lib.load().lr_rope(
        q.data_ptr(), q_ts, q_hs, heads, *k_args, positions.data_ptr(), wide, inv_freq.data_ptr(),
        float(factor), tokens, d, rotary, bool(interleaved), q_out.data_ptr(), ptr(k_out), stream_of(query)), "rope")
    return q_out, k_out
