"""Attention on the sm_100a tcgen05 kernels: the core of the fused DiT block, and packed prompts.

``attention_bshd(query, key, value)`` computes softmax(scale * Q K^T) V for
bf16 [B, S, H, 128] tensors (heads contiguous within a token; the strided
Q/K/V views of a fused QKV projection are used in place), fp32 scores and
softmax, bf16 output [B, S, H, 128]. It stands where FusedAttention calls
diffusers' attention dispatcher (model/fusion.py:55-57). Unsupported inputs
(a mask, another head size, another dtype) raise ValueError; torch's SDPA
remains available as ``fusion.sdpa_bshd`` for callers that need those.

``attention_packed`` is the attention of prompts of different lengths, packed
without padding: causal or full, with grouped key/value heads, and with fewer
queries than keys (a decoding step, a piece of a prompt). ``attention_shared`` is the same for sequences that all
continue one prefix, whose keys and values are stored and read once.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib
from ._lib import check, ptr, stream_of

__all__ = ["attention_bshd", "attention_packed", "attention_shared"]


def _token_view(t: torch.Tensor) -> torch.Tensor:
    """[B, S, H, D] with unit element stride, heads contiguous, batch stride =
    S * token stride and 16-byte aligned rows (what the kernel's TMA maps
    address), else a contiguous copy."""
    b, s, h, d = t.shape
    if (t.stride(3) == 1 and t.stride(2) == d and (b == 1 or t.stride(0) == s * t.stride(1))
            and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0):
        return t
    return t.contiguous()


def attention_bshd(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, attn_mask=None,
                   scale: float | None = None) -> torch.Tensor:
    if attn_mask is not None:
        raise ValueError("attention_bshd: attention masks are not supported by the sm_100a kernel")
    for name, t in (("query", query), ("key", key), ("value", value)):
        if t.dtype != torch.bfloat16 or not t.is_cuda or t.ndim != 4:
            raise ValueError(f"attention_bshd: {name} must be a CUDA bf16 [B, S, H, D] tensor")
    b, sq, h, d = query.shape
    if key.shape[0] != b or key.shape[2:] != (h, d) or value.shape != key.shape:
        raise ValueError("attention_bshd: query/key/value shapes disagree")
    if d != 128:
        raise ValueError(f"attention_bshd: head_dim {d} (the kernel handles 128)")
    skv = key.shape[1]
    query, key, value = _token_view(query), _token_view(key), _token_view(value)
    out = torch.empty((b, sq, h, d), device=query.device, dtype=torch.bfloat16)
    sc = 1.0 / math.sqrt(d) if scale is None else float(scale)
    check(_lib.load().lr_attention_bf16(
        ptr(query), query.stride(1), ptr(key), key.stride(1), ptr(value), value.stride(1), b, sq, skv, h, d, sc,
        ptr(out), out.stride(1), stream_of(query)), "attention_bshd")
    return out


def _head_view(t: torch.Tensor):
    """(t, token stride, head stride) of [tokens, heads, D] with contiguous columns and 16-byte aligned tokens and heads
    that do not overlap (what TMA maps address); of a contiguous copy where t is not so."""
    ts, hs, cs = t.stride()
    d = t.shape[2]
    if cs == 1 and ts % 8 == 0 and hs % 8 == 0 and ts >= d and hs >= d and t.data_ptr() % 16 == 0:
        return t, ts, hs
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.shape[1] * d, d


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device: int, seqs: int, tq: int, tk: int, heads: int, kv_heads: int, d: int) -> int:
    """lr_attention_packed's need for these counts on this device (a function of them alone)."""
    return _lib.load().lr_attention_packed_workspace_bytes(seqs, tq, tk, heads, kv_heads, d)


def attention_packed(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cu_seqlens_q: torch.Tensor,
                     cu_seqlens_k: torch.Tensor | None = None, *, causal: bool = True,
                     scale: float | None = None) -> torch.Tensor:
    """Attention of packed sequences of different lengths -> bf16 [tokens, heads, D].

    query [Tq, heads, D], key and value [Tk, kv_heads, D]: bf16, D 64 or 128, strided views are used in place; heads a
    multiple of kv_heads (query head h reads key/value head h // (heads / kv_heads)). cu_seqlens_q, cu_seqlens_k: int32
    [sequences + 1] offsets on the device (never read by the host); the keys' default to the queries'. ``causal``: the
    queries are the last ones of their sequence, each sees the keys up to its own position (one query a sequence is a
    decoding step). Rows without a visible key, and tokens past the last offset, give zeros. Values of other sequences
    never reach a row; within a sequence, values of masked keys must be finite.

    Kernels are chosen by the average number of queries a sequence: whole prompts and single tokens in one batch are much
    faster as two calls."""
    device = query.device
    for name, t in (("query", query), ("key", key), ("value", value)):
        if t.dtype != torch.bfloat16 or t.ndim != 3 or not t.is_cuda:
            raise ValueError(f"attention_packed: {name} must be a CUDA bf16 [tokens, heads, D] tensor")
    if key.device != device or value.device != device:
        raise ValueError("attention_packed: query, key and value are on different devices")
    tq, h, d = query.shape
    tk, hk, dk = key.shape
    if value.shape != key.shape or dk != d:
        raise ValueError("attention_packed: query/key/value shapes disagree")
    if d not in (64, 128):
        raise ValueError(f"attention_packed: head_dim {d} (the kernel handles 64 and 128)")
    if hk == 0 or h == 0 or h % hk:
        raise ValueError(f"attention_packed: {h} query heads do not share {hk} key/value heads evenly")
    if cu_seqlens_k is None:
        if tk != tq:
            raise ValueError("attention_packed: cu_seqlens_k is needed where queries and keys differ in tokens")
        cu_seqlens_k = cu_seqlens_q
    count = cu_seqlens_q.numel()
    for t in (cu_seqlens_q, cu_seqlens_k):
        if t.dtype != torch.int32 or t.ndim != 1 or count < 2 or t.device != device:
            raise ValueError("attention_packed: cu_seqlens must be int32 [sequences + 1] on the query's device")
    if cu_seqlens_k.numel() != count:
        raise ValueError("attention_packed: cu_seqlens_q and cu_seqlens_k differ in sequences")
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    (query, q_ts, q_hs), (key, k_ts, k_hs), (value, v_ts, v_hs) = _head_view(query), _head_view(key), _head_view(value)
    out = torch.empty(tq, h, d, dtype=torch.bfloat16, device=device)
    sc = 1.0 / math.sqrt(d) if scale is None else float(scale)
    lib, seqs = _lib.load(), count - 1
    need = _workspace_bytes(query.get_device(), seqs, tq, tk, h, hk, d)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    check(lib.lr_attention_packed(
        query.data_ptr(), q_ts, q_hs, key.data_ptr(), k_ts, k_hs, value.data_ptr(), v_ts, v_hs, cu_seqlens_q.data_ptr(),
        cu_seqlens_k.data_ptr(), seqs, tq, tk, h, hk, d, bool(causal), sc, out.data_ptr(), ptr(workspace), need,
        stream_of(query)), "attention_packed")
    return out


@functools.lru_cache(maxsize=4096)
def _shared_workspace_bytes(device: int, seqs: int, tq: int, tk: int, prefix: int, heads: int, kv_heads: int, d: int) -> int:
    """lr_attention_shared's need for these counts on this device (a function of them alone)."""
    return _lib.load().lr_attention_shared_workspace_bytes(seqs, tq, tk, prefix, heads, kv_heads, d)


def attention_shared(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, prefix_key: torch.Tensor,
                     prefix_value: torch.Tensor, cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor | None = None, *,
                     causal: bool = True, scale: float | None = None) -> torch.Tensor:
    """Attention of packed sequences that all continue one prefix -> bf16 [tokens, heads, D].

    As ``attention_packed``, with prefix_key and prefix_value bf16 [prefix, kv_heads, D] in front of every sequence's keys:
    each query sees the whole prefix and, of its own sequence's keys, those that ``attention_packed`` shows it (a query
    that sees none of those still sees the prefix; tokens past the last offset give zeros). The prefix's
    keys and values are shared by all sequences, not copied; a single length for it, known to the host. Values of other
    sequences never reach a row; within a sequence, values of masked keys must be finite.

    Scores, softmax and sums are fp32; the probabilities, of at most 2^8 before they are divided by their sum, are rounded to bf16 for the
    second product. Kernels are chosen by counts alone: the average number of queries and keys a sequence, and the prefix."""
    device = query.get_device()
    given = (query, key, value, prefix_key, prefix_value)
    for t, name in zip(given, ("query", "key", "value", "prefix_key", "prefix_value")):
        if t.dtype is not torch.bfloat16 or t.ndim != 3 or not t.is_cuda:
            raise ValueError(f"attention_shared: {name} must be a CUDA bf16 [tokens, heads, D] tensor")
        if t.get_device() != device:
            raise ValueError("attention_shared: query, keys and values are on different devices")
    tq, h, d = query.shape
    tk, hk, dk = shape = key.shape
    prefix, *rest = prefix_shape = prefix_key.shape
    if value.shape != shape or dk != d or prefix_value.shape != prefix_shape or rest != [hk, dk]:
        raise ValueError("attention_shared: query/key/value/prefix shapes disagree")
    if d not in (64, 128):
        raise ValueError(f"attention_shared: head_dim {d} (the kernel handles 64 and 128)")
    if hk == 0 or h == 0 or h % hk:
        raise ValueError(f"attention_shared: {h} query heads do not share {hk} key/value heads evenly")
    if cu_seqlens_k is None:
        if tk != tq:
            raise ValueError("attention_shared: cu_seqlens_k is needed where queries and keys differ in tokens")
        cu_seqlens_k = cu_seqlens_q
    if prefix == 0:
        return attention_packed(query, key, value, cu_seqlens_q, cu_seqlens_k, causal=causal, scale=scale)
    count = cu_seqlens_q.numel()
    for t in (cu_seqlens_q, cu_seqlens_k):
        if t.dtype is not torch.int32 or t.ndim != 1 or count < 2 or t.get_device() != device:
            raise ValueError("attention_shared: cu_seqlens must be int32 [sequences + 1] on the query's device")
    if cu_seqlens_k.numel() != count:
        raise ValueError("attention_shared: cu_seqlens_q and cu_seqlens_k differ in sequences")
    if device != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return attention_shared(*given, cu_seqlens_q, cu_seqlens_k, causal=causal, scale=scale)
    operands, kept = [], []  # pointer, token and head stride of each; the copies among them
    for t in given:
        ts, hs, cs = t.stride()
        at = t.data_ptr()
        if cs != 1 or ts % 8 or hs % 8 or ts < d or hs < d or at % 16:  # as in _head_view
            t = t.clone(memory_format=torch.contiguous_format)
            kept.append(t)
            at, ts, hs = t.data_ptr(), t.shape[1] * d, d
        operands += (at, ts, hs)
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    need = _shared_workspace_bytes(device, count - 1, tq, tk, prefix, h, hk, d)
    workspace = torch.empty(need, dtype=torch.uint8, device=query.device) if need else None
    check(_lib.load().lr_attention_shared(
        *operands, cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), count - 1, tq, tk, prefix, h, hk, d, bool(causal),
        1.0 / math.sqrt(d) if scale is None else float(scale), out.data_ptr(), ptr(workspace), need, stream_of(query)),
        "attention_shared")
    return out
