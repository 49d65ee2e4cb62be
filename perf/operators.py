"""Workloads of the prompt-path operators: packed causal attention, rotary positions and 4-bit floating-point projections.

Every case runs in two forms: ``own`` false computes it with elementary torch operations in fp32 and rounds once at
the end; ``own`` true calls this package's entry points on the same inputs. ``exact`` restates each operator in 64 bits.

Layouts shared by both forms:
  * packed sequences: tokens of all sequences one after another, int32 offsets ``cu`` [sequences + 1];
  * 4-bit codes: two e2m1 values per byte, the even column in the low nibble;
  * block scales: bytes [ceil(rows / 128), ceil(blocks / 4), 32, 4, 4], element [R, C, r, j, c] being the scale of row
    128 R + 32 j + r and block 4 C + c (the order in which the tensor core reads them; zeros past the matrix).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # One 512-token prompt, the text context's length and width (32 x 128 = 4096): the smallest whole-prompt call.
        dict(name="attention prompt 512", op="attention", seqs=1, shortest=512, longest=512, queries=0, heads=32,
             kv_heads=8, head_dim=128),
        # A batch of prompts of very different lengths, one head of keys for each head of queries, 64 wide.
        dict(name="attention packed ragged d64", op="attention", seqs=16, shortest=1, longest=2048, queries=0, heads=24,
             kv_heads=24, head_dim=64),
        # One long document as a prompt: the largest call, bound by the tensor cores.
        dict(name="attention prompt 16384", op="attention", seqs=1, shortest=16384, longest=16384, queries=0, heads=32,
             kv_heads=8, head_dim=128),
        # A serving step: one new token for each of 64 requests whose contexts differ, bound by reading keys and values.
        dict(name="attention 64 requests 1 token", op="attention", seqs=64, shortest=256, longest=8192, queries=1, heads=32,
             kv_heads=8, head_dim=128),
        # One new token of one request with a long context: latency, and the split of one row over the GPU.
        dict(name="attention 1 request 1 token", op="attention", seqs=1, shortest=32768, longest=32768, queries=1, heads=32,
             kv_heads=8, head_dim=128),
        # One token at a far position: the smallest rotary call.
        dict(name="rope 1 token", op="rope", tokens=1, heads=32, kv_heads=8, head_dim=128, rotary=128, interleaved=False,
             scaling=1.0, last=100000),
        # A long packed prompt, interleaved pairs over half of each head, scaled fourfold.
        dict(name="rope 16384 tokens interleaved", op="rope", tokens=16384, heads=32, kv_heads=8, head_dim=128, rotary=64,
             interleaved=True, scaling=4.0, last=16384),
        # The activations of one latent (12240 tokens) quantised to blocks of 16 and read back.
        dict(name="fp4 rows 12240x6144 nvfp4", op="rows", rows=12240, width=6144, format="nvfp4"),
        # A few rows of a wide feed-forward activation in blocks of 32: latency.
        dict(name="fp4 rows 37x24576 mxfp4", op="rows", rows=37, width=24576, format="mxfp4"),
        # One token through the fused query-key-value projection: bound by reading the weight.
        dict(name="fp4 linear 1x6144 to 18432", op="linear", rows=1, width=6144, outputs=18432, format="nvfp4", bias=True),
        # The text context (512 x 4096) through a projection of its own width's triple.
        dict(name="fp4 linear 512x4096 to 12288 mx", op="linear", rows=512, width=4096, outputs=12288, format="mxfp4",
             bias=False),
        # The feed-forward's first projection over one latent: bound by the tensor cores.
        dict(name="fp4 linear 12240x6144 to 24576", op="linear", rows=12240, width=6144, outputs=24576, format="nvfp4",
             bias=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rope", "rows", "linear", "linear"])
    if op == "attention":
        head_dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
        heads = max(kv_heads, min(heads, 32) // kv_heads * kv_heads)
        if rng.random() < 0.5:  # whole prompts
            longest = _spread(rng, 1, 6000)
            seqs = _spread(rng, 1, max(1, min(64, 12000 // longest)))
            queries = 0
        else:  # the last one to eight tokens of each request
            longest = _spread(rng, 8, 32768)
            seqs = _spread(rng, 1, max(1, min(64, 200000 // longest)))
            queries = rng.choice([1, 1, 2, 5, 8])
        return dict(op=op, seqs=seqs, shortest=max(1, queries, longest // 40), longest=longest, queries=queries, heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim)
    if op == "rope":
        head_dim = rng.choice([64, 96, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        return dict(op=op, tokens=_spread(rng, 1, 16384), heads=kv_heads * rng.choice([1, 3, 4]), kv_heads=kv_heads,
                    head_dim=head_dim, rotary=rng.choice([32, head_dim // 2, head_dim]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice([1.0, 2.0, 8.0]), last=_spread(rng, 16384, 500000))
    format = rng.choice(["nvfp4", "mxfp4"])
    if op == "rows":
        return dict(op=op, rows=_spread(rng, 1, 12240), width=32 * _spread(rng, 2, 192), format=format)
    return dict(op=op, rows=_spread(rng, 1, 12240), width=32 * _spread(rng, 4, 192), outputs=_spread(rng, 128, 18432), format=format,
                bias=rng.random() < 0.5)


# ------------------------------------------------------------------ the cases' data
def _lengths(case):
    """Key lengths of the sequences, spread over [shortest, longest] on a logarithmic scale; one is the longest."""
    rng = random.Random(case["seqs"] * 1000003 + case["longest"])
    got = [_spread(rng, case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    got[rng.randrange(len(got))] = case["longest"]
    return got


def _query_lengths(case):
    return [min(n, case["queries"]) if case["queries"] else n for n in _lengths(case)]


def _offsets(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device=DEVICE)


def _block(case):
    return 16 if case["format"] == "nvfp4" else 32


def _inverse_frequencies(case):
    """1 / base^(2 i / rotary), the slow half of them divided by the scaling factor through a linear ramp over the index."""
    half = case["rotary"] // 2
    i = torch.arange(half, dtype=torch.float64)
    f = 10000.0 ** (-i / half)
    keep = (1 - i / max(1, half - 1)).clamp(0, 1)
    return (f * keep + f / case["scaling"] * (1 - keep)).float().to(DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)

    s = {"case": case}
    if case["op"] == "attention":
        d, h, hk = case["head_dim"], case["heads"], case["kv_heads"]
        lk, lq = _lengths(case), _query_lengths(case)
        s["cu_k"], s["cu_q"] = _offsets(lk), _offsets(lq)
        s["q"] = normal(sum(lq), h, d).bfloat16()
        s["k"] = normal(sum(lk), hk, d).bfloat16()
        s["v"] = normal(sum(lk), hk, d).bfloat16()
    elif case["op"] == "rope":
        n, d, h, hk = case["tokens"], case["head_dim"], case["heads"], case["kv_heads"]
        # a fused query-key-value projection's output, of which query and key are strided views
        qkv = normal(n, (h + 2 * hk) * d).bfloat16()
        s["q"] = qkv[:, : h * d].unflatten(1, (h, d))
        s["k"] = qkv[:, h * d:(h + hk) * d].unflatten(1, (hk, d))
        first = case["last"] - n if n > 1 else case["last"]
        s["positions"] = torch.arange(first, first + n, device=DEVICE, dtype=torch.int64)
        s["inv_freq"] = _inverse_frequencies(case)
        s["factor"] = 1.0 if case["scaling"] == 1.0 else 0.1 * math.log(case["scaling"]) + 1.0
    else:
        rows, width = case["rows"], case["width"]
        x = normal(rows, width)
        x[:, torch.rand(width, generator=g, device=DEVICE) < 0.005] *= 20  # outlier channels
        s["x"] = x.bfloat16()
        if case["op"] == "linear":
            n, blocks = case["outputs"], width // _block(case)
            s["codes"] = torch.randint(0, 256, (n, width // 2), generator=g, device=DEVICE, dtype=torch.uint8)
            low, high = (32, 96) if case["format"] == "nvfp4" else (119, 125)  # e4m3 2^-3 .. 32; e8m0 2^-8 .. 2^-3
            plain = torch.randint(low, high, (n, blocks), generator=g, device=DEVICE, dtype=torch.uint8)
            s["scales"] = _tiled(plain)
            s["column_scale"] = None
            if case["format"] == "nvfp4":
                s["column_scale"] = torch.rand(n, generator=g, device=DEVICE) * 1.5e-3 + 0.5e-3
            s["bias"] = (0.02 * normal(n)).bfloat16() if case["bias"] else None
    return s


def _tiled(plain):
    """[rows, blocks] scale bytes in the tensor core's order, zeros past the matrix."""
    rows, blocks = plain.shape
    whole = torch.zeros((-(-rows // 128) * 128, -(-blocks // 4) * 4), dtype=torch.uint8, device=plain.device)
    whole[:rows, :blocks] = plain
    return whole.unflatten(0, (-1, 4, 32)).unflatten(3, (-1, 4)).permute(0, 3, 2, 1, 4).contiguous()


def _untiled(scales, rows, blocks):
    return scales.permute(0, 3, 2, 1, 4).flatten(3, 4).flatten(0, 2)[:rows, :blocks]


# ------------------------------------------------------------------ one pass
def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def _own_attention(s):
    from lynnreal_omni_b200.attention import attention_packed
    return attention_packed(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=True)


def _own_rope(s):
    from lynnreal_omni_b200.rotary import rope
    return rope(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["case"]["interleaved"], factor=s["factor"])


def _own_rows(s):
    from lynnreal_omni_b200.fp4 import dequantize_rows_fp4, quantize_rows_fp4
    codes, scales, row_scale = quantize_rows_fp4(s["x"], format=s["case"]["format"])
    return dequantize_rows_fp4(codes, scales, row_scale, format=s["case"]["format"])


def _own_linear(s):
    from lynnreal_omni_b200.fp4 import fp4_matmul, quantize_rows_fp4
    codes, scales, row_scale = quantize_rows_fp4(s["x"], format=s["case"]["format"])
    return fp4_matmul(codes, scales, s["codes"], s["scales"], row_scale, s["column_scale"], s["bias"],
                      format=s["case"]["format"])


_OWN = {"attention": _own_attention, "rope": _own_rope, "rows": _own_rows, "linear": _own_linear}


def _plain_attention(s):
    """Every query against every key, the pairs of other sequences and of later positions masked."""
    q, k, v, cu_q, cu_k = (s[n] for n in ("q", "k", "v", "cu_q", "cu_k"))
    tq, h, d = q.shape
    tk, hk, _ = k.shape
    at_q = torch.arange(tq, device=q.device, dtype=torch.int32)
    at_k = torch.arange(tk, device=q.device, dtype=torch.int32)
    seq_q = torch.searchsorted(cu_q, at_q, right=True) - 1
    seq_k = torch.searchsorted(cu_k, at_k, right=True) - 1
    # a query's last visible key: queries are the last tokens of their sequence
    last = cu_k[seq_q + 1] - (cu_q[seq_q + 1] - at_q)
    hidden = (seq_q[:, None] != seq_k) | (at_k > last[:, None])
    qf = q.float().unflatten(1, (hk, h // hk)).permute(1, 2, 0, 3).reshape(hk, -1, d)  # [kv head, group x query, d]
    scores = torch.matmul(qf, k.float().permute(1, 2, 0)).mul_(d ** -0.5).unflatten(1, (h // hk, tq))
    scores.masked_fill_(hidden, -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.flatten(1, 2), v.float().permute(1, 0, 2)).unflatten(1, (h // hk, tq)) / total
    return out.permute(2, 0, 1, 3).reshape(tq, h, d).bfloat16()


def _rotated(x, cos, sin, rotary, interleaved):
    x = x.float()
    part, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., : rotary // 2], part[..., rotary // 2:]
        part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((part, rest), -1).bfloat16()


def _plain_rope(s):
    c = s["case"]
    angle = (s["positions"].float()[:, None] * s["inv_freq"])[:, None]
    cos, sin = angle.cos() * s["factor"], angle.sin() * s["factor"]
    return tuple(_rotated(x, cos, sin, c["rotary"], c["interleaved"]) for x in (s["q"], s["k"]))


def _e2m1(x):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with x's sign, ties to the even code."""
    a = x.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6), x)


def _power(e):
    """2^e in fp32 for whole numbers e in [-127, 127], exactly."""
    e = e.int()
    return ((e.clamp(min=-126) + 127) << 23).view(torch.float32) * torch.where(e < -126, 0.5, 1.0)


def _quantized(x, format):
    """The values that the 4-bit form of x's rows stands for, in fp32."""
    x = x.float()
    if format == "nvfp4":
        most = x.abs().amax(1, keepdim=True).clamp(min=1e-8)
        b = x.unflatten(1, (-1, 16))
        stored = (b.abs().amax(2) * 448 / most).to(torch.float8_e4m3fn).float()
        # 2688 / .. by a tensor: a true division, of which ties between two codes come out as ties
        inverse = torch.where(stored == 0, 0, torch.full_like(stored, 2688) / (stored * most))
        scale = stored * (most * (1 / 2688))
    else:
        b = x.unflatten(1, (-1, 32))
        exponent = (torch.frexp(b.abs().amax(2))[1] - 3).clamp(-127, 127)
        exponent = torch.where(b.abs().amax(2) == 0, -127, exponent)
        scale, inverse = _power(exponent), _power(-exponent)
    return (_e2m1(b * inverse[..., None]) * scale[..., None]).flatten(1)


def _plain_rows(s):
    return _quantized(s["x"], s["case"]["format"]).bfloat16()


def _plain_weight(s):
    c = s["case"]
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=DEVICE)
    w = values[torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).flatten(1).int()]
    raw = _untiled(s["scales"], c["outputs"], c["width"] // _block(c))
    scale = raw.view(torch.float8_e4m3fn).float() if c["format"] == "nvfp4" else _power(raw.int() - 127)
    return (w.unflatten(1, (-1, _block(c))) * scale[..., None]).flatten(1)


def _plain_linear(s):
    y = torch.matmul(_quantized(s["x"], s["case"]["format"]), _plain_weight(s).t())
    if s["column_scale"] is not None:
        y = y * s["column_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.bfloat16()


_PLAIN = {"attention": _plain_attention, "rope": _plain_rope, "rows": _plain_rows, "linear": _plain_linear}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "attention":
        lk, lq = _lengths(case), _query_lengths(case)
        pairs = sum(q * k - q * (q - 1) // 2 for q, k in zip(lq, lk))
        d = case["head_dim"]
        return {"bytes": 4 * sum(lq) * case["heads"] * d + 4 * sum(lk) * case["kv_heads"] * d,
                "flops": 4 * pairs * case["heads"] * d}
    if case["op"] == "rope":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 4 * values + 8 * case["tokens"], "flops": 3 * values * case["rotary"] // case["head_dim"]}
    values = case["rows"] * case["width"]
    packed = 0.5 + 1 / _block(case)
    if case["op"] == "rows":  # quantised (2 bytes in, the packed form out) and read back (the other way round)
        return {"bytes": values * (4 + 2 * packed), "flops": 4 * values}
    n, k = case["outputs"], case["width"]
    return {"bytes": values * (2 + 2 * packed) + n * k * packed + 2 * case["rows"] * n, "flops": 2 * case["rows"] * n * k}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "rope":
        return tuple(_exact_rope(s, x) for x in (s["q"], s["k"]))
    x = _exact_quantized(s["x"].double(), case["format"])
    if case["op"] == "rows":
        return x
    grid = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], device=DEVICE, dtype=torch.float64) / 2
    w = torch.empty((case["outputs"], case["width"]), device=DEVICE, dtype=torch.float64)
    for odd in (0, 1):
        code = (s["codes"].long() >> (4 * odd)) & 15
        w[:, odd::2] = grid[code & 7] * (1 - 2 * (code >> 3))
    n, block = case["outputs"], _block(case)
    for c in range(case["width"] // block):
        tile = s["scales"][:, c // 4, :, :, c % 4]  # [row tile, row in 32, 32-row group]
        raw = tile.transpose(1, 2).reshape(-1)[:n].long()
        if case["format"] == "nvfp4":
            e, m = (raw >> 3) & 15, (raw & 7).double()
            scale = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * _exact_power(e - 10))
        else:
            scale = _exact_power(raw - 127)
        w[:, c * block:(c + 1) * block] *= scale[:, None]
    y = x @ w.t()
    if s["column_scale"] is not None:
        y *= s["column_scale"].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    return y


def _exact_power(e):
    """2^e in 64 bits for whole numbers e, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_attention(s):
    """One sequence and one head of keys at a time."""
    q, k, v = s["q"], s["k"], s["v"]
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    group = q.shape[1] // k.shape[1]
    out = torch.empty(q.shape, device=DEVICE, dtype=torch.float64)
    for b in range(len(cu_q) - 1):
        lq, lk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        for hk in range(k.shape[1]):
            kb, vb = (t[cu_k[b]:cu_k[b + 1], hk].double() for t in (k, v))
            for first in range(0, lq, 4096):
                at = slice(cu_q[b] + first, cu_q[b] + min(lq, first + 4096))
                n = at.stop - at.start
                qb = q[at, hk * group:(hk + 1) * group].double()
                scores = torch.einsum("ngd,kd->gnk", qb, kb) / math.sqrt(q.shape[2])
                reach = torch.arange(n, device=DEVICE)[:, None] + first + lk - lq
                scores = scores.masked_fill(torch.arange(lk, device=DEVICE) > reach, -math.inf)
                out[at, hk * group:(hk + 1) * group] = torch.einsum("gnk,kd->ngd", scores.softmax(-1), vb)
    return out


def _exact_rope(s, x):
    c, x = s["case"], x.double()
    angle = torch.outer(s["positions"].double(), s["inv_freq"].double())[:, None]
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)
    half = c["rotary"] // 2
    if c["interleaved"]:
        first, second = torch.arange(half) * 2, torch.arange(half) * 2 + 1
    else:
        first, second = torch.arange(half), torch.arange(half) + half
    z = torch.complex(x[..., first], x[..., second]) * turn
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_quantized(x, format):
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEVICE, dtype=torch.float64)
    # the upper end of each code's interval; a tie goes to the even code
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEVICE, dtype=torch.float64)
    block = 16 if format == "nvfp4" else 32
    out = torch.empty_like(x)
    row = x.abs().amax(1).clamp(min=1e-8)
    for c in range(x.shape[1] // block):
        b = x[:, c * block:(c + 1) * block]
        most = b.abs().amax(1)
        if format == "nvfp4":
            t = 448 * most / row
            e = (torch.frexp(t)[1] - 1).clamp(-6, 8)
            unit = _exact_power(e - 3)
            stored, whole = (torch.round(t / unit) * unit).clamp(max=448) * row, 2688
        else:
            stored, whole = _exact_power((torch.frexp(most)[1] - 3).clamp(-127, 127)), 1
        a = (b.abs() * whole / torch.where(stored == 0, 1, stored)[:, None]).where(stored[:, None] > 0, 0)
        scale = stored / whole
        low, high = torch.searchsorted(edges, a), torch.searchsorted(edges, a, right=True)
        code = torch.where(low % 2 == 0, low, high)  # they differ at a tie alone
        out[:, c * block:(c + 1) * block] = grid[code] * torch.sign(b) * scale[:, None]
    return out
