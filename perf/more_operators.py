"""Workloads of serving many requests at once: attention behind a shared prefix, and low-rank adapters of many requests.

Every case runs in two forms: ``own`` false computes it with elementary torch operations in fp32 and rounds once at
the end; ``own`` true calls this package's entry points on the same inputs. ``exact`` restates each operator in 64 bits.

Layouts shared by both forms:
  * packed sequences: tokens of all sequences one after another, int32 offsets ``cu`` [sequences + 1]; the keys of the
    shared prefix stand in a tensor of their own, in front of every sequence's keys;
  * adapters: ``down`` [adapters, rank, in], ``up`` [adapters, out, rank], a scale for each, and for each token the number
    of its adapter, -1 for none.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # Four requests behind a text context of 512 keys, one new token each: latency.
        dict(name="prefix 512 4x1 tokens", op="attention", prefix=512, seqs=4, shortest=1, longest=64, queries=1,
             heads=32, kv_heads=8, head_dim=128),
        # A serving step: 64 requests behind one long instruction, each with an answer of its own under way.
        dict(name="prefix 8192 64x1 tokens", op="attention", prefix=8192, seqs=64, shortest=64, longest=1024,
             queries=1, heads=32, kv_heads=8, head_dim=128),
        # A large batch with one head of keys for each head of queries, 64 wide, behind a prefix of odd length.
        dict(name="prefix 2011 256x1 tokens d64", op="attention", prefix=2011, seqs=256, shortest=1, longest=512,
             queries=1, heads=24, kv_heads=24, head_dim=64),
        # Eight tokens a request at once (drafts to be checked) behind a document.
        dict(name="prefix 16384 32x8 tokens", op="attention", prefix=16384, seqs=32, shortest=8, longest=300,
             queries=8, heads=32, kv_heads=8, head_dim=128),
        # Prompts of very different lengths behind a template.
        dict(name="prefix 1000 48 prompts", op="attention", prefix=1000, seqs=48, shortest=1, longest=512, queries=0,
             heads=32, kv_heads=8, head_dim=128),
        # Long prompts behind a long document: the largest call, bound by the tensor cores.
        dict(name="prefix 8192 8 prompts", op="attention", prefix=8192, seqs=8, shortest=512, longest=2048, queries=0,
             heads=32, kv_heads=8, head_dim=128),
        # One token through the adapter of a fused query-key-value projection: latency.
        dict(name="adapters 1x6144 to 18432 r16", op="adapters", tokens=1, requests=1, adapters=8, rank=16, width=6144,
             outputs=18432),
        # A serving step in which every request has an adapter of its own, beside the text context's projection.
        dict(name="adapters 64x4096 of 64 r16", op="adapters", tokens=64, requests=64, adapters=64, rank=16,
             width=4096, outputs=12288),
        # A large serving step over a few adapters of high rank.
        dict(name="adapters 256x6144 of 8 r64", op="adapters", tokens=256, requests=256, adapters=8, rank=64,
             width=6144, outputs=6144),
        # Packed prompts of 24 requests; a small rank.
        dict(name="adapters 2500x4096 of 24 r8", op="adapters", tokens=2500, requests=24, adapters=24, rank=8,
             width=4096, outputs=12288),
        # One context of 512 tokens through an adapter of the highest rank.
        dict(name="adapters 512x4096 of 1 r128", op="adapters", tokens=512, requests=1, adapters=1, rank=128,
             width=4096, outputs=4096),
        # Two requests' shares of a latent through the feed-forward's first projection: bound by the base rows' traffic.
        dict(name="adapters 12240x6144 of 2 r32", op="adapters", tokens=12240, requests=2, adapters=2, rank=32,
             width=6144, outputs=24576),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        head_dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
        heads = max(kv_heads, min(heads, 32) // kv_heads * kv_heads)
        if rng.random() < 0.4:  # whole prompts
            prefix = _spread(rng, 16, 8192)
            longest = _spread(rng, 1, 2048)
            seqs = _spread(rng, 1, max(1, min(64, 8000 // longest)))
            queries = 0
        else:  # the last one to eight tokens of each request
            prefix = _spread(rng, 16, 32768)
            longest = _spread(rng, 1, 4096)
            seqs = _spread(rng, 1, max(1, min(256, 60000 // longest)))
            queries = rng.choice([1, 1, 1, 2, 5, 8])
        return dict(op="attention", prefix=prefix, seqs=seqs, shortest=max(1, longest // 40), longest=longest, queries=queries,
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim)
    adapters = _spread(rng, 1, 64)
    if rng.random() < 0.5:  # one token a request
        tokens = requests = _spread(rng, 1, 256)
    else:
        tokens = _spread(rng, 64, 12240)
        requests = _spread(rng, 1, 32)
    outputs = _spread(rng, 128, 18432)
    if rng.random() < 0.75:
        outputs = -(-outputs // 8) * 8
    return dict(op="adapters", tokens=tokens, requests=requests, adapters=adapters, rank=8 * _spread(rng, 1, 16),
                width=32 * _spread(rng, 4, 192), outputs=outputs)


# ------------------------------------------------------------------ the cases' data
def _lengths(case):
    """Own key lengths of the sequences, spread over [shortest, longest] on a logarithmic scale; one is the longest."""
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


def _token_adapters(case):
    """The adapter of every token: requests are runs of tokens; about one in ten has none where there are several."""
    rng = random.Random(case["tokens"] * 1000003 + case["adapters"])
    tokens, requests = case["tokens"], min(case["requests"], case["tokens"])
    cuts = [0] + sorted(rng.sample(range(1, tokens), requests - 1)) + [tokens]
    got = []
    for i in range(requests):
        number = i % case["adapters"] if requests <= case["adapters"] else rng.randrange(case["adapters"])
        if requests > 4 and rng.random() < 0.1:
            number = -1
        got += [number] * (cuts[i + 1] - cuts[i])
    return got


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
        s["prefix_k"] = normal(case["prefix"], hk, d).bfloat16()
        s["prefix_v"] = normal(case["prefix"], hk, d).bfloat16()
    else:
        n, k, e, r = case["outputs"], case["width"], case["adapters"], case["rank"]
        s["x"] = normal(case["tokens"], k).bfloat16()
        s["base"] = normal(case["tokens"], n).bfloat16()
        s["down"] = (normal(e, r, k) * k ** -0.5).bfloat16()
        s["up"] = (normal(e, n, r) * (0.3 * r ** -0.5)).bfloat16()
        s["scale"] = torch.rand(e, generator=g, device=DEVICE) * 1.5 + 0.5
        s["index"] = torch.tensor(_token_adapters(case), dtype=torch.int32, device=DEVICE)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def _own_attention(s):
    from lynnreal_omni_b200.attention import attention_shared
    return attention_shared(s["q"], s["k"], s["v"], s["prefix_k"], s["prefix_v"], s["cu_q"], s["cu_k"], causal=True)


def _own_adapters(s):
    from lynnreal_omni_b200.adapters import add_adapters
    return add_adapters(s["base"], s["x"], s["down"], s["up"], s["index"], s["scale"])


_OWN = {"attention": _own_attention, "adapters": _own_adapters}


def _plain_attention(s):
    """Every query against the prefix and against every sequence's keys, those of other sequences and of later positions
    masked; one softmax over both."""
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
    qf = q.float().unflatten(1, (hk, h // hk)).permute(1, 2, 0, 3).reshape(hk, -1, d) * d ** -0.5  # [kv head, group x query, d]
    mine = torch.matmul(qf, k.float().permute(1, 2, 0)).unflatten(1, (h // hk, tq))
    mine = mine.masked_fill_(hidden, -math.inf).flatten(1, 2)
    shared = torch.matmul(qf, s["prefix_k"].float().permute(1, 2, 0))
    top = torch.maximum(mine.amax(-1, keepdim=True), shared.amax(-1, keepdim=True))
    mine.sub_(top).exp_()
    shared.sub_(top).exp_()
    total = mine.sum(-1, keepdim=True) + shared.sum(-1, keepdim=True)
    out = torch.matmul(mine, v.float().permute(1, 0, 2)) + torch.matmul(shared, s["prefix_v"].float().permute(1, 0, 2))
    return (out / total).unflatten(1, (h // hk, tq)).permute(2, 0, 1, 3).reshape(tq, h, d).bfloat16()


def _plain_adapters(s):
    """Adapter by adapter over all tokens, those of other adapters masked."""
    x, out = s["x"].float(), s["base"].float()
    for number in range(s["case"]["adapters"]):
        mine = (s["index"] == number).float()[:, None]
        inner = torch.matmul(x, s["down"][number].float().t()) * (s["scale"][number] * mine)
        out.addmm_(inner, s["up"][number].float().t())
    return out.bfloat16()


_PLAIN = {"attention": _plain_attention, "adapters": _plain_adapters}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "attention":
        lk, lq = _lengths(case), _query_lengths(case)
        pairs = sum(q * k - q * (q - 1) // 2 for q, k in zip(lq, lk)) + sum(lq) * case["prefix"]
        d = case["head_dim"]
        return {"bytes": 4 * sum(lq) * case["heads"] * d + 4 * (sum(lk) + case["prefix"]) * case["kv_heads"] * d,
                "flops": 4 * pairs * case["heads"] * d}
    n, k, r = case["outputs"], case["width"], case["rank"]
    index = _token_adapters(case)
    used, adapted = len(set(index) - {-1}), sum(i >= 0 for i in index)
    return {"bytes": 2 * adapted * k + 4 * len(index) * n + used * 2 * r * (n + k), "flops": 2 * adapted * r * (n + k)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attention(s) if case["op"] == "attention" else _exact_adapters(s)


def _exact_attention(s):
    """One sequence and one head of keys at a time: prefix and own keys one after another."""
    q, k, v = s["q"], s["k"], s["v"]
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    group, prefix = q.shape[1] // k.shape[1], s["prefix_k"].shape[0]
    out = torch.empty(q.shape, device=DEVICE, dtype=torch.float64)
    for hk in range(k.shape[1]):
        pk, pv = s["prefix_k"][:, hk].double(), s["prefix_v"][:, hk].double()
        for b in range(len(cu_q) - 1):
            lq, lk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
            kb, vb = (torch.cat((p, t[cu_k[b]:cu_k[b + 1], hk].double())) for p, t in ((pk, k), (pv, v)))
            at = slice(cu_q[b], cu_q[b + 1])
            qb = q[at, hk * group:(hk + 1) * group].double()
            scores = torch.einsum("ngd,kd->gnk", qb, kb) / math.sqrt(q.shape[2])
            reach = prefix + torch.arange(lq, device=DEVICE)[:, None] + lk - lq
            scores = scores.masked_fill(torch.arange(prefix + lk, device=DEVICE) > reach, -math.inf)
            out[at, hk * group:(hk + 1) * group] = torch.einsum("gnk,kd->ngd", scores.softmax(-1), vb)
    return out


def _exact_adapters(s):
    """The rows of one adapter at a time."""
    out = s["base"].double()
    for number in sorted(set(s["index"].tolist()) - {-1}):
        rows = (s["index"] == number).nonzero()[:, 0]
        inner = torch.einsum("tk,rk->tr", s["x"][rows].double(), s["down"][number].double())
        out[rows] += s["scale"][number].double() * torch.einsum("tr,nr->tn", inner, s["up"][number].double())
    return out
