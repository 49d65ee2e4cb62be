"""GPU tests of attention.attention_shared against attention in 64 bits over prefix and own keys one after another.

Tolerance per value, as for attention_packed: probabilities rounded to bf16 (at most 2^-8 each, so 2^-8 of sum p |v|, half of
that on average), the output too (2^-8 |ref|); fp32 sums, exponentials (below 2^-12) and the joining of parts fit in what the
average leaves: 2^-8 (sum p |v| + |ref|).
"""
from __future__ import annotations

import math

import pytest
import torch

from lynnreal_omni_b200 import _lib
from lynnreal_omni_b200.attention import attention_packed, attention_shared
from test_gpu_attention_packed import compare, offsets, tensors

pytestmark = pytest.mark.gpu
DEV = "cuda"


def prefix_tensors(prefix, hk, d, seed=0):
    g = torch.Generator().manual_seed(1000 + seed)
    return [torch.randn(prefix, hk, d, generator=g).bfloat16().to(DEV) for _ in range(2)]


def reference(q, k, v, pk, pv, lq, lk, causal, scale):
    q, k, v, pk, pv = (t.double() for t in (q, k, v, pk, pv))
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    group, prefix = q.shape[1] // k.shape[1], pk.shape[0]
    iq = ik = 0
    for nq, nk in zip(lq, lk):
        for h in range(q.shape[1]):
            own = slice(ik, ik + nk)
            ks, vs = torch.cat((pk[:, h // group], k[own, h // group])), torch.cat((pv[:, h // group], v[own, h // group]))
            s = q[iq:iq + nq, h] @ ks.t() * scale
            if causal:
                last = torch.arange(nq, device=q.device)[:, None] + nk - nq  # of the own keys
                at = torch.arange(nk + prefix, device=q.device) - prefix
                s = s.masked_fill((at > last) & (at >= 0), -math.inf)
            p = s.softmax(-1)
            out[iq:iq + nq, h], size[iq:iq + nq, h] = p @ vs, p @ vs.abs()
        iq, ik = iq + nq, ik + nk
    return out, size


def check(prefix, lq, lk, h, hk, d, causal=True, seed=0, spread=1.0, scale=None):
    q, k, v = tensors(lq, lk, h, hk, d, seed, spread)
    pk, pv = prefix_tensors(prefix, hk, d, seed)
    got = attention_shared(q, k, v, pk, pv, offsets(lq), offsets(lk), causal=causal, scale=scale)
    compare(got, reference(q, k, v, pk, pv, lq, lk, causal, 1 / math.sqrt(d) if scale is None else scale))
    assert _lib.device_status() == 0
    return got


PROMPTS = [[1], [64], [129], [300], [5, 130, 1, 64, 257], [0, 7, 0, 0, 200, 0], [640, 3]]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prefix", [1, 127, 128, 129, 500, 1000])
@pytest.mark.parametrize("lengths", PROMPTS, ids=str)
def test_whole_prompts(lengths, prefix, d):
    check(prefix, lengths, lengths, 4, 2, d, seed=sum(lengths))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("prefix", [1, 128, 333])
def test_many_prompts(prefix, causal, d):
    """Enough blocks that each takes the whole prefix before its own keys; some sequences without keys or queries."""
    lq = [37 * i % 190 + 20 for i in range(60)]
    lk = [0 if i % 7 == 3 else n + 50 * (i % 3) for i, n in enumerate(lq)]
    lq[5] = lq[11] = 0
    check(prefix, lq, lk, 6, 2, d, causal, seed=prefix)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk", [(1, 1), (3, 3), (3, 1), (5, 1), (6, 2), (7, 1), (12, 4), (32, 8), (16, 1), (48, 1), (128, 1),
                                  (130, 1), (200, 1)])
def test_head_groups(h, hk, causal):
    check(200, [3, 150, 41], [3, 150, 41], h, hk, 64, causal)
    check(333, [1, 2, 9], [77, 260, 9], h, hk, 128, causal)
    check(140, [1], [5], h, hk, 128, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1], [3000]), ([1, 1, 1], [5, 3000, 129]), ([2, 5, 8], [2, 700, 1025]),
                                   ([100, 1], [700, 700]), ([1] * 70, list(range(1, 71))), ([4, 4], [3, 0]), ([130], [7]),
                                   ([0, 3], [50, 60]), ([1, 0], [0, 9]), ([20] * 30, [20, 300, 40] * 10),
                                   ([1] * 300, [(7 * i) % 300 for i in range(300)])])
def test_fewer_or_more_queries_than_keys(lq, lk, causal, d):
    """Decoding steps and pieces of prompts; a query without an own key sees the prefix."""
    for prefix in (3, 260, 1111):
        check(prefix, lq, lk, 4, 1, d, causal)


@pytest.mark.parametrize("tokens", [1, 2, 4, 5, 16, 17, 31, 32, 33, 63, 64, 65, 128, 200])
def test_batches_of_single_tokens(tokens):
    """Every way in which the prefix is cut, at its edges."""
    for h, hk in ((4, 1), (8, 8)):
        check(2000, [1] * tokens, [1 + 40 * i % 170 for i in range(tokens)], h, hk, 128, seed=tokens)


@pytest.mark.parametrize("seqs", [31, 32, 33, 256])
def test_many_sequences(seqs):
    lengths = [0 if i % 3 == 2 else 40 + 53 * i % 97 for i in range(seqs)]
    check(300, lengths, lengths, 2, 1, 64, seed=seqs)


@pytest.mark.parametrize("seqs", [127, 128, 129, 2047, 2048, 2049, 66000])
def test_very_many_sequences(seqs):
    """One token and, for two sequences of three, one own key each: every round of the look-up of a slot and a token."""
    g = torch.Generator().manual_seed(seqs)
    lk = torch.tensor([0 if i % 3 == 1 else 1 for i in range(seqs)])
    q, k, v = (torch.randn(n, 1, 64, generator=g).bfloat16().to(DEV) for n in (seqs, int(lk.sum()), int(lk.sum())))
    pk, pv = prefix_tensors(37, 1, 64)
    cu_q, cu_k = torch.arange(seqs + 1, dtype=torch.int32), torch.cat((torch.zeros(1, dtype=torch.int64), lk.cumsum(0))).int()
    got = attention_shared(q, k, v, pk, pv, cu_q.to(DEV), cu_k.to(DEV))
    assert _lib.device_status() == 0
    qd, (kd, vd) = q[:, 0].double(), (torch.zeros(seqs, 64, dtype=torch.float64, device=DEV) for _ in range(2))
    there = (lk == 1).to(DEV)
    kd[there], vd[there] = k[:, 0].double(), v[:, 0].double()
    own = ((qd * kd).sum(-1, keepdim=True) / 8).masked_fill(~there[:, None], -math.inf)
    p = torch.cat((qd @ pk[:, 0].double().t() / 8, own), 1).softmax(-1)
    ref, size = (p[:, :-1] @ x + p[:, -1:] * y for x, y in ((pv[:, 0].double(), vd), (pv[:, 0].double().abs(), vd.abs())))
    compare(got[:, 0], (ref, size))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([100], [100]), ([64] * 4, [64] * 4), ([30, 0, 200], [300, 5, 200]), ([33], [20]), ([90], [0])])
def test_few_prompts_behind_a_long_prefix(lq, lk, causal, d):
    """Prompts whose prefix is cut into parts because their own blocks would not fill the GPU."""
    check(5000, lq, lk, 8, 2, d, causal, seed=d)
    check(3001, lq, lk, 5, 5, d, causal, seed=d)


def test_long():
    check(20000, [1, 1], [5, 700], 8, 1, 128, seed=1)
    check(40000, [1] * 20, [30] * 20, 8, 2, 64, seed=2)
    check(9000, [700], [900], 4, 1, 128, seed=3)
    check(17000, [30, 40], [30, 400], 4, 2, 64, seed=4)


@pytest.mark.parametrize("lq,lk", [([260, 40], [260, 40]), ([1, 1], [600, 400]), ([1] * 40, [60] * 40)])
@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_flat_and_peaked_scores(spread, lq, lk):
    check(700, lq, lk, 4, 2, 128, spread=spread)
    for scale in (0.0, -0.1, 0.5):
        check(300, lq, lk, 4, 2, 64, scale=scale)


CASES = [([40, 30, 60], [40, 30, 60]), ([1, 1, 1], [40, 30, 60]), ([1, 1, 1], [1500, 1430, 1160]), ([8] * 6, [50, 9, 400, 8, 20, 8]),
         ([150, 130, 70] + [90] * 60, [150, 130, 70] + [90] * 60)]  # enough blocks to take the prefix in one piece


@pytest.mark.parametrize("lq,lk", CASES)
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_neighbours_do_not_reach_a_sequence(lq, lk, bad):
    q, k, v = tensors(lq, lk, 4, 2, 128)
    pk, pv = prefix_tensors(333, 2, 128)
    clean = attention_shared(q, k, v, pk, pv, offsets(lq), offsets(lk))
    aq, ak = lq[0], lk[0]
    for t, a, n in ((q, aq, lq[1]), (k, ak, lk[1]), (v, ak, lk[1])):
        t[:a] = bad
        t[a + n:] = bad
    got = attention_shared(q, k, v, pk, pv, offsets(lq), offsets(lk))
    assert torch.equal(got[aq:aq + lq[1]], clean[aq:aq + lq[1]])
    assert not bool(torch.isfinite(got[:aq]).any()) and not bool(torch.isfinite(got[aq + lq[1]:]).any())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", CASES)
def test_scores_that_are_not_finite(lq, lk, d):
    """All visible scores minus infinity: NaN. A NaN key in the prefix: NaN everywhere. Keys of score minus infinity weigh
    nothing, however large their values."""
    q, k, v = tensors(lq, lk, 4, 2, d, seed=11)
    pk, pv = prefix_tensors(333, 2, d)
    k[..., 0], pk[..., 0] = -k[..., 0].abs() - 1, -pk[..., 0].abs() - 1
    cu_q, cu_k = offsets(lq), offsets(lk)
    lost = q.clone()
    rows = slice(0, None, 3)
    lost[rows, 1, 0] = math.inf
    got, clean = attention_shared(lost, k, v, pk, pv, cu_q, cu_k), attention_shared(q, k, v, pk, pv, cu_q, cu_k)
    assert bool(torch.isnan(got[rows, 1]).all())
    got[rows, 1] = clean[rows, 1]
    assert torch.equal(got, clean)
    for at in (0, 7, 130, 332):
        bad = pk.clone()
        bad[at, 1, 3] = math.nan
        got = attention_shared(q, k, v, bad, pv, cu_q, cu_k)
        assert bool(torch.isnan(got[:, 2:]).all()) and torch.equal(got[:, :2], clean[:, :2])
    q[..., 0] = 1
    k[1::2, :, 0], v[1::2], pk[::2, :, 0], pv[::2] = -math.inf, 2.0 ** 127, -math.inf, 2.0 ** 127
    got = attention_shared(q, k, v, pk, pv, cu_q, cu_k)
    v[1::2], pv[::2] = 0, 0
    compare(got, reference(q, k, v, pk, pv, lq, lk, True, 1 / math.sqrt(d)))
    pk[..., 0] = -math.inf  # the whole prefix weighs nothing: attention of the own keys
    pv[:] = 2.0 ** 127
    got, (ref, size) = attention_shared(q, k, v, pk, pv, cu_q, cu_k), reference(q, k, v, pk, 0 * pv, lq, lk, True, 1 / math.sqrt(d))
    nothing = torch.isnan(ref)  # rows whose own keys all have minus infinity, too: no softmax
    assert torch.equal(torch.isnan(got), nothing)
    compare(got[~nothing], (ref[~nothing], size[~nothing]))


def test_as_attention_over_copies_of_the_prefix():
    """The same sequences with the prefix copied in front of each, through attention_packed."""
    lq, lk, prefix = [1, 1, 1, 1], [30, 200, 5, 77], 400
    q, k, v = tensors(lq, lk, 8, 2, 128, seed=5)
    pk, pv = prefix_tensors(prefix, 2, 128)
    whole_k, whole_v = (torch.cat([x for part in t.split(lk) for x in (p, part)]) for t, p in ((k, pk), (v, pv)))
    other = attention_packed(q, whole_k, whole_v, offsets(lq), offsets([prefix + n for n in lk]))
    got = attention_shared(q, k, v, pk, pv, offsets(lq), offsets(lk))
    assert float((got.double() - other.double()).norm()) <= 2.0 ** -7 * float(other.double().norm())
    empty = prefix_tensors(0, 2, 128)
    assert torch.equal(attention_shared(q, k, v, *empty, offsets(lq), offsets(lk)),
                       attention_packed(q, k, v, offsets(lq), offsets(lk)))


@pytest.mark.parametrize("lq,lk", [([60, 100], [60, 100]), ([1, 1], [60, 100]), ([12, 12], [60, 100])])
def test_strided_views(lq, lk):
    """Fused projections in place, heads before tokens, broadcast heads, and views that have to be copied."""
    g = torch.Generator().manual_seed(3)
    nq, nk, prefix = sum(lq), sum(lk), 300
    fused = torch.randn(prefix + nk, (4 + 2 + 2) * 128, generator=g).bfloat16().to(DEV)

    def views(f):
        q, k, v = (t.unflatten(1, (-1, 128)) for t in f.split([512, 256, 256], 1))
        return q[prefix:prefix + nq], k[prefix:], v[prefix:], k[:prefix], v[:prefix]

    cu = offsets(lq), offsets(lk)
    expected = attention_shared(*(t.contiguous() for t in views(fused)), *cu)
    assert torch.equal(attention_shared(*views(fused), *cu), expected)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in views(fused)]
    assert torch.equal(attention_shared(*heads_first, *cu), expected)
    odd = torch.cat((fused[:, :1], fused), 1)[:, 1:]  # 2-byte aligned
    assert torch.equal(attention_shared(*views(odd), *cu), expected)
    q, *rest = views(fused)
    shared = [t[:, :1].expand(-1, 4, -1) for t in rest]
    assert torch.equal(attention_shared(q, *shared, *cu), attention_shared(q, *(t.contiguous() for t in shared), *cu))


def test_tokens_past_the_last_offset_give_zeros():
    for lq, lk, tokens in (([40, 60], [40, 60], 300), ([1, 1, 1], [90, 100, 20], 40), ([1, 1], [9, 9], 3), ([5] * 8, [50] * 8, 60)):
        q, k, v = tensors([tokens], [400], 4, 2, 128)
        pk, pv = prefix_tensors(222, 2, 128)
        n = sum(lq)
        got = attention_shared(q, k, v, pk, pv, offsets(lq), offsets(lk))
        assert not bool(got[n:].any())
        compare(got[:n], reference(q[:n], k, v, pk, pv, lq, lk, True, 128 ** -0.5))


@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [900, 300, 4000]), ([1] * 50, [70] * 50), ([200, 100], [200, 100])])
def test_results_repeat_and_streams(lq, lk):
    q, k, v = tensors(lq, lk, 8, 2, 128)
    pk, pv = prefix_tensors(3000, 2, 128)
    args = (q, k, v, pk, pv, offsets(lq), offsets(lk))
    expected = attention_shared(*args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(attention_shared(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, expected) for g in got)


@pytest.mark.parametrize("first,others", [([100, 100], ([1, 255], [200, 0])), ([20] * 12, ([1] * 12, [0, 40] * 6))])
def test_graph_replay_follows_new_lengths(first, others):
    q, k, v = tensors([256], [256], 4, 2, 64)
    pk, pv = prefix_tensors(500, 2, 64)
    cu = offsets(first)
    attention_shared(q, k, v, pk, pv, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention_shared(q, k, v, pk, pv, cu)
    for lengths in (first, *others):
        cu.copy_(offsets(lengths))
        graph.replay()
        torch.cuda.synchronize()
        n = sum(lengths)
        compare(out[:n], reference(q[:n], k[:n], v[:n], pk, pv, lengths, lengths, True, 1 / 8))
        assert not bool(out[n:].any())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tq,tk,prefix,cu_q,cu_k", [
    (100, 100, 70, [0, 50, 500], None), (100, 100, 300, [0, 80, 40], None), (100, 100, 70, [-5, 20, 100], None),
    (100, 100, 70, [3, 50, 100], None), (100, 100, 129, [0, -2 ** 31, 2 ** 31 - 1], None), (100, 300, 70, [0, 100], [0, 301]),
    (2, 3000, 70, [0, 1, 2], [0, 2500, 1200]), (2, 3000, 600, [0, 1, 2], [-7, 5000, 3000]),
    (2, 3000, 70, [1, 0, 9], [0, 2 ** 31 - 1, -2 ** 31]),
    (40, 900, 1000, [i * 29 % 61 - 9 for i in range(40)], [i * 607 % 1400 - 200 for i in range(40)]),
    (80, 900, 1000, [i * 29 % 91 - 9 for i in range(40)], [i * 607 % 1400 - 200 for i in range(40)])], ids=str)
def test_wrong_offsets_stay_inside_the_tensors(tq, tk, prefix, cu_q, cu_k, d):
    """All operands lie between NaN, output and workspace between marks: none of it is read or written."""
    h, hk, margin, mark = 4, 2, 256, 7.0
    lib = _lib.load()
    cu_q, cu_k = (torch.tensor(c, dtype=torch.int32, device=DEV) for c in (cu_q, cu_k or cu_q))
    seqs = cu_q.numel() - 1

    def between(tokens, heads, edge):
        whole = torch.full((tokens + 2 * margin, heads, d), edge, device=DEV, dtype=torch.bfloat16)
        return whole, whole[margin:-margin]

    q, k, v, pk, pv = (between(n, heads, math.nan)[1] for n, heads in ((tq, h), (tk, hk), (tk, hk), (prefix, hk), (prefix, hk)))
    for t, source in zip((q, k, v, pk, pv), tensors([tq], [tk], h, hk, d, seed=tq + tk) + prefix_tensors(prefix, hk, d)):
        t.copy_(source)
    out_all, out = between(tq, h, mark)
    need = lib.lr_attention_shared_workspace_bytes(seqs, tq, tk, prefix, h, hk, d)
    work_all = torch.zeros((need + 8192,), dtype=torch.uint8, device=DEV)
    work_all[:4096], work_all[4096 + need:] = 171, 171
    work = work_all[4096:4096 + need]
    for causal in (0, 1):
        status = lib.lr_attention_shared(
            q.data_ptr(), h * d, d, k.data_ptr(), hk * d, d, v.data_ptr(), hk * d, d, pk.data_ptr(), hk * d, d, pv.data_ptr(), hk * d,
            d, cu_q.data_ptr(), cu_k.data_ptr(), seqs, tq, tk, prefix, h, hk, d, causal, d ** -0.5, out.data_ptr(),
            work.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream)
        assert status == 0 and _lib.device_status() == 8
        assert bool((out_all[:margin] == mark).all()) and bool((out_all[-margin:] == mark).all())
        assert bool((work_all[:4096] == 171).all()) and bool((work_all[4096 + need:] == 171).all())


def test_empty_and_refusals():
    q, k, v = tensors([8], [8], 4, 2, 64)
    pk, pv = prefix_tensors(5, 2, 64)
    cu = offsets([8])
    assert attention_shared(q[:0], k, v, pk, pv, offsets([0]), cu).shape == (0, 4, 64)
    none = attention_shared(q, k[:0], v[:0], pk, pv, cu, offsets([0]))
    compare(none, reference(q, k[:0], v[:0], pk, pv, [8], [0], True, 1 / 8))
    many = torch.ones(700, 4, 64, device=DEV, dtype=torch.bfloat16)
    compare(attention_shared(many, k[:0], v[:0], pk, pv, offsets([700]), offsets([0])),
            reference(many, k[:0], v[:0], pk, pv, [700], [0], True, 1 / 8))

    def refused(match, *args):
        with pytest.raises(ValueError, match=match):
            attention_shared(*args)

    refused("bf16", q.float(), k, v, pk, pv, cu)
    refused("bf16", q, k, v, pk.float(), pv, cu)
    refused("CUDA", q, k, v, pk.cpu(), pv, cu)
    refused("head_dim", q[..., :32], k[..., :32], v[..., :32], pk[..., :32], pv[..., :32], cu)
    refused("evenly", q[:, :3], k, v, pk, pv, cu)
    refused("disagree", q, k, v[:4], pk, pv, cu)
    refused("disagree", q, k, v, pk, pv[:4], cu)
    refused("disagree", q, k, v, pk[:, :1], pv[:, :1], cu)
    refused("int32", q, k, v, pk, pv, cu.long())
    refused("differ in sequences", q, k, v, pk, pv, cu, offsets([4, 4]))
    refused("cu_seqlens_k is needed", q[:4], k, v, pk, pv, cu)
