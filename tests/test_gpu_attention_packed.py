"""GPU tests of attention.attention_packed against attention in 64 bits, one sequence and head at a time.

Tolerance per value: the probabilities are rounded to bf16 (at most 2^-8 each, so 2^-8 of sum p |v|, half of that on
average), the output too (2^-8 |ref|); fp32 sums and exponentials (below 2^-12) fit in what the average leaves:
2^-8 (sum p |v| + |ref|).
"""
from __future__ import annotations

import math

import pytest
import torch

from lynnreal_omni_b200 import _lib
from lynnreal_omni_b200.attention import attention_packed

pytestmark = pytest.mark.gpu
DEV = "cuda"


def offsets(lengths):
    return torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32, device=DEV)


def tensors(lq, lk, h, hk, d, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    q = spread * torch.randn(sum(lq), h, d, generator=g)
    k, v = (torch.randn(sum(lk), hk, d, generator=g) for _ in range(2))
    return [t.bfloat16().to(DEV) for t in (q, k, v)]


def reference(q, k, v, lq, lk, causal, scale):
    q, k, v = (t.double() for t in (q, k, v))
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    iq = ik = 0
    for nq, nk in zip(lq, lk):
        for h in range(q.shape[1]):
            qs, ks, vs = q[iq:iq + nq, h], k[ik:ik + nk, h // group], v[ik:ik + nk, h // group]
            s = qs @ ks.t() * scale
            if causal:
                hidden = torch.arange(nk, device=q.device) > torch.arange(nq, device=q.device)[:, None] + nk - nq
                s = s.masked_fill(hidden, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)) if nk else s
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0)
            out[iq:iq + nq, h], size[iq:iq + nq, h] = p @ vs, p @ vs.abs()
        iq, ik = iq + nq, ik + nk
    return out, size


def check(lq, lk, h, hk, d, causal=True, seed=0, spread=1.0, scale=None):
    q, k, v = tensors(lq, lk, h, hk, d, seed, spread)
    got = attention_packed(q, k, v, offsets(lq), offsets(lk), causal=causal, scale=scale)
    compare(got, reference(q, k, v, lq, lk, causal, 1 / math.sqrt(d) if scale is None else scale))
    assert _lib.device_status() == 0
    return got


def compare(got, expected):
    ref, size = expected
    err, bound = (got.double() - ref).abs(), 2.0 ** -8 * (size + ref.abs()) + 1e-30
    assert bool((err <= bound).all()), (float((err / bound).max()), (~(err <= bound)).nonzero()[:4].tolist())


PROMPTS = [[1], [2], [63], [64], [65], [127], [128], [129], [300], [1, 1, 1], [5, 130, 1, 64, 257], [0, 7, 0, 0, 200, 0],
           [1000], [640, 3]]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths", PROMPTS, ids=str)
def test_whole_prompts(lengths, d):
    check(lengths, lengths, 4, 2, d, seed=sum(lengths))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk", [(1, 1), (3, 3), (3, 1), (5, 1), (6, 2), (7, 1), (8, 1), (12, 4), (32, 8), (16, 1), (48, 1),
                                  (128, 1), (130, 1), (200, 1)])
def test_head_groups(h, hk, causal):
    check([3, 150, 41], [3, 150, 41], h, hk, 64, causal)
    check([1, 2, 9], [77, 260, 9], h, hk, 128, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1], [4096]), ([1, 1, 1], [5, 3000, 129]), ([2, 5, 8], [2, 700, 1025]),
                                   ([100, 1], [2500, 2500]), ([1] * 70, list(range(1, 71))), ([4, 4], [3, 0]),
                                   ([130], [7]), ([0, 3], [50, 60]), ([1, 0], [0, 9])])
def test_fewer_or_more_queries_than_keys(lq, lk, causal, d):
    """Decoding steps and pieces of prompts; rows before the first key give zeros."""
    got = check(lq, lk, 4, 1, d, causal)
    if causal and lq == [130]:
        assert not bool(got[:123].any()) and bool(got[123:].any())
    if lk == [3, 0]:
        assert not bool(got[4:].any())


@pytest.mark.parametrize("seqs", [31, 32, 33, 255, 256, 400])
def test_many_sequences(seqs):
    """Both ways of finding a block's sequence, at the edges of their ranges; every third sequence is empty."""
    lengths = [0 if i % 3 == 2 else 40 + 53 * i % 97 for i in range(seqs)]
    check(lengths, lengths, 2, 1, 64, seed=seqs)


def test_long_sequences():
    check([4100], [4100], 2, 1, 128)
    check([1], [70000], 8, 1, 128, seed=1)
    check([1, 3], [9000, 20000], 8, 2, 64, seed=2)


def test_workspace_is_bounded_by_the_keys():
    """Split sequences among many short ones: the parts lie close together, whatever the number of sequences."""
    need = _lib.load().lr_attention_packed_workspace_bytes
    assert need(100000, 100000, 10 ** 8, 32, 8, 128) == need(2, 2, 10 ** 8, 32, 8, 128) < 1 << 24
    lk = [700, 3, 2900, 257, 1, 513, 0, 4000] + [5] * 50 + [1200]
    check([1] * len(lk), lk, 8, 2, 128)
    check([1, 2] * (len(lk) // 2) + [1], lk, 4, 2, 64, seed=3)


@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_flat_and_peaked_scores(spread):
    check([260, 40], [260, 40], 4, 2, 128, spread=spread)
    check([1, 1], [2600, 400], 4, 2, 128, spread=spread)


def test_scale():
    for scale in (0.0, -0.1, 0.5):
        check([140], [140], 2, 1, 64, scale=scale)


@pytest.mark.parametrize("lq,lk", [([40, 30, 60], [40, 30, 60]), ([1, 1, 1], [40, 30, 60]), ([1, 1, 1], [1500, 1430, 1160])])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_neighbours_do_not_reach_a_sequence(lq, lk, bad):
    """Infinities and NaN in the other sequences' queries, keys and values leave a sequence's rows as they were."""
    q, k, v = tensors(lq, lk, 4, 2, 128)
    clean = attention_packed(q, k, v, offsets(lq), offsets(lk))
    aq, ak = lq[0], lk[0]
    for t, a, n in ((q, aq, lq[1]), (k, ak, lk[1]), (v, ak, lk[1])):
        t[:a] = bad
        t[a + n:] = bad
    got = attention_packed(q, k, v, offsets(lq), offsets(lk))
    assert torch.equal(got[aq:aq + lq[1]], clean[aq:aq + lq[1]])
    assert not bool(torch.isfinite(got[:aq]).any()) and not bool(torch.isfinite(got[aq + lq[1]:]).any())


def test_non_finite_queries_stay_in_their_rows():
    q, k, v = tensors([200], [200], 4, 2, 64)
    clean = attention_packed(q, k, v, offsets([200]))
    q[50, 1] = math.nan
    got = attention_packed(q, k, v, offsets([200]))
    assert bool(torch.isnan(got[50, 1]).all())
    got[50, 1] = clean[50, 1]
    assert torch.equal(got, clean)


def test_strided_views():
    """Views of a fused projection in place, heads before tokens, and views that have to be copied."""
    lengths = [60, 100]
    g = torch.Generator().manual_seed(3)
    fused = torch.randn(160, (4 + 2 + 2) * 128, generator=g).bfloat16().to(DEV)
    q, k, v = (t.unflatten(1, (-1, 128)) for t in fused.split([512, 256, 256], 1))
    expected = attention_packed(q.contiguous(), k.contiguous(), v.contiguous(), offsets(lengths))
    assert torch.equal(attention_packed(q, k, v, offsets(lengths)), expected)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(attention_packed(*heads_first, offsets(lengths)), expected)
    shared = [t[:, :1].expand(-1, 4, -1) for t in (k, v)]  # broadcast heads
    assert torch.equal(attention_packed(q, *shared, offsets(lengths)),
                       attention_packed(q, k[:, :1], v[:, :1], offsets(lengths)))
    odd = torch.cat((fused[:, :1], fused), 1)[:, 1:]  # 2-byte aligned
    views = [t.unflatten(1, (-1, 128)) for t in odd.split([512, 256, 256], 1)]
    assert torch.equal(attention_packed(*views, offsets(lengths)), expected)


def test_tokens_past_the_last_offset_give_zeros():
    q, k, v = tensors([300], [300], 2, 1, 128)
    got = attention_packed(q, k, v, offsets([40, 60]))
    assert not bool(got[100:].any())
    assert torch.equal(got[:100], attention_packed(q[:100], k[:100], v[:100], offsets([40, 60])))
    few = attention_packed(q[:9], k, v, offsets([1, 1, 1]), offsets([90, 100, 20]))
    assert not bool(few[3:].any()) and bool(few[:3].any())


@pytest.mark.parametrize("cu", [[0, 50, 500], [0, 80, 40], [-5, 20, 100], [3, 50, 100]])
def test_wrong_offsets_are_reported(cu):
    """Offsets outside the tensors, or going down, raise the status bit; nothing outside is read or written."""
    q, k, v = tensors([100], [100], 2, 1, 64)
    bad = torch.tensor(cu, dtype=torch.int32, device=DEV)
    attention_packed(q, k, v, bad)
    assert _lib.device_status() == 8
    attention_packed(q[:2], k, v, offsets([1, 1]), bad)
    assert _lib.device_status() == 8
    assert _lib.device_status() == 0


def test_results_repeat_and_streams():
    q, k, v = tensors([1, 1, 1], [9000, 300, 4000], 8, 2, 128)
    cu_q, cu_k = offsets([1, 1, 1]), offsets([9000, 300, 4000])
    expected = attention_packed(q, k, v, cu_q, cu_k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [attention_packed(q, k, v, cu_q, cu_k) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(g, expected) for g in got)


def test_graph_replay_follows_new_lengths():
    """Lengths live on the device: a captured call serves other lengths of the same buffers."""
    q, k, v = tensors([256], [256], 4, 2, 64)
    cu = offsets([100, 100])
    attention_packed(q, k, v, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention_packed(q, k, v, cu)
    for lengths in ([100, 100], [1, 255], [200, 0]):
        cu.copy_(offsets(lengths))
        graph.replay()
        torch.cuda.synchronize()
        n = sum(lengths)
        compare(out[:n], reference(q[:n], k[:n], v[:n], lengths, lengths, True, 1 / 8))
        assert not bool(out[n:].any())


def test_empty_and_refusals():
    q, k, v = tensors([8], [8], 4, 2, 64)
    cu = offsets([8])
    assert attention_packed(q[:0], k, v, offsets([0]), cu).shape == (0, 4, 64)
    assert not bool(attention_packed(q, k[:0], v[:0], cu, offsets([0])).any())
    many = torch.ones(700, 4, 64, device=DEV, dtype=torch.bfloat16)
    assert not bool(attention_packed(many, k[:0], v[:0], offsets([700]), offsets([0])).any())
    with pytest.raises(ValueError, match="bf16"):
        attention_packed(q.float(), k, v, cu)
    with pytest.raises(ValueError, match="head_dim"):
        attention_packed(q[..., :32], k[..., :32], v[..., :32], cu)
    with pytest.raises(ValueError, match="evenly"):
        attention_packed(q[:, :3], k, v, cu)
    with pytest.raises(ValueError, match="disagree"):
        attention_packed(q, k, v[:4], cu)
    with pytest.raises(ValueError, match="int32"):
        attention_packed(q, k, v, cu.long())
    with pytest.raises(ValueError, match="differ in sequences"):
        attention_packed(q, k, v, cu, offsets([4, 4]))
    with pytest.raises(ValueError, match="cu_seqlens_k is needed"):
        attention_packed(q[:4], k, v, cu)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk,causal", [([300], [300], True), ([200], [515], False), ([1], [3000], False)])
def test_scores_that_are_not_finite(lq, lk, causal, d):
    """Rows whose visible scores are all minus infinity have no softmax and give NaN; a NaN key gives NaN to every row
    that sees it, wherever in a tile it lies; keys of score minus infinity weigh nothing, however large their values."""
    q, k, v = tensors(lq, lk, 4, 2, d, seed=11)
    k[..., 0] = -k[..., 0].abs() - 1
    cu_q, cu_k = offsets(lq), offsets(lk)
    rows = slice(0, None, 7)
    lost = q.clone()
    lost[rows, 1, 0] = math.inf
    got, clean = attention_packed(lost, k, v, cu_q, cu_k, causal=causal), attention_packed(q, k, v, cu_q, cu_k, causal=causal)
    assert bool(torch.isnan(got[rows, 1]).all())
    got[rows, 1] = clean[rows, 1]
    assert torch.equal(got, clean)

    for at in range(5, 13):
        bad = k.clone()
        bad[at, 1, 3] = math.nan
        got = attention_packed(q, bad, v, cu_q, cu_k, causal=causal)
        first = at if causal else 0  # heads 2 and 3 read key head 1
        assert bool(torch.isnan(got[first:, 2:]).all())
        assert torch.equal(got[:first], clean[:first]) and torch.equal(got[:, :2], clean[:, :2])

    q[..., 0] = 1
    k[1::2, :, 0], v[1::2] = -math.inf, 2.0 ** 127
    got = attention_packed(q, k, v, cu_q, cu_k, causal=causal)
    v[1::2] = 0
    compare(got, reference(q, k, v, lq, lk, causal, 1 / math.sqrt(d)))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tq,tk,cu_q,cu_k", [
    (100, 100, [0, 50, 500], None), (100, 100, [0, 80, 40], None), (100, 100, [-5, 20, 100], None), (100, 100, [3, 50, 100], None),
    (100, 100, [0, -2 ** 31, 2 ** 31 - 1], None), (100, 300, [0, 100], [0, 301]), (100, 300, [0, 100], [-400, 900]),
    (100, 100, [i * 37 % 131 - 20 for i in range(40)], None), (70, 900, [0, 30, 70], [700, 200, 2000]),
    (2, 3000, [0, 1, 2], [0, 2500, 1200]), (2, 3000, [0, 1, 2], [-7, 5000, 3000]), (2, 3000, [1, 0, 9], [0, 2 ** 31 - 1, -2 ** 31]),
    (40, 9000, [i * 29 % 61 - 9 for i in range(40)], [i * 6007 % 14000 - 2000 for i in range(40)])], ids=str)
def test_wrong_offsets_stay_inside_the_tensors(tq, tk, cu_q, cu_k, d):
    """Queries, keys and values lie between NaN, output and workspace between marks: none of it is read or written."""
    h, hk, margin, mark = 4, 2, 256, 7.0
    lib = _lib.load()
    cu_q, cu_k = (torch.tensor(c, dtype=torch.int32, device=DEV) for c in (cu_q, cu_k or cu_q))
    seqs = cu_q.numel() - 1

    def between(tokens, heads, edge):
        whole = torch.full((tokens + 2 * margin, heads, d), edge, device=DEV, dtype=torch.bfloat16)
        return whole, whole[margin:-margin]

    q, k, v = (between(n, heads, math.nan)[1] for n, heads in ((tq, h), (tk, hk), (tk, hk)))
    for t, source in zip((q, k, v), tensors([tq], [tk], h, hk, d, seed=tq + tk)):
        t.copy_(source)
    out_all, out = between(tq, h, mark)
    need = lib.lr_attention_packed_workspace_bytes(seqs, tq, tk, h, hk, d)
    work_all = torch.full((need + 8192,), 171, dtype=torch.uint8, device=DEV)
    work = work_all[4096:4096 + need]
    for causal in (0, 1):
        status = lib.lr_attention_packed(
            q.data_ptr(), h * d, d, k.data_ptr(), hk * d, d, v.data_ptr(), hk * d, d, cu_q.data_ptr(), cu_k.data_ptr(), seqs,
            tq, tk, h, hk, d, causal, d ** -0.5, out.data_ptr(), work.data_ptr() if need else None, need,
            torch.cuda.current_stream().cuda_stream)
        assert status == 0 and _lib.device_status() == 8
        assert bool(torch.isfinite(out).all())
        assert bool((out_all[:margin] == mark).all()) and bool((out_all[-margin:] == mark).all())
        assert bool((work_all[:4096] == 171).all()) and bool((work_all[4096 + need:] == 171).all())
