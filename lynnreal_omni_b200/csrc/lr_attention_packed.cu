// Attention over packed sequences of different lengths, causal or full, with
// query heads sharing key/value heads in groups:
//   out[i, h, :] = sum_j softmax_j(scale * q[i, h, :] . k[j, h / group, :]) v[j, h / group, :]
// over the keys j of query i's own sequence (causal: the queries are the last
// ones of their sequence, and query i of Lq sees keys j <= i + Lk - Lq).
//
// The offsets stay on the device, so the grids are bounds: a sequence that
// starts at token c gets its blocks of B tokens from slot c / B + b on. Slots
// of sequence b + 1 start at least ceil(length / B) later, at most one slot a
// sequence stays empty, and the sequence of a slot is found by search.
//
// The rows of a tile are the (token, head) pairs of one key/value head's group:
// keys and values are read once for all its query heads.
//
//   * prompt_kernel: many queries a sequence; bound by the tensor cores and the
//     softmax under them. One prompt of 16384 tokens, 32 query and 8 key/value
//     heads of 128: 2.00 ms, 1098 TFLOP/s, 0.66 of the measured bf16 burst rate
//     (the GPU is at its power limit then; 0.78 of the sustained rate).
//   * step_kernel (+ join_kernel): up to 64 rows a sequence on average
//     (decoding); bound by reading keys and values, which are split over the
//     GPU and joined. 64 requests of one token against 1024 to 5056 keys: 134
//     us, 5.9 TB/s, 0.91 of the measured copy rate; one against 32768: 27 us.
//     The prompt kernel would leave all but `group` of a tile's 256 rows empty
//     and one CTA to a sequence's keys.
#include "lr_common.cuh"
#include "lr_host.h"
#include "lr_tc.cuh"

namespace lr {

static __device__ unsigned int g_packed_status = 0;

namespace packed {
namespace {

using namespace tc;
using bf16 = __nv_bfloat16;

struct Args {
  const bf16 *q, *k, *v;
  bf16* out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const int32_t *cu_q, *cu_k;
  int seqs, total_q, total_k, heads, kv_heads, group, causal;
  float scale_log2;
};

// Raise the status bit unless both offset arrays start at 0, never go down and
// end within their tensors. `count` threads, this one the `first`-th.
__device__ void check_offsets(const Args& a, int first, int count) {
  bool bad = false;
  for (int i = first; i <= a.seqs; i += count) {
    const int q = a.cu_q[i], k = a.cu_k[i];
    bad |= q < (i ? a.cu_q[i - 1] : 0) || k < (i ? a.cu_k[i - 1] : 0) || q > a.total_q || k > a.total_k;
    bad |= i == 0 && (q | k) != 0;
  }
  if (bad) atomicOr(&g_packed_status, (unsigned)kDevErrOffsets);
}

__device__ __forceinline__ int clamped(const int32_t* cu, int i, int total) { return min(max(cu[i], 0), total); }
// First slot of sequence b where blocks are `block` tokens.
__device__ __forceinline__ int first_slot(const int32_t* cu, int b, int total, int block) {
  return (int)((uint32_t)clamped(cu, b, total) / (uint32_t)block) + b;
}
// The last b in [0, last] whose first slot is at or before `slot`. A whole warp
// searches: 32 candidates a step.
__device__ __forceinline__ int find_sequence(const int32_t* cu, int last, int total, int block, int slot, int lane) {
  int lo = 0, n = last + 1;  // the answer lies in [lo, lo + n)
  while (n > 1) {
    const int stride = (n + 31) / 32;
    const int b = lo + lane * stride;
    const bool at = b < lo + n && first_slot(cu, b, total, block) <= slot;
    const int hits = __popc(__ballot_sync(0xffffffffu, at));
    const int step = max(hits - 1, 0) * stride;
    n = min(stride, n - step);
    lo += step;
  }
  return lo;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// ------------------------------------------------------------------ prompts
constexpr int kRows = 128;    // rows of a query tile (TMEM lanes)
constexpr int kKeys = 128;    // keys of a tile
constexpr int kHalf = 64;     // keys whose probabilities are handed over together
constexpr int kAtom = 128 * 128;  // 128 rows x 64 columns, 128-byte swizzle
constexpr int kPromptThreads = 384;

// Largest scaled score of 64 (of the first `valid` of them).
template <bool MASKED>
__device__ __forceinline__ float half_maximum(const uint32_t* s, float scale, int valid) {
  if constexpr (MASKED) {
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 64; ++e)
      if (e < valid) mx = fmaxf(mx, __uint_as_float(s[e]) * scale);
    return mx;
  } else {
    float m4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) m4[e] = __uint_as_float(s[e]);
    if (scale >= 0.0f) {
#pragma unroll
      for (int e = 4; e < 64; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(s[e]));
      return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * scale;
    }
#pragma unroll
    for (int e = 4; e < 64; ++e) m4[e & 3] = fminf(m4[e & 3], __uint_as_float(s[e]));
    return fminf(fminf(m4[0], m4[1]), fminf(m4[2], m4[3])) * scale;
  }
}

template <int D>
struct Prompt {
  static constexpr int kTile = D / 64 * kAtom;
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr int kQ = 0, kRing = 2 * kTile, kBars = kRing + kSlots * kTile;
  static constexpr int kBarBytes = 768;  // barriers and items
  static constexpr size_t kSmem = 1024 + kBars + kBarBytes;
  static constexpr uint32_t kColO = 256;  // scores of tile t at 128 t, output of tile t at 256 + D t
  static_assert(kSmem <= 232448, "shared memory");
};

// Instruction descriptors, kind::f16: fp32 accumulator, bf16 operands, N / 8 at
// 17, M / 16 at 24; bit 16: B is MN-major (V).
constexpr uint32_t kDescQK = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kKeys / 8) << 17) | ((uint32_t)(kRows / 16) << 24);
template <int D>
constexpr uint32_t kDescPV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D / 8) << 17) |
                             ((uint32_t)(kRows / 16) << 24);

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(desc), "r"(accumulate)
      : "memory");
}
// Issue a 32-column load; its registers are valid after tmem_wait32 of them. The
// access is .sync.aligned, as the store below: the lanes meet first.
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait32(uint32_t* a) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]),
                 "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]),
                 "+r"(a[15]), "+r"(a[16]), "+r"(a[17]), "+r"(a[18]), "+r"(a[19]), "+r"(a[20]), "+r"(a[21]),
                 "+r"(a[22]), "+r"(a[23]), "+r"(a[24]), "+r"(a[25]), "+r"(a[26]), "+r"(a[27]), "+r"(a[28]),
                 "+r"(a[29]), "+r"(a[30]), "+r"(a[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 2^x for a pair on the FMA pipe: x = n + f with n = round(x), f in [-1/2, 1/2];
// 2^f by a cubic fitted to it there (relative error below 7.5e-5, far under the
// bf16 rounding of the probabilities), times 2^n. x is held above -125, so that
// the result stays a normal number, and what the cubic gives there is taken off
// again (nothing against any result above 2^-100): a score of minus infinity, or
// one that far below the maximum, weighs exactly 0, however large its value row.
// 2^n as a factor and not as a sum of exponent fields lets NaN through.
__device__ __forceinline__ float2 exp2_poly2(float2 x) {
  constexpr float kMagic = 12582912.0f;
  constexpr float kOne = 0.9999280572f;  // the cubic at 0
  constexpr float kFloor = -kOne * 0x1p-125f;
  x.x = max_nan(x.x, -125.0f);
  x.y = max_nan(x.y, -125.0f);
  const float2 t = __fadd2_rn(x, make_float2(kMagic, kMagic));
  const float2 n = __fadd2_rn(t, make_float2(-kMagic, -kMagic));
  const float2 f = __ffma2_rn(n, make_float2(-1.0f, -1.0f), x);  // exact
  float2 p = __ffma2_rn(f, make_float2(0.0551716685f, 0.0551716685f), make_float2(0.2426111400f, 0.2426111400f));
  p = __ffma2_rn(p, f, make_float2(0.6932609677f, 0.6932609677f));
  p = __ffma2_rn(p, f, make_float2(kOne, kOne));
  const float2 power = make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                                   __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u));
  return __ffma2_rn(p, power, make_float2(kFloor, kFloor));
}

// One pair in `kPolyEvery` of a full tile goes through exp2_poly2: the special
// function unit (16 values a cycle) is as busy as the tensor core otherwise. At
// 64 columns, where the products take half as long, one in three (8192 tokens:
// 452 us without, 418 us one in four, 410 us one in three), at 128 one in four
// (16384 tokens: 2066, 1955, 2030 us).
template <int D>
constexpr int kPolyEvery = D == 64 ? 3 : 4;

struct PromptShape {
  int tokens_tile;  // query tokens of a tile
  int tile_heads;   // query heads of a tile (the group, or a part of a group above 128)
  int head_parts;   // tiles that a group is cut into
  int slots;
  int items;        // slots * kv_heads * head_parts
  int wide_out;     // out is 32-byte aligned
};

// A block of work: two query tiles of one key/value head (or a part of its group).
struct PromptItem {
  int q_row;       // first query token
  int tok0;        // the same within its sequence
  int lq, lk;      // lengths of the sequence
  int k_row;       // first key
  int kv_head, head0, heads_here;
  int tiles[2];    // key tiles that each query tile sees
};
constexpr int kItemSlots = 4;

// Work item `index`, or false for an empty slot; the heads of a block stand
// side by side. Later blocks of a sequence see more keys and come first: from
// two to 31 sequences all the sequences' blocks by their number in the sequence
// (16 sequences of up to 2048 tokens, 24 heads of 64: 51 -> 41 us; 24 of up to
// 1500, 32 heads of 128: 229 -> 196 us), else each sequence's in turn (40 such
// sequences are as fast either way: there are blocks enough to even out).
__device__ __forceinline__ bool prompt_item(const Args& a, const PromptShape& ps, int index, int lane, PromptItem& w) {
  const int parts = a.kv_heads * ps.head_parts;
  const int part = index % parts, rank = index / parts;
  w.kv_head = part / ps.head_parts;
  const int in_group = part % ps.head_parts * ps.tile_heads;
  w.heads_here = min(ps.tile_heads, a.group - in_group);
  w.head0 = w.kv_head * a.group + in_group;
  const int block = 2 * ps.tokens_tile;
  // "Sequence" a.seqs is what lies past the last offset: queries without keys.
  int b, qs, qe, ke;
  if (a.seqs < 32) {  // every offset in one lane: one round of loads
    const int q = clamped(a.cu_q, min(lane, a.seqs), a.total_q), k = clamped(a.cu_k, min(lane, a.seqs), a.total_k);
    if (a.seqs == 1) {
      const int slot = ps.slots - 1 - rank, slot1 = (int)((uint32_t)__shfl_sync(0xffffffffu, q, 1) / (uint32_t)block) + 1;
      b = slot >= slot1 ? 1 : 0;
      w.tok0 = (slot - (b ? slot1 : (int)((uint32_t)__shfl_sync(0xffffffffu, q, 0) / (uint32_t)block))) * block;
    } else {
      const int q_next = __shfl_down_sync(0xffffffffu, q, 1);
      const int length = lane > a.seqs ? 0 : max((lane == a.seqs ? a.total_q : q_next) - q, 0);
      const int blocks = (int)(((uint32_t)length + (uint32_t)block - 1) / (uint32_t)block);
      // S(i) = number of blocks that are the i-th or a later one of their sequence; the item is a block i with
      // S(i + 1) <= rank < S(i)
      auto later = [&](int i) { return __reduce_add_sync(0xffffffffu, max(blocks - i, 0)); };
      if (rank >= later(0)) return false;
      int lo = 0, hi = __reduce_max_sync(0xffffffffu, blocks);  // S(lo) > rank >= S(hi)
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (later(mid) > rank) lo = mid; else hi = mid;
      }
      b = (int)__fns(__ballot_sync(0xffffffffu, blocks > lo), 0, rank - later(lo + 1) + 1);
      w.tok0 = lo * block;
    }
    qs = __shfl_sync(0xffffffffu, q, b);
    qe = __shfl_sync(0xffffffffu, q, min(b + 1, a.seqs));
    w.k_row = __shfl_sync(0xffffffffu, k, b);
    ke = __shfl_sync(0xffffffffu, k, min(b + 1, a.seqs));
  } else {
    const int slot = ps.slots - 1 - rank;
    b = find_sequence(a.cu_q, a.seqs, a.total_q, block, slot, lane);
    qs = clamped(a.cu_q, b, a.total_q);
    qe = clamped(a.cu_q, min(b + 1, a.seqs), a.total_q);
    w.k_row = clamped(a.cu_k, b, a.total_k);
    ke = clamped(a.cu_k, min(b + 1, a.seqs), a.total_k);
    w.tok0 = (slot - (int)((uint32_t)qs / (uint32_t)block) - b) * block;
  }
  if (b == a.seqs) qe = a.total_q;
  w.lk = max(ke - w.k_row, 0);
  w.lq = max(qe - qs, 0);
  w.q_row = qs + w.tok0;
  if (w.tok0 < 0 || w.tok0 >= w.lq) return false;  // below 0: offsets that go down
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = w.tok0 + t * ps.tokens_tile, last = min(first + ps.tokens_tile, w.lq) - 1;
    const int seen = first >= w.lq ? 0 : a.causal ? min(max(last + w.lk - w.lq + 1, 0), w.lk) : w.lk;
    w.tiles[t] = (seen + kKeys - 1) / kKeys;
  }
  return true;
}

// Probabilities of 64 scores (bf16 pairs into s[0..31]) and their sum.
template <bool MASKED, int D>
__device__ __forceinline__ void probabilities(uint32_t* s, float2 sc2, float2 nm2, int valid, float2& sum) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), sc2, nm2);
    float2 p;
    if (!MASKED && i % kPolyEvery<D> == kPolyEvery<D> - 1)
      p = exp2_poly2(x);
    else
      p = make_float2(ex2(x.x), ex2(x.y));
    if (MASKED) {
      p.x = 2 * i < valid ? p.x : 0.0f;
      p.y = 2 * i + 1 < valid ? p.y : 0.0f;
    }
    sum = __fadd2_rn(sum, p);
    s[i] = cvt2(p.x, p.y);
  }
}

// 16 bf16 values; rows lie far apart, so a lane's store should fill a 32-byte sector.
__device__ __forceinline__ void store_16(bf16* dst, const uint32_t* y, int wide) {
  if (wide)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(y[0]), "r"(y[1]), "r"(y[2]),
                 "r"(y[3]), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
                 : "memory");
  else
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<uint4*>(dst + 8 * i) = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
}

// Persistent, one CTA an SM; warp roles: 0 copies, 1 MMAs, 3 finds the items,
// 4-7 and 8-11 the softmax of query tiles 0 and 1. While one item's last
// products and its output are under way, the next one's queries and keys load
// and its first scores are computed. (A block of its own for each item spent
// 7.8 us of set-up and end on it: 16 prompts of 2048 tokens, 48 heads, took 1326
// us and take 1016 us.) Scores and probabilities share tensor memory: of the 512
// columns two query tiles' outputs hold 256 and their scores 256, and a tile's
// probabilities, half a column a key, overwrite its own scores. The softmax
// therefore reads a tile's first half twice instead of holding 128 scores a
// thread, and hands the second half over first.
template <int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Args a, const PromptShape ps) {
  using C = Prompt<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* q_full = bars;               // [tile] queries landed
  uint64_t* q_empty = bars + 2;          // [tile] read by their last scores
  uint64_t* full = bars + 4;             // [slot] K or V tile landed
  uint64_t* empty = full + C::kSlots;    // [slot] read by all its MMAs
  uint64_t* s_full = empty + C::kSlots;  // [tile] scores ready; the previous P V is done, too
  uint64_t* p_half = s_full + 2;         // [tile] the second half's probabilities written, output rescaled
  uint64_t* p_full = s_full + 4;         // [tile] all of them
  uint64_t* o_done = s_full + 6;         // [tile] last P V of the item done
  uint64_t* o_empty = s_full + 8;        // [tile] output read
  uint64_t* i_full = s_full + 10;        // [item slot] published
  uint64_t* i_empty = i_full + kItemSlots;  // [item slot] read by every role
  uint64_t* drain = i_empty + kItemSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  PromptItem* items = reinterpret_cast<PromptItem*>(tmem_slot + 2);
  static_assert((14 + 2 * C::kSlots + 2 * kItemSlots + 1) * 8 + 8 + kItemSlots * sizeof(PromptItem) <= C::kBarBytes, "barriers");
  const Watch watch{tmem_slot + 1, &g_packed_status};

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_map(&map_q);
    if (a.total_k > 0) {  // else there is no map
      prefetch_map(&map_k);
      prefetch_map(&map_v);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&q_full[t]), 1);
      mbar_init(smem_u32(&q_empty[t]), 1);
      mbar_init(smem_u32(&s_full[t]), 1);
      mbar_init(smem_u32(&p_half[t]), 4);
      mbar_init(smem_u32(&p_full[t]), 4);
      mbar_init(smem_u32(&o_done[t]), 1);
      mbar_init(smem_u32(&o_empty[t]), 4);
    }
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int s = 0; s < kItemSlots; ++s) {
      mbar_init(smem_u32(&i_full[s]), 1);
      mbar_init(smem_u32(&i_empty[s]), 10);  // copies, MMAs, eight softmax warps
    }
    mbar_init(smem_u32(drain), 1);
    *watch.abort_flag = 0u;
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc<1>(smem_u32(tmem_slot), 512);
  // Items are dealt out forth and back, so that every CTA gets as many heavy ones.
  auto item_index = [&](int round) {
    return round * (int)gridDim.x + (round & 1 ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
  };
  PromptItem first{};
  bool first_there = false;
  if (warp == 3) first_there = prompt_item(a, ps, item_index(0), lane, first);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  // The ring holds K_0 V_0 K_1 V_1 ... of all items in turn; entry e is in slot e % kSlots.
  auto entry_bar = [&](uint64_t* set, uint32_t e) { return smem_u32(&set[e % C::kSlots]); };
  auto entry_addr = [&](uint32_t e) { return smem_u32(smem + C::kRing + (e % C::kSlots) * C::kTile); };
  auto entry_phase = [&](uint32_t e) { return (e / C::kSlots) & 1u; };
  // The next item, the number-th of this CTA; false at the end (no keys and no queries) or when giving up.
  auto next_item = [&](uint32_t number, PromptItem& w) {
    const uint32_t s = number % kItemSlots;
    if (!warp_wait(smem_u32(&i_full[s]), (number / kItemSlots) & 1u, watch, lane)) return false;
    w = items[s];
    w.lk = uniform(w.lk);
    w.tiles[0] = uniform(w.tiles[0]);
    w.tiles[1] = uniform(w.tiles[1]);
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&i_empty[s]));
    return w.lq > 0;
  };

  if (warp < 4) {
    if (warp == 3) {
      // ------------------------------------------------------- items
      if (blockIdx.x == 0) check_offsets(a, lane, 32);
      uint32_t number = 0;
      for (int round = 0;; ++round) {
        PromptItem w{};
        const bool end = round * (int64_t)gridDim.x >= ps.items;
        if (round == 0) {
          if (!first_there) continue;
          w = first;
        } else if (!end && (item_index(round) >= ps.items || !prompt_item(a, ps, item_index(round), lane, w))) {
          continue;
        }
        const uint32_t s = number % kItemSlots;
        if (!warp_wait(smem_u32(&i_empty[s]), ((number / kItemSlots) & 1u) ^ 1u, watch, lane)) break;
        if (lane == 0) {
          items[s] = w;  // all zeros at the end
          mbar_arrive(smem_u32(&i_full[s]));
        }
        __syncwarp();
        ++number;
        if (end) break;
      }
    } else if (warp == 0) {
      // ------------------------------------------------------ copies
      const bool el = elect_one();
      uint32_t e = 0, uses[2] = {0, 0};
      bool ok = true;
      PromptItem w;
      for (uint32_t number = 0; ok && next_item(number, w); ++number) {
        const int most = max(w.tiles[0], w.tiles[1]);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (w.tiles[t] == 0) continue;
          ok = ok && warp_wait(smem_u32(&q_empty[t]), (uses[t] & 1u) ^ 1u, watch, lane);
          if (el && ok) {
            const uint32_t bar = smem_u32(&q_full[t]), dst = smem_u32(smem + C::kQ + t * C::kTile);
            mbar_expect_tx(bar, (uint32_t)(D / 64 * 128 * ps.tile_heads * ps.tokens_tile));
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
              tma_load_3d(dst + x * kAtom, &map_q, bar, x * 64, w.head0, w.q_row + t * ps.tokens_tile);
          }
          __syncwarp();
          ++uses[t];
        }
        for (int i = 0; i < 2 * most && ok; ++i, ++e) {
          ok = warp_wait(entry_bar(empty, e), entry_phase(e) ^ 1u, watch, lane);
          if (el && ok) {
            const uint32_t bar = entry_bar(full, e), dst = entry_addr(e);
            mbar_expect_tx(bar, C::kTile);
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
              tma_load_3d(dst + x * kAtom, i & 1 ? &map_v : &map_k, bar, x * 64, w.kv_head, w.k_row + (i >> 1) * kKeys);
          }
          __syncwarp();
        }
      }
      if (!ok) {  // giving up: time for the copies in flight to land before the CTA can exit
        const unsigned long long t0 = globaltimer();
        while (globaltimer() - t0 < 100000ull) {
        }
      }
    } else if (warp == 1) {
      // -------------------------------------------------------- MMAs
      // Per key tile j: P_0 V_j, Q_0 K_{j+1}, P_1 V_j, Q_1 K_{j+1}: the softmax of one query tile runs under the
      // other's MMAs. P V starts on the second half of the keys while the first half's probabilities are computed.
      const bool el = elect_one();
      bool ok = true;
      uint32_t e0 = 0, done[2] = {0, 0}, uses[2] = {0, 0};  // ring entries, key tiles and items so far
      PromptItem w;
      for (uint32_t number = 0; ok && next_item(number, w); ++number) {
        const int most = max(w.tiles[0], w.tiles[1]);
        for (int j = -1; j < most && ok; ++j) {
          const uint32_t ev = e0 + 2 * j + 1, ek = ev + 1;  // V_j, K_{j+1}
          if (j >= 0 && !(ok = warp_wait(entry_bar(full, ev), entry_phase(ev), watch, lane))) break;
          if (j >= 0 && j == most - 1 && most * kKeys > w.lk) {
            // The last V tile ends past the sequence: its rows there, another sequence's, become zeros (their
            // probabilities are 0, but 0 times an infinity is not).
            uint8_t* tile = smem + C::kRing + (ev % C::kSlots) * C::kTile;
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
              for (int i = (w.lk - j * kKeys) * 8 + lane; i < kKeys * 8; i += 32)
                *reinterpret_cast<uint4*>(tile + x * kAtom + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            fence_async_smem();
            __syncwarp();
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint32_t s_col = tmem + (uint32_t)(t * 128), o_col = tmem + C::kColO + (uint32_t)(t * D);
            if (j >= 0 && j < w.tiles[t]) {
              const uint32_t parity = (done[t] + (uint32_t)j) & 1u;
              if (!(ok = warp_wait(smem_u32(&p_half[t]), parity, watch, lane))) break;
              // the item's first product writes over the previous item's output
              if (j == 0 && !(ok = warp_wait(smem_u32(&o_empty[t]), (uses[t] & 1u) ^ 1u, watch, lane))) break;
              const uint32_t v = entry_addr(ev);
#pragma unroll
              for (int h = 1; h >= 0; --h) {
                if (h == 0 && !(ok = warp_wait(smem_u32(&p_full[t]), parity, watch, lane))) break;
                tc_fence_after();
                if (el) {
#pragma unroll
                  for (int kk = 0; kk < kHalf / 16; ++kk)
                    mma_ts(o_col, s_col + h * kHalf + kk * 8, desc_mnmajor(v + (h * kHalf + kk * 16) * 128, kAtom),
                           kDescPV<D>, j > 0 || h == 0 || kk > 0 ? 1u : 0u);
                }
                __syncwarp();
              }
              if (!ok) break;
              if (el && j == w.tiles[t] - 1) mma_commit(smem_u32(&o_done[t]));
            }
            if (j + 1 < w.tiles[t]) {
              if (j < 0 && !(ok = warp_wait(smem_u32(&q_full[t]), uses[t] & 1u, watch, lane))) break;
              if (!(ok = warp_wait(entry_bar(full, ek), entry_phase(ek), watch, lane))) break;
              tc_fence_after();
              if (el) {
                const uint32_t q = smem_u32(smem + C::kQ + t * C::kTile), k = entry_addr(ek);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                  const uint32_t off = (uint32_t)((kk >> 2) * kAtom + (kk & 3) * 32);
                  mma_ss(s_col, desc_kmajor(q + off), desc_kmajor(k + off), kDescQK, kk != 0 ? 1u : 0u);
                }
                mma_commit(smem_u32(&s_full[t]));
                if (j + 1 == w.tiles[t] - 1) mma_commit(smem_u32(&q_empty[t]));
              }
            }
            __syncwarp();
          }
          if (el && ok) {
            if (j >= 0) mma_commit(entry_bar(empty, ev));
            if (j + 1 < most) mma_commit(entry_bar(empty, ek));
          }
          __syncwarp();
        }
        e0 += 2 * (uint32_t)most;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          done[t] += (uint32_t)w.tiles[t];
          uses[t] += w.tiles[t] > 0 ? 1u : 0u;
        }
      }
      // Every MMA is done before tensor memory can be released.
      if (el) mma_commit(smem_u32(drain));
      __syncwarp();
      drain_bounded(smem_u32(drain), 0u);
    }
  } else {
    // ---------------------------------------------------------- softmax
    const int t = (warp - 4) >> 2, quad = warp & 3;
    const int row = quad * 32 + lane;
    const int in_tile = row / ps.tile_heads, head = row - in_tile * ps.tile_heads;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_col = tmem + lanes + (uint32_t)(t * 128), o_col = tmem + lanes + C::kColO + (uint32_t)(t * D);
    uint32_t done = 0, uses = 0;
    bool ok = true;
    PromptItem w;
    for (uint32_t number = 0; ok && next_item(number, w); ++number) {
      // keys that this row sees, -1 for a row that stands for nothing
      int seen = -1;
      bf16* dst = a.out;
      {
        const int offset = t * ps.tokens_tile + in_tile;  // of this row's token in the block
        const int token = w.tok0 + offset;
        if (in_tile < ps.tokens_tile && head < w.heads_here && token < w.lq) {
          seen = a.causal ? min(max(token + w.lk - w.lq + 1, 0), w.lk) : w.lk;
          dst += ((int64_t)(w.q_row + offset) * a.heads + w.head0 + head) * D;
        }
      }
      const int n = w.tiles[t];
      float m_run = -INFINITY, l_run = 0.0f;
      for (int j = 0; j < n; ++j, ++done) {
        if (!(ok = warp_wait(smem_u32(&s_full[t]), done & 1u, watch, lane))) break;
        tc_fence_after();
        // Both halves for the maximum; the second stays in registers, the first is read again for its probabilities.
        const int valid = seen - j * kKeys;
        const bool full_tile = __all_sync(0xffffffffu, valid >= kKeys);
        uint32_t s[kHalf];
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tmem_ld32_nowait(s_col + (uint32_t)(h * kHalf), s);
          tmem_ld32_nowait(s_col + (uint32_t)(h * kHalf) + 32u, s + 32);
          tmem_wait32(s);
          tmem_wait32(s + 32);
          mx = fmaxf(mx, full_tile ? half_maximum<false>(s, a.scale_log2, kHalf)
                                   : half_maximum<true>(s, a.scale_log2, valid - h * kHalf));
        }
        // The running maximum moves only when it would grow by more than 2^8: probabilities stay below 2^8 and the
        // output is rescaled rarely, exactly.
        const bool move = mx > m_run + 8.0f;
        const float m_use = move ? mx : m_run;
        const float alpha = move ? ex2(m_run - m_use) : 1.0f;
        const float m_sub = m_use == -INFINITY ? 0.0f : m_use;
        if (j > 0 && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_col + (uint32_t)c, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(o_col + (uint32_t)c, o);
          }
        }
        const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), nm2 = make_float2(-m_sub, -m_sub);
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int h = 1; h >= 0; --h) {
          if (h == 0) {
            tmem_ld32_nowait(s_col, s);
            tmem_ld32_nowait(s_col + 32u, s + 32);
            tmem_wait32(s);
            tmem_wait32(s + 32);
          }
          if (full_tile)
            probabilities<false, D>(s, sc2, nm2, kHalf, sum);
          else
            probabilities<true, D>(s, sc2, nm2, valid - h * kHalf, sum);
          tmem_st32(s_col + (uint32_t)(h * kHalf), s);  // over the first of the half's own columns
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(h == 1 ? &p_half[t] : &p_full[t]));
        }
        l_run = fmaf(l_run, alpha, sum.x + sum.y);
        m_run = m_use;
      }
      if (n > 0) {
        ok = ok && warp_wait(smem_u32(&o_done[t]), uses & 1u, watch, lane);
        ++uses;
      }
      if (!ok) break;
      tc_fence_after();
      const float inv = 1.0f / l_run;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(o_col + (uint32_t)c, o);
          if (c == D - 32) {  // the output is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&o_empty[t]));
          }
        }
        if (seen < 0) continue;
        uint32_t y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          y[e] = seen == 0 ? 0u : cvt2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
#pragma unroll
        for (int x = 0; x < 2; ++x) store_16(dst + c + 16 * x, y + 8 * x, ps.wide_out);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, 512);
  }
}

// ------------------------------------------------------------------ steps
// Scores and products are transposed: S^T [16 keys x 8 rows] = K Q^T and
// O^T [16 columns x 8 rows] += V^T P^T with mma.sync m16n8k16, so that the few
// rows (the query heads of one key/value head, times the few tokens) are the
// narrow side and keys and values go from global memory straight to operand
// registers, 16 bytes a load: the sum over columns (S) and the order of the
// columns (O) do not mind a permutation, so the 16 bytes that a thread loads
// are the columns that it stands for. Memory-bound work at an eighth of the
// legacy tensor path's rate; no shared memory, no barrier in the loop.
constexpr int kStepWarps = 4;
constexpr int kStepKeys = 16;

struct StepShape {
  int chunk;      // keys of a slot
  int slots;
  int max_rows;   // rows a sequence up to which its keys are split
  float* part_o;    // [parts][kv_heads][max_rows][D] unnormalised
  float2* part_ml;  // [parts][kv_heads][max_rows] maximum (base 2, scaled) and sum
};
// First part of a sequence of more than `chunk` keys that starts at key `ks`: such a sequence of l keys has
// ceil(l / chunk) <= floor(2 l / chunk) pieces, so the next one's parts start behind them.
__device__ __forceinline__ int64_t first_part(int ks, int chunk) { return (2 * (int64_t)ks + chunk - 1) / chunk; }

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// NT tiles of 8 rows. A CTA takes one slot's keys for one key/value head and
// every gridDim.z-th group of 8 NT rows.
template <int D, int NT>
__global__ void __launch_bounds__(32 * kStepWarps) step_kernel(const Args a, const StepShape ss) {
  constexpr int R = 8 * NT;
  __shared__ float sh_m[kStepWarps][R], sh_l[kStepWarps][R];
  __shared__ float sh_o[kStepWarps][R][D + 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int slot = blockIdx.x, kv_head = blockIdx.y;
  if (slot == 0 && kv_head == 0 && blockIdx.z == 0 && warp == 0) check_offsets(a, lane, 32);
  if (slot == 0 && blockIdx.z == 0) {  // tokens past the last offset
    const int from = clamped(a.cu_q, a.seqs, a.total_q);
    const int64_t count = (int64_t)(a.total_q - from) * a.group * (D / 8);
    for (int64_t i = threadIdx.x; i < count; i += 32 * kStepWarps) {
      const int64_t row = i / (D / 8);
      const int64_t at = ((from + row / a.group) * a.heads + kv_head * a.group + row % a.group) * D + i % (D / 8) * 8;
      *reinterpret_cast<uint4*>(a.out + at) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const int b = find_sequence(a.cu_k, a.seqs - 1, a.total_k, ss.chunk, slot, lane);
  const int ks = clamped(a.cu_k, b, a.total_k), lk = max(clamped(a.cu_k, b + 1, a.total_k) - ks, 0);
  const int qs = clamped(a.cu_q, b, a.total_q), lq = max(clamped(a.cu_q, b + 1, a.total_q) - qs, 0);
  const int rows = lq * a.group;
  const int index = slot - (int)((uint32_t)ks / (uint32_t)ss.chunk) - b;
  const int pieces = max((int)((lk + (int64_t)ss.chunk - 1) / ss.chunk), 1);
  // a sequence with more rows than the parts have room for is not split
  const bool split = pieces > 1 && rows <= ss.max_rows;
  if (index < 0 || index >= pieces || (index > 0 && !split)) return;
  const int k0 = split ? index * ss.chunk : 0, k1 = split ? min(k0 + ss.chunk, lk) : lk;

  for (int r0 = blockIdx.z * R; r0 < rows; r0 += gridDim.z * R) {
    // Q^T: row g of each row tile, the columns that this thread loads of K.
    uint32_t q[NT][D / 32][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = min(r0 + n * 8 + g, rows - 1);
      const bf16* src = a.q + (int64_t)(qs + r / a.group) * a.q_ts + (int64_t)(kv_head * a.group + r % a.group) * a.q_hs;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(src + c * 32 + t * 8);
        q[n][c][0] = w.x, q[n][c][1] = w.y, q[n][c][2] = w.z, q[n][c][3] = w.w;
      }
    }
    // Keys that rows 2 t, 2 t + 1 of each tile see.
    int see[NT][2];
    float m[NT][2], l[NT][2], o[NT][D / 16][4];
    int least = k1;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + n * 8 + 2 * t + e;
        see[n][e] = r >= rows ? k1 : a.causal ? min(max(r / a.group + lk - lq + 1, 0), lk) : lk;
        least = min(least, see[n][e]);
        m[n][e] = -INFINITY;
        l[n][e] = 0.0f;
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
    least = __reduce_min_sync(0xffffffffu, least);

    for (int k = k0 + warp * kStepKeys; k < k1; k += kStepWarps * kStepKeys) {
      // K: keys g, g + 8; V: keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9, columns 8 g of each 64
      uint4 kr[2][D / 32], vr[4][D / 64];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16* src = a.k + (int64_t)(ks + min(k + g + 8 * h, k1 - 1)) * a.k_ts + (int64_t)kv_head * a.k_hs + t * 8;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) kr[h][c] = ld_stream(src + c * 32);
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int key = k + 2 * t + (h & 1) + (h >> 1) * 8;
        const bf16* src = a.v + (int64_t)(ks + min(key, k1 - 1)) * a.v_ts + (int64_t)kv_head * a.v_hs + g * 8;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          vr[h][c] = ld_stream(src + c * 64);
          if (key >= k1) vr[h][c] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          mma_16816(s, kr[0][c].x, kr[1][c].x, kr[0][c].y, kr[1][c].y, q[n][c][0], q[n][c][1]);
          mma_16816(s, kr[0][c].z, kr[1][c].z, kr[0][c].w, kr[1][c].w, q[n][c][2], q[n][c][3]);
        }
        // s[e], s[2 + e]: keys k + g, k + g + 8 of row 2 t + e
        const bool masked = k + kStepKeys > least;
        float top[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[e] *= a.scale_log2;
          s[2 + e] *= a.scale_log2;
          if (masked && k + g >= see[n][e]) s[e] = -INFINITY;
          if (masked && k + g + 8 >= see[n][e]) s[2 + e] = -INFINITY;
          top[e] = fmaxf(s[e], s[2 + e]);
        }
        // as above: the maximum moves when it would grow by more than 2^8
        if (__any_sync(0xffffffffu, top[0] > m[n][0] + 8.0f || top[1] > m[n][1] + 8.0f)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], off));
            const float mn = fmaxf(m[n][e], top[e]);
            const float alpha = mn == -INFINITY ? 1.0f : ex2(m[n][e] - mn);
            m[n][e] = mn;
            l[n][e] *= alpha;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              o[n][i][e] *= alpha;
              o[n][i][2 + e] *= alpha;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float sub = m[n][e] == -INFINITY ? 0.0f : m[n][e];
          s[e] = ex2(s[e] - sub);
          s[2 + e] = ex2(s[2 + e] - sub);
          l[n][e] += s[e] + s[2 + e];
        }
        pb[n][0] = transpose8x8(cvt2(s[0], s[1]));
        pb[n][1] = transpose8x8(cvt2(s[2], s[3]));
      }
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const uint32_t v0[4] = {vr[0][c].x, vr[0][c].y, vr[0][c].z, vr[0][c].w};
        const uint32_t v1[4] = {vr[1][c].x, vr[1][c].y, vr[1][c].z, vr[1][c].w};
        const uint32_t v2[4] = {vr[2][c].x, vr[2][c].y, vr[2][c].z, vr[2][c].w};
        const uint32_t v3[4] = {vr[3][c].x, vr[3][c].y, vr[3][c].z, vr[3][c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // output rows g and g + 8 of the MMA are columns 8 g + 2 i and + 1
          const uint32_t a0 = __byte_perm(v0[i], v1[i], 0x5410), a1 = __byte_perm(v0[i], v1[i], 0x7632);
          const uint32_t a2 = __byte_perm(v2[i], v3[i], 0x5410), a3 = __byte_perm(v2[i], v3[i], 0x7632);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816(o[n][c * 4 + i], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        }
      }
    }
    allow_dependent();  // join_kernel looks its row up meanwhile
    // The warps' parts to shared memory, added in order.
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], off);
        const int r = n * 8 + 2 * t + e;
        if (g == 0) {
          sh_m[warp][r] = m[n][e];
          sh_l[warp][r] = l[n][e];
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          float* dst = &sh_o[warp][r][i / 4 * 64 + 8 * g + 2 * (i % 4)];
          dst[0] = o[n][i][e];
          dst[1] = o[n][i][2 + e];
        }
      }
    __syncthreads();
    for (int r = warp; r < R && r0 + r < rows; r += kStepWarps) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kStepWarps; ++w) top = fmaxf(top, sh_m[w][r]);
      const float sub = top == -INFINITY ? 0.0f : top;
      float f[kStepWarps], sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kStepWarps; ++w) {
        f[w] = ex2(sh_m[w][r] - sub);
        sum = fmaf(sh_l[w][r], f[w], sum);
      }
      float y[D / 32];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        y[c] = 0.0f;
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w) y[c] = fmaf(sh_o[w][r][c * 32 + lane], f[w], y[c]);
      }
      const int row = r0 + r;
      if (split) {
        const int64_t at = ((first_part(ks, ss.chunk) + index) * a.kv_heads + kv_head) * ss.max_rows + row;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) ss.part_o[at * D + c * 32 + lane] = y[c];
        if (lane == 0) ss.part_ml[at] = make_float2(top, sum);
      } else {
        const int token = row / a.group;
        const int seen = a.causal ? min(token + lk - lq + 1, lk) : lk;
        const float inv = 1.0f / sum;
        bf16* dst = a.out + ((int64_t)(qs + token) * a.heads + kv_head * a.group + row % a.group) * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) dst[c * 32 + lane] = __float2bfloat16_rn(seen > 0 ? y[c] * inv : 0.0f);
      }
    }
  }
}

// The parts of the sequences whose keys were split: a block a row, a thread a
// column and every THREADS / D-th part; the groups' sums are added in order.
template <int D, int THREADS>
__global__ void __launch_bounds__(THREADS) join_kernel(const Args a, const StepShape ss) {
  constexpr int kGroups = THREADS / D;
  __shared__ float sh_y[kGroups][D], sh_l[kGroups];
  const int lane = threadIdx.x & 31;
  const int col = threadIdx.x % D, group = threadIdx.x / D;
  const int64_t item = blockIdx.x;
  const int tok = (int)(item / a.heads), head = (int)(item % a.heads);
  int b = 0, n = a.seqs;  // the last sequence that starts at or before the token
  while (n > 1) {
    const int stride = (n + 31) / 32, at = b + lane * stride;
    const int hits = __popc(__ballot_sync(0xffffffffu, at < b + n && a.cu_q[at] <= tok));
    const int step = max(hits - 1, 0) * stride;
    n = min(stride, n - step);
    b += step;
  }
  const int qs = clamped(a.cu_q, b, a.total_q), lq = max(clamped(a.cu_q, b + 1, a.total_q) - qs, 0);
  const int ks = clamped(a.cu_k, b, a.total_k), lk = max(clamped(a.cu_k, b + 1, a.total_k) - ks, 0);
  const int pieces = (int)((lk + (int64_t)ss.chunk - 1) / ss.chunk);
  if (pieces <= 1 || (int64_t)lq * a.group > ss.max_rows || tok < qs || tok >= qs + lq) {
    wait_for_predecessor();
    return;
  }
  const int row = (tok - qs) * a.group + head % a.group;
  const int seen = a.causal ? min(tok - qs + lk - lq + 1, lk) : lk;
  const int64_t stride = (int64_t)a.kv_heads * ss.max_rows;
  const int64_t at = (first_part(ks, ss.chunk) * a.kv_heads + head / a.group) * ss.max_rows + row;
  wait_for_predecessor();
  float top = -INFINITY;
  for (int p = lane; p < pieces; p += 32) top = fmaxf(top, ss.part_ml[at + p * stride].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  const float sub = top == -INFINITY ? 0.0f : top;
  float y = 0.0f, sum = 0.0f;
#pragma unroll 8
  for (int p = group; p < pieces; p += kGroups) {
    const float2 ml = ss.part_ml[at + p * stride];
    const float f = ex2(ml.x - sub);
    sum = fmaf(ml.y, f, sum);
    y = fmaf(ss.part_o[(at + p * stride) * D + col], f, y);
  }
  sh_y[group][col] = y;
  if (col == 0) sh_l[group] = sum;
  __syncthreads();
  if (group != 0) return;
#pragma unroll
  for (int w = 1; w < kGroups; ++w) {
    y += sh_y[w][col];
    sum += sh_l[w];
  }
  a.out[item * D + col] = __float2bfloat16_rn(seen > 0 ? y * (1.0f / sum) : 0.0f);
}

// ------------------------------------------------------------------ host
// How a call is laid out, from what the host knows: token and sequence counts.
struct Plan {
  bool step;
  int chunk, slots, max_rows;
  int64_t parts;  // room for parts, 0 where no sequence can be long enough to be split
  int64_t bytes;  // of workspace
};
Plan plan(int64_t seqs, int64_t total_q, int64_t total_k, int64_t group, int64_t kv_heads, int64_t head_dim) {
  Plan p{};
  const int64_t queries = (total_q + seqs - 1) / seqs;  // a sequence, on average
  p.step = queries * group <= 64;
  if (!p.step) return p;
  // slots for three waves of four CTAs an SM, for one whole wave when there is one sequence
  const int64_t want = (int64_t)sm_count() * 4 * (seqs > 1 ? 3 : 1) / kv_heads;
  int64_t chunk = (total_k + (want > 0 ? want : 1) - 1) / (want > 0 ? want : 1);
  chunk = (chunk + 63) / 64 * 64;
  // Shorter pieces cost more at the join than they save; up to 512 keys none is made (300 keys: one kernel takes 6.8 us, two
  // 7.7; 1000 keys in pieces of 256, 512, 1024: 9.1, 11.7, 16.1 us).
  if (chunk < 256) chunk = total_k <= 512 ? 512 : 256;
  p.chunk = (int)chunk;
  p.slots = (int)(total_k / chunk + seqs);
  int64_t most = 1;
  while (most < queries) most *= 2;
  p.max_rows = (int)(most * group);
  p.parts = total_k > chunk ? 2 * total_k / chunk + 2 : 0;
  p.bytes = p.parts * kv_heads * p.max_rows * (head_dim + 2) * 4;
  return p;
}

template <int D>
int head_map(CUtensorMap* map, const void* base, int64_t heads, int64_t tokens, int64_t ts, int64_t hs, uint32_t box_heads,
             uint32_t box_tokens) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)ts * 2};
  const cuuint32_t box[3] = {64, box_heads, box_tokens};
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D>
int launch_prompt(const Args& a, cudaStream_t stream) {
  using C = Prompt<D>;
  PromptShape ps;
  ps.head_parts = (a.group + kRows - 1) / kRows;
  ps.tile_heads = (a.group + ps.head_parts - 1) / ps.head_parts;
  ps.tokens_tile = kRows / ps.tile_heads;
  ps.slots = a.total_q / (2 * ps.tokens_tile) + a.seqs + 1;
  const int64_t items = (int64_t)ps.slots * a.kv_heads * ps.head_parts;
  LR_REQUIRE(items <= INT32_MAX - 65536, "attention_packed: too many blocks");
  ps.items = (int)items;
  ps.wide_out = aligned(a.out, 32);
  CUtensorMap mq, mk{}, mv{};
  int st = head_map<D>(&mq, a.q, a.heads, a.total_q, a.q_ts, a.q_hs, (uint32_t)ps.tile_heads, (uint32_t)ps.tokens_tile);
  if (st) return st;
  if (a.total_k > 0 && ((st = head_map<D>(&mk, a.k, a.kv_heads, a.total_k, a.k_ts, a.k_hs, 1, kKeys)) ||
                        (st = head_map<D>(&mv, a.v, a.kv_heads, a.total_k, a.v_ts, a.v_hs, 1, kKeys))))
    return st;
  static bool done[64] = {};
  if ((st = configure_smem(prompt_kernel<D>, C::kSmem, done))) return st;
  prompt_kernel<D><<<(unsigned)(items < sm_count() ? items : sm_count()), kPromptThreads, C::kSmem, stream>>>(mq, mk, mv, a, ps);
  return launch_status("attention_packed (prompts)");
}

template <int D>
int launch_step(const Args& a, const Plan& p, void* workspace, cudaStream_t stream) {
  StepShape ss{p.chunk, p.slots, p.max_rows, nullptr, nullptr};
  if (p.bytes > 0) {
    ss.part_o = static_cast<float*>(workspace);
    ss.part_ml = reinterpret_cast<float2*>(ss.part_o + p.parts * a.kv_heads * p.max_rows * D);
  }
  const int nt = p.max_rows <= 8 ? 1 : 2;
  const dim3 grid((unsigned)p.slots, (unsigned)a.kv_heads, (unsigned)((p.max_rows + 8 * nt - 1) / (8 * nt)));
  if (nt == 1)
    step_kernel<D, 1><<<grid, 32 * kStepWarps, 0, stream>>>(a, ss);
  else
    step_kernel<D, 2><<<grid, 32 * kStepWarps, 0, stream>>>(a, ss);
  int st = launch_status("attention_packed (steps)");
  if (st || p.bytes == 0) return st;
  const int64_t rows = (int64_t)a.total_q * a.heads;
  LR_REQUIRE(rows <= INT32_MAX, "attention_packed: too many rows");
  // a thread takes about eight parts at most: one token against 32768 keys 33.8 us with 256 threads, 30.2 us with 512
  // (64 requests of a few parts each, 139 us, lose 5 us to the larger blocks)
  const int parts_each = p.slots / a.seqs;
  const auto join = parts_each > 32 ? join_kernel<D, 1024> : parts_each > 8 ? join_kernel<D, 512> : join_kernel<D, 128>;
  const unsigned threads = parts_each > 32 ? 1024 : parts_each > 8 ? 512 : 128;
  return launch("attention_packed (join)", join, dim3((unsigned)rows), threads, 0, stream, 1, true, a, ss);
}

}  // namespace
}  // namespace packed

int read_status_packed(unsigned int* bits, int clear) {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_packed_status, sizeof(v)) != cudaSuccess)
    return launch_status("reading the device status");
  if (clear) {
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbol(g_packed_status, &zero, sizeof(zero)) != cudaSuccess)
      return launch_status("clearing the device status");
  }
  *bits |= v;
  return LR_OK;
}

}  // namespace lr

static int check_packed(int64_t seqs, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  using namespace lr;
  LR_REQUIRE(seqs > 0 && total_q >= 0 && total_k >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
             "attention_packed: invalid shape");
  LR_REQUIRE(seqs < (1 << 30) && total_q < (1 << 30) && total_k < (1 << 30) && heads <= 65535, "attention_packed: shape too large");
  if (head_dim != 64 && head_dim != 128)
    return set_error(LR_ERR_UNSUPPORTED, "attention_packed: head_dim %lld (64 or 128)", (long long)head_dim);
  return LR_OK;
}

extern "C" int64_t lr_attention_packed_workspace_bytes(int64_t seqs, int64_t total_q, int64_t total_k, int64_t heads,
                                                       int64_t kv_heads, int64_t head_dim) {
  if (check_packed(seqs, total_q, total_k, heads, kv_heads, head_dim) || total_q == 0) return 0;
  return lr::packed::plan(seqs, total_q, total_k, heads / kv_heads, kv_heads, head_dim).bytes;
}

extern "C" int lr_attention_packed(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                   int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                   int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_q,
                                   const int32_t* cu_k, int64_t seqs, int64_t total_q, int64_t total_k, int64_t heads,
                                   int64_t kv_heads, int64_t head_dim, int causal, float scale, void* out,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lr;
  const int st = check_packed(seqs, total_q, total_k, heads, kv_heads, head_dim);
  if (st) return st;
  if (total_q == 0) return LR_OK;
  LR_REQUIRE(q && out && cu_q && cu_k && (total_k == 0 || (k && v)), "attention_packed: null pointer");
  LR_REQUIRE(q_token_stride >= 0 && q_head_stride >= 0 && k_token_stride >= 0 && k_head_stride >= 0 &&
                 v_token_stride >= 0 && v_head_stride >= 0,
             "attention_packed: negative strides");
  if (q_token_stride % 8 || q_head_stride % 8 || k_token_stride % 8 || k_head_stride % 8 || v_token_stride % 8 ||
      v_head_stride % 8 || !aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
    return set_error(LR_ERR_UNSUPPORTED, "attention_packed: pointers and strides must be 16-byte aligned");
  const int64_t group = heads / kv_heads;
  const packed::Plan p = packed::plan(seqs, total_q, total_k, group, kv_heads, head_dim);
  LR_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && aligned(workspace, 16)),
             "attention_packed: a workspace of %lld bytes is needed", (long long)p.bytes);
  const packed::Args a{static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(k),
                       static_cast<const __nv_bfloat16*>(v), static_cast<__nv_bfloat16*>(out), q_token_stride,
                       q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride, cu_q, cu_k,
                       (int)seqs, (int)total_q, (int)total_k, (int)heads, (int)kv_heads, (int)group, causal,
                       (float)((double)scale * 1.4426950408889634)};
  auto* s = static_cast<cudaStream_t>(stream);
  if (p.step)
    return head_dim == 64 ? packed::launch_step<64>(a, p, workspace, s) : packed::launch_step<128>(a, p, workspace, s);
  return head_dim == 64 ? packed::launch_prompt<64>(a, s) : packed::launch_prompt<128>(a, s);
}
