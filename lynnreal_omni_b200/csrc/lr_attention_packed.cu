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
//   * behind a prefix that all sequences share: prompt_kernel with the prefix's key
//     tiles first, or both kernels side by side on parts, and join_prefix_kernel.
#include <type_traits>

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

// What a prefix in front of every sequence adds to the prompt kernel.
enum PrefixMode {
  kNoPrefix,
  kWithPrefix,  // a block takes the prefix's keys, then its sequence's
  kPrefixPart,  // a block takes a run of the prefix's keys for rows of any sequences and leaves a part
};
struct Prefix {
  int keys, tiles;
  int chunk, chunks;  // kPrefixPart: keys of a run, runs
  float* part_o;      // [chunks][total_q][heads][D] unnormalised
  float2* part_ml;    // [chunks][total_q][heads] maximum (base 2, scaled) and sum
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
template <int MODE>
__device__ __forceinline__ bool prompt_item(const Args& a, const PromptShape& ps, const Prefix& px, int index, int lane,
                                            PromptItem& w) {
  const int parts = a.kv_heads * ps.head_parts;
  const int part = index % parts, rank = index / parts;
  w.kv_head = part / ps.head_parts;
  const int in_group = part % ps.head_parts * ps.tile_heads;
  w.heads_here = min(ps.tile_heads, a.group - in_group);
  w.head0 = w.kv_head * a.group + in_group;
  const int block = 2 * ps.tokens_tile;
  if constexpr (MODE == kPrefixPart) {  // rank: run of keys, then block of tokens
    w.tok0 = rank / px.chunks * block;
    w.q_row = w.tok0;
    w.lq = a.total_q;
    w.k_row = rank % px.chunks * px.chunk;
    w.lk = min(px.chunk, px.keys - w.k_row);
#pragma unroll
    for (int t = 0; t < 2; ++t) w.tiles[t] = w.tok0 + t * ps.tokens_tile < w.lq ? (w.lk + kKeys - 1) / kKeys : 0;
    return true;
  }
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
    if (MODE == kWithPrefix && first < w.lq && b < a.seqs) w.tiles[t] += px.tiles;
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
//
// With a prefix (kWithPrefix) its key tiles come first, from maps of their own;
// as parts (kPrefixPart) map_k and map_v are the prefix's.
template <int D, int MODE>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Args a, const PromptShape ps,
                  const __grid_constant__ CUtensorMap map_pk, const __grid_constant__ CUtensorMap map_pv, const Prefix px) {
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
    if (MODE == kPrefixPart || a.total_k > 0) {  // else there is no map
      prefetch_map(&map_k);
      prefetch_map(&map_v);
    }
    if (MODE == kWithPrefix) {
      prefetch_map(&map_pk);
      prefetch_map(&map_pv);
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
  if (MODE == kPrefixPart) allow_dependent();  // step_kernel, a block of which waits for this one, so that the join finds both's parts
  if (warp == 3) first_there = prompt_item<MODE>(a, ps, px, item_index(0), lane, first);
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
      if (MODE != kPrefixPart && blockIdx.x == 0) check_offsets(a, lane, 32);
      uint32_t number = 0;
      for (int round = 0;; ++round) {
        PromptItem w{};
        const bool end = round * (int64_t)gridDim.x >= ps.items;
        if (round == 0) {
          if (!first_there) continue;
          w = first;
        } else if (!end && (item_index(round) >= ps.items || !prompt_item<MODE>(a, ps, px, item_index(round), lane, w))) {
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
            const int tile = i >> 1;
            if (MODE == kWithPrefix && tile < px.tiles) {
#pragma unroll
              for (int x = 0; x < D / 64; ++x)
                tma_load_3d(dst + x * kAtom, i & 1 ? &map_pv : &map_pk, bar, x * 64, w.kv_head, tile * kKeys);
            } else {
              const int row = w.k_row + (MODE == kWithPrefix ? tile - px.tiles : tile) * kKeys;
#pragma unroll
              for (int x = 0; x < D / 64; ++x) tma_load_3d(dst + x * kAtom, i & 1 ? &map_v : &map_k, bar, x * 64, w.kv_head, row);
            }
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
          const int before = MODE == kWithPrefix ? px.tiles : 0;  // tiles of the prefix: past its end there are zeros
          if (j >= before && j == most - 1 && (most - before) * kKeys > w.lk) {
            // The last V tile ends past the sequence: its rows there, another sequence's, become zeros (their
            // probabilities are 0, but 0 times an infinity is not).
            uint8_t* tile = smem + C::kRing + (ev % C::kSlots) * C::kTile;
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
              for (int i = (w.lk - (j - before) * kKeys) * 8 + lane; i < kKeys * 8; i += 32)
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
      bool there = false;
      bf16* dst = a.out;
      int64_t part = 0;
      {
        const int offset = t * ps.tokens_tile + in_tile;  // of this row's token in the block
        const int token = w.tok0 + offset;
        if (in_tile < ps.tokens_tile && head < w.heads_here && token < w.lq) {
          there = true;
          seen = MODE != kPrefixPart && a.causal ? min(max(token + w.lk - w.lq + 1, 0), w.lk) : w.lk;
          const int64_t at = (int64_t)(w.q_row + offset) * a.heads + w.head0 + head;
          dst += at * D;
          if (MODE == kPrefixPart) part = (int64_t)(w.k_row / px.chunk) * a.total_q * a.heads + at;
        } else if (MODE != kNoPrefix) {
          // A row that stands for nothing sees every key, so that its warp has no mask to test: 48 prompts of 1 to 512 tokens
          // behind 1000 keys 183 us with no key, 167 us with all.
          seen = w.lk;
        }
      }
      const int n = w.tiles[t];
      float m_run = -INFINITY, l_run = 0.0f;
      for (int j = 0; j < n; ++j, ++done) {
        if (!(ok = warp_wait(smem_u32(&s_full[t]), done & 1u, watch, lane))) break;
        tc_fence_after();
        // Both halves for the maximum; the second stays in registers, the first is read again for its probabilities.
        const int valid = MODE == kWithPrefix ? (j < px.tiles ? px.keys - j * kKeys : seen - (j - px.tiles) * kKeys)
                                              : seen - j * kKeys;
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
        if (!there) continue;
        if constexpr (MODE == kPrefixPart) {
          float* to = px.part_o + part * D + c;
#pragma unroll
          for (int x = 0; x < 4; ++x)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + 8 * x), "r"(o[8 * x]),
                         "r"(o[8 * x + 1]), "r"(o[8 * x + 2]), "r"(o[8 * x + 3]), "r"(o[8 * x + 4]), "r"(o[8 * x + 5]),
                         "r"(o[8 * x + 6]), "r"(o[8 * x + 7])
                         : "memory");
          if (c == 0) px.part_ml[part] = make_float2(m_run, l_run);
        } else {
          uint32_t y[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            y[e] = (MODE == kWithPrefix ? n == 0 : seen == 0)
                       ? 0u
                       : cvt2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
#pragma unroll
          for (int x = 0; x < 2; ++x) store_16(dst + c + 16 * x, y + 8 * x, ps.wide_out);
        }
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

// The last sequence of which before(its first key, its first query, its number) holds, with both its ranges. One round of
// loads, four candidates a lane, up to 127 sequences, two up to 2047.
struct Ranges {
  int ks, ke, qs, qe, b;
};
template <typename Before>
__device__ __forceinline__ Ranges find_ranges(const Args& a, int lane, Before before) {
  const auto key = [&](int i) { return clamped(a.cu_k, min(i, a.seqs), a.total_k); };
  const auto query = [&](int i) { return clamped(a.cu_q, min(i, a.seqs), a.total_q); };
  int lo = 0;
  if (a.seqs > 127) {
    int64_t stride = 64;  // the answer lies in [lo, lo + 32 stride)
    while (32 * stride < a.seqs) stride *= 32;
    for (;; stride /= 32) {
      const int64_t at = lo + lane * stride;
      const bool there = at < a.seqs;
      const int i = there ? (int)at : 0;
      const int hits = __popc(__ballot_sync(0xffffffffu, there && before(key(i), query(i), i)));
      lo += max(hits - 1, 0) * (int)stride;
      if (stride == 64) break;
    }
  }
  int k[4], q[4], hits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = key(lo + 32 * i + lane), q[i] = query(lo + 32 * i + lane);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = lo + 32 * i + lane;
    hits += __popc(__ballot_sync(0xffffffffu, at < a.seqs && before(k[i], q[i], at)));
  }
  const int b = min(max(hits - 1, 0), 126);  // as many hold where offsets do not go down
  const auto pick = [&](const int(&v)[4], int at) {
    const int i = at >> 5;
    return __shfl_sync(0xffffffffu, i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3], at & 31);
  };
  return Ranges{pick(k, b), pick(k, b + 1), pick(q, b), pick(q, b + 1), lo + b};
}

// What a prefix in front of every sequence adds to the step kernel.
struct StepPrefix {
  const bf16 *k, *v;
  int64_t k_ts, k_hs, v_ts, v_hs;
  int keys;
  int chunk, chunks;  // keys of a part of the prefix, parts
  int slots;          // chunks where this kernel makes the prefix's parts itself, 0 where prompt_kernel does
  float *part_o, *own_o;      // [chunks][total_q][heads][D], [total_q][heads][D] (the sequences that are not split)
  float2 *part_ml, *own_ml;
};

// NT tiles of 8 rows. A CTA takes one slot's keys for one key/value head and
// every gridDim.z-th group of 8 NT rows.
//
// SHARED: behind a prefix; every row leaves a part, which join_prefix_kernel joins
// with the prefix's. Those either come from this kernel's first slots, for the
// rows of all sequences, or from prompt_kernel, which runs meanwhile: one block
// waits for it, so that this kernel does not end before it.
//
// WARPS: of a slot and head. One where there are enough slots and heads to fill
// the GPU: a block is then that many heads side by side, and no warp waits for
// another.
template <int D, int NT, int WARPS, bool SHARED>
__global__ void __launch_bounds__(32 * kStepWarps, NT == 1 ? (WARPS == 1 && D == 64 ? 3 : 4) : 2) step_kernel(const Args a, const StepShape ss, const StepPrefix sp) {
  constexpr int R = 8 * NT;
  constexpr int kHeads = kStepWarps / WARPS;
  // Steps whose keys are under way together: 64 columns are half as many bytes, and a warp alone has no other to wait with.
  constexpr int kUnder = WARPS == 1 && D == 64 && NT == 1 ? 2 : 1;
  __shared__ float sh_m[kStepWarps][R], sh_l[kStepWarps][R];
  __shared__ float sh_o[kStepWarps][R][D + 4];
  if (SHARED && blockIdx.x == gridDim.x - 1) {
    if ((blockIdx.y | blockIdx.z) == 0) wait_for_predecessor();
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const bool of_prefix = SHARED && (int)blockIdx.x < sp.slots;
  const int slot = SHARED ? (int)blockIdx.x - sp.slots : (int)blockIdx.x;
  const int kv_head = kHeads == 1 ? (int)blockIdx.y : (int)blockIdx.y * kHeads + warp;
  const int first_warp = kHeads == 1 ? 0 : warp;  // of this head's
  if (kHeads > 1 && kv_head >= a.kv_heads) return;
  if (slot == 0 && kv_head == 0 && blockIdx.z == 0 && warp == 0) check_offsets(a, lane, 32);
  if (slot == 0 && blockIdx.z == 0) {  // tokens past the last offset
    const int from = clamped(a.cu_q, a.seqs, a.total_q);
    const int64_t count = (int64_t)(a.total_q - from) * a.group * (D / 8);
    for (int64_t i = threadIdx.x - 32 * first_warp; i < count; i += 32 * WARPS) {
      const int64_t row = i / (D / 8);
      const int64_t at = ((from + row / a.group) * a.heads + kv_head * a.group + row % a.group) * D + i % (D / 8) * 8;
      *reinterpret_cast<uint4*>(a.out + at) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  int ks = 0, lk = sp.keys, qs = 0, lq = a.total_q, index = blockIdx.x, k0, k1;
  bool split = false, causal = false;
  const bf16 *keys = a.k, *values = a.v;
  int64_t k_ts = a.k_ts, k_hs = a.k_hs, v_ts = a.v_ts, v_hs = a.v_hs;
  if (SHARED && of_prefix) {
    keys = sp.k, values = sp.v;
    k_ts = sp.k_ts, k_hs = sp.k_hs, v_ts = sp.v_ts, v_hs = sp.v_hs;
    k0 = index * sp.chunk;
    k1 = min(k0 + sp.chunk, lk);
  } else {
    int b;
    if constexpr (SHARED) {
      const Ranges r = find_ranges(a, lane, [&](int k, int, int at) { return (int)((uint32_t)k / (uint32_t)ss.chunk) + at <= slot; });
      b = r.b, ks = r.ks, lk = max(r.ke - ks, 0), qs = r.qs, lq = max(r.qe - qs, 0);
    } else {
      b = find_sequence(a.cu_k, a.seqs - 1, a.total_k, ss.chunk, slot, lane);
      ks = clamped(a.cu_k, b, a.total_k), lk = max(clamped(a.cu_k, b + 1, a.total_k) - ks, 0);
      qs = clamped(a.cu_q, b, a.total_q), lq = max(clamped(a.cu_q, b + 1, a.total_q) - qs, 0);
    }
    index = slot - (int)((uint32_t)ks / (uint32_t)ss.chunk) - b;
    const int pieces = max((int)((lk + (int64_t)ss.chunk - 1) / ss.chunk), 1);
    // a sequence with more rows than the parts have room for is not split
    split = pieces > 1 && (int64_t)lq * a.group <= ss.max_rows;
    if (index < 0 || index >= pieces || (index > 0 && !split)) return;
    k0 = split ? index * ss.chunk : 0, k1 = split ? min(k0 + ss.chunk, lk) : lk;
    causal = a.causal;
  }
  const int rows = lq * a.group;

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
        see[n][e] = r >= rows ? k1 : causal ? min(max(r / a.group + lk - lq + 1, 0), lk) : lk;
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

    for (int kk = k0 + (warp - first_warp) * kStepKeys; kk < k1; kk += kUnder * WARPS * kStepKeys) {
      // K: keys g, g + 8; V: keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9, columns 8 g of each 64
      uint4 kr[kUnder][2][D / 32], vr[kUnder][4][D / 64];
#pragma unroll
      for (int u = 0; u < kUnder; ++u) {
        const int k = kk + u * WARPS * kStepKeys;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16* src = keys + (int64_t)(ks + min(k + g + 8 * h, k1 - 1)) * k_ts + (int64_t)kv_head * k_hs + t * 8;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) kr[u][h][c] = ld_stream(src + c * 32);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int key = k + 2 * t + (h & 1) + (h >> 1) * 8;
          const bf16* src = values + (int64_t)(ks + min(key, k1 - 1)) * v_ts + (int64_t)kv_head * v_hs + g * 8;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            vr[u][h][c] = ld_stream(src + c * 64);
            if (key >= k1) vr[u][h][c] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnder; ++u) {
        const int k = kk + u * WARPS * kStepKeys;
        if (u > 0 && k >= k1) break;
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            mma_16816(s, kr[u][0][c].x, kr[u][1][c].x, kr[u][0][c].y, kr[u][1][c].y, q[n][c][0], q[n][c][1]);
            mma_16816(s, kr[u][0][c].z, kr[u][1][c].z, kr[u][0][c].w, kr[u][1][c].w, q[n][c][2], q[n][c][3]);
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
          const uint32_t v0[4] = {vr[u][0][c].x, vr[u][0][c].y, vr[u][0][c].z, vr[u][0][c].w};
          const uint32_t v1[4] = {vr[u][1][c].x, vr[u][1][c].y, vr[u][1][c].z, vr[u][1][c].w};
          const uint32_t v2[4] = {vr[u][2][c].x, vr[u][2][c].y, vr[u][2][c].z, vr[u][2][c].w};
          const uint32_t v3[4] = {vr[u][3][c].x, vr[u][3][c].y, vr[u][3][c].z, vr[u][3][c].w};
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
    }
    allow_dependent();  // join_kernel looks its row up meanwhile
    // The warps' parts to shared memory, added in order.
    if (kHeads == 1) __syncthreads(); else __syncwarp();
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
    if (kHeads == 1) __syncthreads(); else __syncwarp();
    for (int r = warp - first_warp; r < R && r0 + r < rows; r += WARPS) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sh_m[first_warp + w][r]);
      const float sub = top == -INFINITY ? 0.0f : top;
      float f[WARPS], sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        f[w] = ex2(sh_m[first_warp + w][r] - sub);
        sum = fmaf(sh_l[first_warp + w][r], f[w], sum);
      }
      float y[D / 32];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        y[c] = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) y[c] = fmaf(sh_o[first_warp + w][r][c * 32 + lane], f[w], y[c]);
      }
      const int row = r0 + r;
      if constexpr (SHARED) {
        const int64_t all = (int64_t)a.total_q * a.heads;
        const int64_t at = (int64_t)(qs + row / a.group) * a.heads + kv_head * a.group + row % a.group;
        if (of_prefix || !split) {
          float* to = of_prefix ? sp.part_o + index * all * D : sp.own_o;
          float2* to_ml = of_prefix ? sp.part_ml + index * all : sp.own_ml;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) to[at * D + c * 32 + lane] = y[c];
          if (lane == 0) to_ml[at] = make_float2(top, sum);
          continue;
        }
      }
      if (split) {
        const int64_t at = ((first_part(ks, ss.chunk) + index) * a.kv_heads + kv_head) * ss.max_rows + row;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) ss.part_o[at * D + c * 32 + lane] = y[c];
        if (lane == 0) ss.part_ml[at] = make_float2(top, sum);
      } else {
        const int token = row / a.group;
        const int seen = causal ? min(token + lk - lq + 1, lk) : lk;
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

// The parts of every row behind a prefix, the prefix's and then its sequence's
// own, added in that order: a warp a row, D / 32 columns a lane. Bound by latency:
// the next AHEAD parts are on their way while one is added, and fewer registers let
// more rows run where there are few parts (2048 rows of 9 parts 7 us, a block of
// 512 threads a row 29; 8192 rows of 5 parts 10.7 us with 8 ahead, 14.8 with 16).
constexpr int kJoinRows = 8;
template <int D, int AHEAD>
__global__ void __launch_bounds__(32 * kJoinRows, AHEAD <= 8 ? 4 : 2) join_prefix_kernel(const Args a, const StepShape ss, const StepPrefix sp) {
  using V = typename std::conditional<D == 128, float4, float2>::type;
  constexpr int kEach = D / 32, kAhead = AHEAD;  // parts whose values are under way together
  const int lane = threadIdx.x & 31;
  const int64_t all = (int64_t)a.total_q * a.heads, item = (int64_t)blockIdx.x * kJoinRows + (threadIdx.x >> 5);
  const int tok = (int)(min(item, all - 1) / a.heads), head = (int)(min(item, all - 1) % a.heads);
  const Ranges r = find_ranges(a, lane, [&](int, int q, int) { return q <= tok; });
  const int qs = r.qs, lq = max(r.qe - qs, 0), ks = r.ks, lk = max(r.ke - ks, 0);
  const int pieces = (int)((lk + (int64_t)ss.chunk - 1) / ss.chunk);
  const bool split = pieces > 1 && (int64_t)lq * a.group <= ss.max_rows;
  const int64_t at = (first_part(ks, ss.chunk) * a.kv_heads + head / a.group) * ss.max_rows + (tok - qs) * a.group + head % a.group;
  const int64_t stride = split ? (int64_t)a.kv_heads * ss.max_rows : 0;
  const float2* own_ml = split ? ss.part_ml + at : sp.own_ml + item;
  const float* own_o = split ? ss.part_o + at * D : sp.own_o + item * D;
  const int own = split ? pieces : 1, parts = sp.chunks + own;
  wait_for_predecessor();
  if (item >= all || tok < qs || tok >= qs + lq) return;  // tokens past the last offset have their zeros
  float top = -INFINITY, sum = 0.0f, y[kEach];
#pragma unroll
  for (int c = 0; c < kEach; ++c) y[c] = 0.0f;
  // 32 parts at a time: a lane has one's maximum and sum
  for (int p0 = 0; p0 < parts; p0 += 32) {
    const int here = min(parts - p0, 32), mine = p0 + lane;
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (mine < parts) ml = mine < sp.chunks ? sp.part_ml[mine * all + item] : own_ml[(mine - sp.chunks) * stride];
    V v[kAhead];
    const auto value = [&](int p) {
      const float* o = p < sp.chunks ? sp.part_o + (p * all + item) * D : own_o + (p - sp.chunks) * stride * D;
      return reinterpret_cast<const V*>(o)[lane];
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (i < here) v[i] = value(p0 + i);
    float most = fmaxf(top, ml.x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    const float sub = most == -INFINITY ? 0.0f : most, again = ex2(top - sub), weight = ex2(ml.x - sub);
    sum *= again;
#pragma unroll
    for (int c = 0; c < kEach; ++c) y[c] *= again;
    top = most;
    for (int p = 0; p < here; p += kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (p + i >= here) break;
        const float f = __shfl_sync(0xffffffffu, weight, p + i);
        sum = fmaf(__shfl_sync(0xffffffffu, ml.y, p + i), f, sum);
        const float* x = reinterpret_cast<const float*>(&v[i]);
#pragma unroll
        for (int c = 0; c < kEach; ++c) y[c] = fmaf(x[c], f, y[c]);
        if (p + i + kAhead < here) v[i] = value(p0 + p + i + kAhead);
      }
    }
  }
  const float inv = 1.0f / sum;
  uint32_t out[kEach / 2];
#pragma unroll
  for (int c = 0; c < kEach / 2; ++c) out[c] = cvt2(y[2 * c] * inv, y[2 * c + 1] * inv);
  using W = typename std::conditional<D == 128, uint2, uint32_t>::type;
  reinterpret_cast<W*>(a.out + item * D)[lane] = *reinterpret_cast<const W*>(out);
}

// ------------------------------------------------------------------ host
// How a call is laid out, from what the host knows: token and sequence counts.
struct Plan {
  bool step;
  bool narrow;  // one warp to a slot and head
  int chunk, slots, max_rows;
  int64_t parts;  // room for parts, 0 where no sequence can be long enough to be split
  int64_t bytes;  // of workspace
};
constexpr int64_t kMostRows = 65535 * 8;
Plan plan(int64_t seqs, int64_t total_q, int64_t total_k, int64_t group, int64_t kv_heads, int64_t head_dim, bool shared = false) {
  Plan p{};
  const int64_t queries = (total_q + seqs - 1) / seqs;  // a sequence, on average
  p.step = queries * group <= 64;
  if (!p.step && !shared) return p;
  // slots for three waves of four CTAs an SM, for one whole wave when there is one sequence
  const int64_t want = (int64_t)sm_count() * 4 * (seqs > 1 ? 3 : 1) / kv_heads;
  int64_t chunk = (total_k + (want > 0 ? want : 1) - 1) / (want > 0 ? want : 1);
  chunk = (chunk + 63) / 64 * 64;
  // Shorter pieces cost more at the join than they save; up to 512 keys none is made (300 keys: one kernel takes 6.8 us, two
  // 7.7; 1000 keys in pieces of 256, 512, 1024: 9.1, 11.7, 16.1 us).
  if (chunk < 256) chunk = total_k <= 512 ? 512 : 256;
  int64_t most = 1;
  while (most < queries) most *= 2;
  // Behind a prefix prompts, too, come here: sequences with more rows than a grid's z has are not split, their blocks go on by grids.
  p.max_rows = (int)(most * group < kMostRows ? most * group : kMostRows);
  if (shared && p.step) {
    // Behind a prefix a warp takes a slot and head alone where those are many, 128 keys each (64 requests of 64 to 1024 own
    // keys: 35.5 us, 41.8 with 256; four warps a slot 41.5 and 38.5). A row's part is as many bytes as a key and value of one
    // head, written and read: at least eight keys a row (58 requests of 8 tokens, up to 989 own keys, 32 rows a head: 93.6 us, 101
    // with 128 keys; 64 of 8 tokens, up to 4045, 64 rows: 600 and 752), and no more slots than four waves of warps take (64 of one
    // token, up to 16181 own keys: 330 and 372). Room for parts then stays below 26 % of the own keys and values.
    p.narrow = (total_k / 128 + seqs) * kv_heads >= 8 * sm_count();
    if (p.narrow) {
      const int64_t waves = 4 * 16 * (int64_t)sm_count(), even = (total_k * kv_heads + waves - 1) / waves;
      chunk = 8 * p.max_rows > 128 ? 8 * p.max_rows : 128;
      chunk = ((chunk > even ? chunk : even) + 63) / 64 * 64;
    }
  } else if (shared) {
    // Of prompts every 16 rows are blocks of their own, which mostly fill the GPU: as many slots as give it two blocks an SM (17
    // queries, 32 / 8 heads, 32768 own keys: 172 us, 536 in one piece, 221 in pieces of 128), else one for every other sequence,
    // which splits those far above the average.
    const int64_t asking = seqs < total_q ? seqs : total_q, blocks = asking * kv_heads * ((queries * group + 15) / 16);
    const int64_t pieces = 2 * sm_count() / blocks, slots = pieces > 1 ? asking * pieces : (asking + 1) / 2;
    chunk = ((total_k + slots - 1) / slots + 63) / 64 * 64;
    if (chunk < 256) chunk = total_k <= 512 ? 512 : 256;
  }
  p.chunk = (int)chunk;
  p.slots = (int)(total_k / chunk + seqs);
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

template <int D, int MODE>
int launch_prompt(const Args& a, const StepPrefix& sp, int64_t most_blocks, cudaStream_t stream) {
  using C = Prompt<D>;
  PromptShape ps;
  ps.head_parts = (a.group + kRows - 1) / kRows;
  ps.tile_heads = (a.group + ps.head_parts - 1) / ps.head_parts;
  ps.tokens_tile = kRows / ps.tile_heads;
  ps.slots = a.total_q / (2 * ps.tokens_tile) + a.seqs + 1;
  if (MODE == kPrefixPart) ps.slots = (a.total_q + 2 * ps.tokens_tile - 1) / (2 * ps.tokens_tile) * sp.chunks;
  const int64_t items = (int64_t)ps.slots * a.kv_heads * ps.head_parts;
  LR_REQUIRE(items <= INT32_MAX - 65536, "attention_packed: too many blocks");
  ps.items = (int)items;
  ps.wide_out = aligned(a.out, 32);
  const Prefix px{sp.keys, (sp.keys + kKeys - 1) / kKeys, sp.chunk, sp.chunks, sp.part_o, sp.part_ml};
  CUtensorMap mq, mk{}, mv{}, mpk{}, mpv{};
  int st = head_map<D>(&mq, a.q, a.heads, a.total_q, a.q_ts, a.q_hs, (uint32_t)ps.tile_heads, (uint32_t)ps.tokens_tile);
  if (st) return st;
  if (MODE != kNoPrefix && ((st = head_map<D>(&mpk, sp.k, a.kv_heads, sp.keys, sp.k_ts, sp.k_hs, 1, kKeys)) ||
                            (st = head_map<D>(&mpv, sp.v, a.kv_heads, sp.keys, sp.v_ts, sp.v_hs, 1, kKeys))))
    return st;
  if (MODE == kPrefixPart) mk = mpk, mv = mpv;
  if (MODE != kPrefixPart && a.total_k > 0 && ((st = head_map<D>(&mk, a.k, a.kv_heads, a.total_k, a.k_ts, a.k_hs, 1, kKeys)) ||
                        (st = head_map<D>(&mv, a.v, a.kv_heads, a.total_k, a.v_ts, a.v_hs, 1, kKeys))))
    return st;
  static bool done[64] = {};
  if ((st = configure_smem(prompt_kernel<D, MODE>, C::kSmem, done))) return st;
  // The ordinary way: behind its parts step_kernel is launched dependent, and reads operands and writes parts and rows of its own
  // without waiting for this one.
  prompt_kernel<D, MODE><<<(unsigned)(items < most_blocks ? items : most_blocks), kPromptThreads, C::kSmem, stream>>>(
      mq, mk, mv, a, ps, mpk, mpv, px);
  return launch_status(MODE == kNoPrefix ? "attention_packed (prompts)" : "attention_shared (prompts)");
}

template <int D, bool SHARED>
int launch_step(const Args& a, const Plan& p, const StepPrefix& sp, void* workspace, cudaStream_t stream) {
  StepShape ss{p.chunk, p.slots, p.max_rows, nullptr, nullptr};
  if (p.bytes > 0) {
    ss.part_o = static_cast<float*>(workspace);
    ss.part_ml = reinterpret_cast<float2*>(ss.part_o + p.parts * a.kv_heads * p.max_rows * D);
  }
  const int most_rows = sp.slots > 0 && a.total_q * a.group > p.max_rows ? a.total_q * a.group : p.max_rows;
  const int nt = most_rows <= 8 ? 1 : 2;
  const dim3 grid((unsigned)(p.slots + sp.slots), (unsigned)a.kv_heads, (unsigned)((most_rows + 8 * nt - 1) / (8 * nt)));
  const int64_t rows = (int64_t)a.total_q * a.heads;
  const StepPrefix none{};
  if constexpr (SHARED) {
    dim3 all = grid;
    all.x += 1;  // the block that waits for prompt_kernel
    if (p.narrow) all.y = (unsigned)((a.kv_heads + kStepWarps - 1) / kStepWarps);
    const auto kernel = nt == 1 ? (p.narrow ? step_kernel<D, 1, 1, true> : step_kernel<D, 1, kStepWarps, true>)
                                : (p.narrow ? step_kernel<D, 2, 1, true> : step_kernel<D, 2, kStepWarps, true>);
    const int st = launch("attention_shared (steps)", kernel, all, 32 * kStepWarps, 0, stream, 1, sp.slots == 0, a, ss, sp);
    if (st) return st;
    const auto join = sp.chunks + p.slots / a.seqs <= 8 ? join_prefix_kernel<D, 8> : join_prefix_kernel<D, 16>;
    return launch("attention_shared (join)", join, dim3((unsigned)((rows + kJoinRows - 1) / kJoinRows)),
                  32 * kJoinRows, 0, stream, 1, true, a, ss, sp);
  }
  const int st = launch("attention_packed (steps)", nt == 1 ? step_kernel<D, 1, kStepWarps, false> : step_kernel<D, 2, kStepWarps, false>,
                        grid, 32 * kStepWarps, 0, stream, 1, false, a, ss, none);
  if (st || p.bytes == 0) return st;
  // a thread takes about eight parts at most: one token against 32768 keys 33.8 us with 256 threads, 30.2 us with 512
  // (64 requests of a few parts each, 139 us, lose 5 us to the larger blocks)
  const int parts_each = p.slots / a.seqs;
  const auto join = parts_each > 32 ? join_kernel<D, 1024> : parts_each > 8 ? join_kernel<D, 512> : join_kernel<D, 128>;
  const unsigned threads = parts_each > 32 ? 1024 : parts_each > 8 ? 512 : 128;
  return launch("attention_packed (join)", join, dim3((unsigned)rows), threads, 0, stream, 1, true, a, ss);
}

// How a call behind a prefix is laid out.
struct SharedPlan {
  bool parts;       // the prefix in parts, else key tiles in front of every block's own
  bool step;        // parts by step_kernel, else by prompt_kernel
  int chunk, chunks;
  Plan own;         // parts: of the sequences' own keys
  int64_t prefix_at, own_at, bytes;  // of workspace: the prefix's parts, the parts of sequences that are not split
};
SharedPlan shared_plan(int64_t seqs, int64_t total_q, int64_t total_k, int64_t prefix, int64_t group, int64_t kv_heads,
                       int64_t head_dim) {
  SharedPlan p{};
  p.own = plan(seqs, total_q, total_k, group, kv_heads, head_dim, true);
  const int64_t rows = total_q * group;
  const int64_t head_parts = (group + kRows - 1) / kRows, tile_heads = (group + head_parts - 1) / head_parts;
  const int64_t tokens = 2 * (kRows / tile_heads), sms = sm_count();
  const int64_t blocks = (total_q + tokens - 1) / tokens * kv_heads * head_parts, tiles = (prefix + kKeys - 1) / kKeys;
  // The prefix in one piece needs a block for every `tokens` tokens, and part of one for each sequence. Where those leave
  // most SMs idle it is cut as for single tokens, although the rows' parts, those of the prefix and those of the own keys, then pass
  // through memory (at about 4 TB/s, and 6 us for the join) and step_kernel takes 16 rows at a time, their keys from L2 for each
  // (about 1.2 us for 16 keys, 8 warps an SM). A key tile takes about 1.65 us, a block 8 more. One prompt of 100 tokens behind 16384 keys:
  // 223 us in one piece, 48 in parts; 16 of 100 behind 2048: 76 and 161; behind 8192, 17 queries against 32768 own keys: 482 and 172;
  // 128 against 32768: 553 and 689; 128 against 8192: 227 and 177; 256 against 8192: 228 and 352.
  const int64_t most = sms / blocks > 1 ? (sms / blocks < tiles ? sms / blocks : tiles) : 1;
  if (!p.own.step) {
    const double own_keys = (double)total_k / seqs, own_tiles = own_keys / kKeys + 1;
    const double own_parts = own_keys > p.own.chunk ? own_keys / p.own.chunk + 1 : 1;
    const int64_t whole = blocks + seqs * kv_heads * head_parts / 2;
    const double whole_us = (double)((whole + sms - 1) / sms) * (8 + 1.65 * (tiles + own_tiles));
    const double parts_us = (double)((blocks * most + sms - 1) / sms) * (8 + 1.65 * ((tiles + most - 1) / most)) + 6 +
                            (double)rows * kv_heads * (most + own_parts) * (head_dim + 2) * 8 / 4e6 +
                            (double)rows / 16 * (own_keys / 16 + 1) * kv_heads * 1.2 / (8 * sms);
    if (parts_us >= whole_us) return p;
  }
  p.parts = true;
  p.step = rows <= 16;
  int64_t want;  // parts
  if (p.step) {
    want = sms * 4 / kv_heads > 1 ? sms * 4 / kv_heads : 1;
    p.chunk = 64;
  } else {
    // step_kernel runs on the SMs that this leaves, and on all of them afterwards: the parts should end when both together
    // would, the sequences' own keys going by at 4.5 TB/s.
    const double together = blocks * tiles * 1.65 / sms + (double)total_k * kv_heads * head_dim * 4 / 4.5e6;
    const int64_t each = together > 8 + 1.65 ? (int64_t)((together - 8) / 1.65) + 1 : 1;
    want = (tiles + each - 1) / each;
    if (want > most) want = most;
    p.chunk = kKeys;
  }
  p.chunk = (int)(((prefix + want - 1) / want + p.chunk - 1) / p.chunk * p.chunk);
  p.chunks = (int)((prefix + p.chunk - 1) / p.chunk);
  p.prefix_at = (p.own.bytes + 31) / 32 * 32;
  const int64_t row_bytes = (head_dim + 2) * 4, all = total_q * group * kv_heads;
  p.own_at = p.prefix_at + p.chunks * all * row_bytes;
  p.own_at = (p.own_at + 31) / 32 * 32;
  p.bytes = p.own_at + all * row_bytes;
  return p;
}

template <int D>
int launch_shared(const Args& a, const SharedPlan& p, StepPrefix sp, void* workspace, cudaStream_t stream) {
  if (!p.parts) return launch_prompt<D, kWithPrefix>(a, sp, sm_count(), stream);
  const int64_t all = (int64_t)a.total_q * a.heads;
  LR_REQUIRE(all <= INT32_MAX, "attention_shared: too many rows");  // of the join's and the steps' grids, before anything runs
  sp.chunk = p.chunk, sp.chunks = p.chunks, sp.slots = p.step ? p.chunks : 0;
  sp.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.prefix_at);
  sp.part_ml = reinterpret_cast<float2*>(sp.part_o + p.chunks * all * D);
  sp.own_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.own_at);
  sp.own_ml = reinterpret_cast<float2*>(sp.own_o + all * D);
  if (!p.step) {
    const int st = launch_prompt<D, kPrefixPart>(a, sp, sm_count(), stream);
    if (st) return st;
  }
  return launch_step<D, true>(a, p.own, sp, workspace, stream);
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
  const packed::StepPrefix none{};
  LR_REQUIRE(!p.step || total_q * heads <= INT32_MAX, "attention_packed: too many rows");
  if (p.step)
    return head_dim == 64 ? packed::launch_step<64, false>(a, p, none, workspace, s)
                          : packed::launch_step<128, false>(a, p, none, workspace, s);
  return head_dim == 64 ? packed::launch_prompt<64, packed::kNoPrefix>(a, none, sm_count(), s)
                        : packed::launch_prompt<128, packed::kNoPrefix>(a, none, sm_count(), s);
}

static int check_shared(int64_t seqs, int64_t total_q, int64_t total_k, int64_t prefix, int64_t heads, int64_t kv_heads,
                        int64_t head_dim) {
  const int st = check_packed(seqs, total_q, total_k, heads, kv_heads, head_dim);
  if (st) return st;
  LR_REQUIRE(prefix > 0 && prefix < (1 << 30), "attention_shared: prefix of %lld keys", (long long)prefix);
  return LR_OK;
}

extern "C" int64_t lr_attention_shared_workspace_bytes(int64_t seqs, int64_t total_q, int64_t total_k, int64_t prefix,
                                                       int64_t heads, int64_t kv_heads, int64_t head_dim) {
  if (check_shared(seqs, total_q, total_k, prefix, heads, kv_heads, head_dim) || total_q == 0) return 0;
  return lr::packed::shared_plan(seqs, total_q, total_k, prefix, heads / kv_heads, kv_heads, head_dim).bytes;
}

extern "C" int lr_attention_shared(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                   int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                   int64_t v_head_stride, const void* prefix_k, int64_t pk_token_stride, int64_t pk_head_stride,
                                   const void* prefix_v, int64_t pv_token_stride, int64_t pv_head_stride, const int32_t* cu_q,
                                   const int32_t* cu_k, int64_t seqs, int64_t total_q, int64_t total_k, int64_t prefix,
                                   int64_t heads, int64_t kv_heads, int64_t head_dim, int causal, float scale, void* out,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lr;
  const int st = check_shared(seqs, total_q, total_k, prefix, heads, kv_heads, head_dim);
  if (st) return st;
  if (total_q == 0) return LR_OK;
  LR_REQUIRE(q && out && cu_q && cu_k && prefix_k && prefix_v && (total_k == 0 || (k && v)), "attention_shared: null pointer");
  const int64_t strides[] = {q_token_stride,  q_head_stride,   k_token_stride,  k_head_stride,   v_token_stride,
                             v_head_stride,   pk_token_stride, pk_head_stride,  pv_token_stride, pv_head_stride};
  for (const int64_t s : strides) {
    LR_REQUIRE(s >= 0, "attention_shared: negative strides");
    if (s % 8) return set_error(LR_ERR_UNSUPPORTED, "attention_shared: strides must be multiples of 16 bytes");
  }
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(prefix_k, 16) || !aligned(prefix_v, 16) ||
      !aligned(out, 16))
    return set_error(LR_ERR_UNSUPPORTED, "attention_shared: pointers must be 16-byte aligned");
  const int64_t group = heads / kv_heads;
  const packed::SharedPlan p = packed::shared_plan(seqs, total_q, total_k, prefix, group, kv_heads, head_dim);
  LR_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && aligned(workspace, 32)),
             "attention_shared: a workspace of %lld bytes is needed", (long long)p.bytes);
  const packed::Args a{static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(k),
                       static_cast<const __nv_bfloat16*>(v), static_cast<__nv_bfloat16*>(out), q_token_stride,
                       q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride, cu_q, cu_k,
                       (int)seqs, (int)total_q, (int)total_k, (int)heads, (int)kv_heads, (int)group, causal,
                       (float)((double)scale * 1.4426950408889634)};
  packed::StepPrefix sp{};
  sp.k = static_cast<const __nv_bfloat16*>(prefix_k), sp.v = static_cast<const __nv_bfloat16*>(prefix_v);
  sp.k_ts = pk_token_stride, sp.k_hs = pk_head_stride, sp.v_ts = pv_token_stride, sp.v_hs = pv_head_stride;
  sp.keys = (int)prefix;
  auto* s = static_cast<cudaStream_t>(stream);
  return head_dim == 64 ? packed::launch_shared<64>(a, p, sp, workspace, s) : packed::launch_shared<128>(a, p, sp, workspace, s);
}
