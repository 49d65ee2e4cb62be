// Low-rank adapters of many requests beside a shared projection:
//   out[t, :] = base[t, :] + scale[e] * up[e] (down[e] x[t, :]),  e = index[t]
// (e < 0: out[t, :] = base[t, :]), where base is the shared projection's output.
//
// The first product makes the few inner values scale[e] down[e] x[t] of every
// token, the second adds up[e] times them to the base row. Both are bound by
// memory: per byte of x or base a rank of 16 to 128 gives the tensor core 8 to 64
// products, so mma.sync is fast enough (tcgen05 where many tokens stream through
// shared memory anyway), and its operands come straight from global memory, 16
// bytes a load: a sum over columns does not mind their order, and neither do the
// outputs of a tile, so what a thread loads at once are the columns that it stands
// for.
//
// Up to kFew tokens, where one token a request is usual, a block stands for one
// adapter and lists its tokens first: few_kernel, both products. Whatever the
// tokens' order an adapter in use is read once for every 16 of them, from memory
// once. The grid counts the adapters that are there: few in use out of many, or most
// tokens with one of them, leave the other blocks idle and that one's 16 tokens
// after one another. More tokens are taken in tiles of neighbours, by shrink_kernel and
// an expand kernel: for each adapter that occurs in a tile the rows of the others are
// neither used nor changed. Either way an infinity in one request's row or adapter
// reaches no other.
#include "lr_common.cuh"
#include "lr_host.h"
#include "lr_tc.cuh"

namespace lr {

static __device__ unsigned int g_adapters_status = 0;

namespace adapters {
namespace {

using bf16 = __nv_bfloat16;

struct Args {
  const bf16 *x, *base, *down, *up;
  const float* scale;
  const int32_t* index;
  bf16 *out, *inner;  // inner: [tokens][padded]
  int64_t x_stride, base_stride, out_stride;
  int tokens, width, outputs, rank, count;
  int padded;  // columns of an inner row
  int groups;  // up to kFew tokens: blocks that stand for adapters
};

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kFew = 2 * kThreads;

__device__ __forceinline__ bool adapter_of(const Args& a, int id) { return id >= 0 && id < a.count; }

// The tokens of one block's adapter, in order (up to kFew tokens). With no more
// adapters than tokens group z is adapter z, else the one of token z if that is
// its first token. Group a.groups is the tokens without one. Whole block; the
// count, and the adapter (-1: none).
struct List {
  uint16_t token[kFew];
  int counts[kFew / 32];
};
__device__ __forceinline__ int list_tokens(const Args& a, List& list, int group, int& adapter) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  adapter = group == a.groups ? -1 : a.count <= a.tokens ? group : a.index[group];
  if (group < a.groups && !adapter_of(a, adapter)) return 0;
  unsigned mine[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = i * kThreads + threadIdx.x;
    const int id = at < a.tokens ? a.index[at] : -1;
    const bool there = adapter_of(a, id);
    if (group == a.groups && id >= a.count) atomicOr(&g_adapters_status, (unsigned)kDevErrAdapter);
    mine[i] = __ballot_sync(0xffffffffu, at < a.tokens && (adapter < 0 ? !there : id == adapter));
    if (lane == 0) list.counts[i * kWarps + warp] = __popc(mine[i]);
  }
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int before = total;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int n = list.counts[i * kWarps + w];
      before += w < warp ? n : 0;
      total += n;
    }
    if (mine[i] >> lane & 1) list.token[before + __popc(mine[i] & ((1u << lane) - 1))] = (uint16_t)(i * kThreads + threadIdx.x);
  }
  __syncthreads();
  if (group < a.groups && a.count > a.tokens && list.token[0] != group) total = 0;
  return total;
}

// The adapters of a tile of 32 W neighbours, one after another, in every warp alike.
template <int W>
struct Groups {
  int id[W];  // of tokens lane + 32 i; -1: none, or had already

  __device__ __forceinline__ void load(const Args& a, int first, int lane) {
#pragma unroll
    for (int i = 0; i < W; ++i) id[i] = first + lane + 32 * i < a.tokens ? a.index[first + lane + 32 * i] : -1;
  }
  // Numbers past the last adapter become none.
  __device__ __forceinline__ void check(const Args& a) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (id[i] >= a.count) {
        atomicOr(&g_adapters_status, (unsigned)kDevErrAdapter);
        id[i] = -1;
      }
  }
  // The next adapter and the tokens that have it; false at the end.
  __device__ __forceinline__ bool next(int& adapter, uint32_t (&members)[W]) {
    bool any = false;
#pragma unroll
    for (int i = W - 1; i >= 0; --i) {
      const unsigned left = __ballot_sync(0xffffffffu, id[i] >= 0);
      if (left) {
        any = true;
        adapter = __shfl_sync(0xffffffffu, id[i], __ffs(left) - 1);
      }
    }
    if (!any) return false;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      members[i] = __ballot_sync(0xffffffffu, id[i] == adapter);
      if (id[i] == adapter) id[i] = -1;
    }
    return true;
  }
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load16(const bf16* p, bool there) {
  return there ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ float cluster_load(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(tc::map_to_rank(tc::smem_u32(p), rank)) : "memory");
  return v;
}

// ------------------------------------------------------------------ shrink
// Many tokens: 128 neighbours against an adapter's N rank rows (padded with zeros)
// on the tensor core, 64 columns of both a stage. The cluster's blocks take every
// gridDim.x-th 64 columns and add their sums in order through shared memory. Up to
// kTogether adapters that occur among the tokens are taken in one pass over the
// rows, each in columns of its own of tensor memory. Bound by memory where tokens
// are many (12240 of 6144 columns, rank 32: 31 us, 0.73 of the measured copy rate;
// with mma.sync and operands straight from global memory 47), else by its chain of
// latencies (2500 tokens: 17 us, an adapter at a time 34).
constexpr int kShrinkRows = 128;
template <int N>
struct Shrink {
  static constexpr int kTogether = N <= 32 ? 4 : N == 64 ? 2 : 1;
  static constexpr int kX = kShrinkRows * 128, kStage = kX + kTogether * N * 128;
  static constexpr int kStages = N == 16 ? 4 : 6;
  static constexpr int kBlocks = N == 16 ? 2 : 1;  // an SM
  static constexpr int kBars = kStages * kStage;  // full, empty, done; TMEM address, abort flag
  static_assert(kBars >= N * kShrinkRows * 4, "the sums fit the ring");
  static constexpr size_t kSmem = 1024 + kBars + (2 * kStages + 1) * 8 + 8;
  static constexpr uint32_t kColumns = kTogether * N;
  // kind::f16: fp32 accumulator, bf16 operands, N / 8 at 17, M / 16 at 24
  static constexpr uint32_t kDesc =
      (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N / 8) << 17) | ((uint32_t)(kShrinkRows / 16) << 24);
};
constexpr int kShrinkThreads = 192;

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"(accumulate)
      : "memory");
}

// Warp 0 copies, warp 1 issues the products, warps 2-5 take the sums.
template <int N>
__global__ void __launch_bounds__(kShrinkThreads)
    shrink_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_down, const Args a) {
  using C = Shrink<N>;
  using namespace tc;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* sums = reinterpret_cast<float*>(smem);  // [N][kShrinkRows], where the ring is between passes
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t *empty = full + C::kStages, *done = empty + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  const Watch watch{tmem_slot + 1, &g_adapters_status};
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int part = blockIdx.x, parts = gridDim.x, first = blockIdx.y * kShrinkRows;
  allow_dependent();
  if (threadIdx.x == 0) {
    prefetch_map(&map_x);
    prefetch_map(&map_down);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(done), 1);
    *watch.abort_flag = 0u;
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc<1>(smem_u32(tmem_slot), C::kColumns);
  Groups<4> groups;
  groups.load(a, first, lane);
  groups.check(a);
  const int row = ((warp & 3) * 32) + lane;  // of the sums' warps
  const int mine = warp >= 2 && first + row < a.tokens ? a.index[first + row] : -1;
  __shared__ float scales[kShrinkRows];
  __shared__ int8_t slots[kShrinkRows];  // each row's adapter among a pass's, -1: none of them
  if (warp >= 2) scales[row] = a.scale && adapter_of(a, mine) ? a.scale[mine] : 1.0f;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);

  const int steps = (a.width + 63) / 64;
  const bool el = elect_one();
  bool ok = true;
  uint32_t stage = 0;  // of the ring, over all passes
  int adapter;
  uint32_t members[4];
  bool more = groups.next(adapter, members);
  for (uint32_t pass = 0; more; ++pass) {
    int taken[C::kTogether], together = 0;  // this pass's adapters
#pragma unroll
    for (int i = 0; i < C::kTogether; ++i) {
      taken[i] = -1;
      if (!more) continue;
      taken[i] = uniform(adapter);
      ++together;
      more = groups.next(adapter, members);
    }
    int slot = -1;  // of this row's adapter among them
#pragma unroll
    for (int i = 0; i < C::kTogether; ++i)
      if (mine >= 0 && mine == taken[i]) slot = i;
    if (warp == 0) {
      for (int step = part; step < steps && ok; step += parts, ++stage) {
        const uint32_t s = stage % C::kStages;
        ok = warp_wait(smem_u32(&empty[s]), ((stage / C::kStages) & 1u) ^ 1u, watch, lane);
        if (el && ok) {
          const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(smem + s * C::kStage);
          mbar_expect_tx(bar, C::kX + together * (N * 128));
          tma_load_2d(dst, &map_x, bar, step * 64, first);
#pragma unroll
          for (int i = 0; i < C::kTogether; ++i)
            if (i < together) tma_load_3d(dst + C::kX + i * (N * 128), &map_down, bar, step * 64, 0, taken[i]);
        }
        __syncwarp();
      }
    } else if (warp == 1) {
      for (int step = part; step < steps && ok; step += parts, ++stage) {
        const uint32_t s = stage % C::kStages;
        ok = warp_wait(smem_u32(&full[s]), (stage / C::kStages) & 1u, watch, lane);
        tc_fence_after();
        if (el && ok) {
          const uint32_t x = smem_u32(smem + s * C::kStage), w = x + C::kX;
#pragma unroll
          for (int i = 0; i < C::kTogether; ++i) {
            if (i >= together) break;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(tmem + i * N, desc_kmajor(x + kk * 32), desc_kmajor(w + i * (N * 128) + kk * 32), C::kDesc,
                     step != part || kk != 0 ? 1u : 0u);
          }
          mma_commit(smem_u32(&empty[s]));
        }
        __syncwarp();
      }
      if (el) mma_commit(smem_u32(done));
      __syncwarp();
    } else {
      ok = ok && warp_wait(smem_u32(done), pass & 1u, watch, lane);
      tc_fence_after();
      slots[row] = (int8_t)slot;
      const float scale = scales[row];
      const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      bf16* dst = a.inner + (int64_t)(first + row) * a.padded;
      for (int i = 0; i < together; ++i) {
#pragma unroll
        for (int c = 0; c < N; c += 16) {
          uint32_t v[16];
          tmem_ld16(lanes + i * N + c, v);
          if (slot != i || !ok) continue;
          if (parts > 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[(c + j) * kShrinkRows + row] = __uint_as_float(v[j]);
          } else {
            uint32_t y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = cvt2(__uint_as_float(v[2 * j]) * scale, __uint_as_float(v[2 * j + 1]) * scale);
            *reinterpret_cast<uint4*>(dst + c) = make_uint4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(y[4], y[5], y[6], y[7]);
          }
        }
      }
      tc_fence_before();
    }
    if (parts > 1) {
      __syncwarp();
      cluster_sync_all();
      // this block's share of the sums, two columns of a row at a time
      const int share = kShrinkRows * N / 2 / parts;
#pragma unroll 4
      for (int i = part * share + (int)threadIdx.x; i < (part + 1) * share; i += kShrinkThreads) {
        const int r = i % kShrinkRows, c = i / kShrinkRows * 2;
        if (slots[r] < 0) continue;
        const float* from = sums + c * kShrinkRows + r;
        float v0 = 0.0f, v1 = 0.0f;
        for (int p = 0; p < parts; ++p) {
          v0 += cluster_load(from, p);
          v1 += cluster_load(from + kShrinkRows, p);
        }
        *reinterpret_cast<uint32_t*>(a.inner + (int64_t)(first + r) * a.padded + c) = cvt2(v0 * scales[r], v1 * scales[r]);
      }
      fence_async_smem();  // the next pass's copies write where the sums were
      __syncwarp();
      cluster_sync_all();
    } else {
      __syncwarp();
      __syncthreads();
    }
    tc_fence_after();
  }
  if (!ok) {  // giving up: time for the copies in flight to land before the block can exit
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 100000ull) {
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, C::kColumns);
  }
}

// ------------------------------------------------------------------ expand
// 32 columns a warp, rank up to 16 KS. The base values are the products'
// accumulators: sums stay in fp32 and are rounded once. A thread's eight columns
// lie side by side: column n of the i-th product stands for column
// 8 (n / 2) + 2 i + n % 2 of the 32.
template <int KS>
struct Up {
  uint32_t w[4][KS][2];
  // From `weight`, the adapter's. Columns past the last are the last one's again: they are not stored.
  __device__ __forceinline__ void load(const bf16* weight, int column, int outputs, int rank, int g, int t) {
    const int n = column + 8 * (g >> 1) + (g & 1), last = outputs - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16* src = weight + (int64_t)min(n + 2 * i, last) * rank;
      if constexpr (KS == 1) {
        const uint2 v = 4 * t < rank ? *reinterpret_cast<const uint2*>(src + 4 * t) : make_uint2(0u, 0u);
        w[i][0][0] = v.x, w[i][0][1] = v.y;
      } else {
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
          const uint4 v = load16(src + 16 * s + 8 * t, 16 * s + 8 * t < rank);
          w[i][s][0] = v.x, w[i][s][1] = v.y;
          w[i][s + 1][0] = v.z, w[i][s + 1][1] = v.w;
        }
      }
    }
  }
};
__device__ __forceinline__ const bf16* up_of(const Args& a, int adapter) { return a.up + (int64_t)adapter * a.outputs * a.rank; }
// The inner values of rows g and g + 8 of 16 that a thread multiplies, zeros past the rank: what the first product leaves there,
// x times zeros, is not zero where x or the scale is infinite.
template <int KS>
struct Inner {
  uint32_t lo[2 * KS], hi[2 * KS];
  // From rows r0 and r1 (zeros where they are not to be read).
  __device__ __forceinline__ void load(const bf16* r0, bool there0, const bf16* r1, bool there1, int t, int rank) {
    if constexpr (KS == 1) {
      there0 &= 4 * t < rank, there1 &= 4 * t < rank;
      const uint2 h0 = there0 ? *reinterpret_cast<const uint2*>(r0 + 4 * t) : make_uint2(0u, 0u);
      const uint2 h1 = there1 ? *reinterpret_cast<const uint2*>(r1 + 4 * t) : make_uint2(0u, 0u);
      lo[0] = h0.x, lo[1] = h0.y, hi[0] = h1.x, hi[1] = h1.y;
    } else {
#pragma unroll
      for (int s = 0; s < KS; s += 2) {
        const bool inside = 16 * s + 8 * t < rank;
        const uint4 h0 = load16(r0 + 16 * s + 8 * t, there0 && inside), h1 = load16(r1 + 16 * s + 8 * t, there1 && inside);
        lo[2 * s] = h0.x, lo[2 * s + 1] = h0.y, lo[2 * s + 2] = h0.z, lo[2 * s + 3] = h0.w;
        hi[2 * s] = h1.x, hi[2 * s + 1] = h1.y, hi[2 * s + 2] = h1.z, hi[2 * s + 3] = h1.w;
      }
    }
  }
};
// acc += inner values times the weights; rows that are not `lo`, `hi` count as zeros.
template <int KS>
__device__ __forceinline__ void add_update(float (&acc)[4][4], const Up<KS>& up, const Inner<KS>& h, bool lo, bool hi) {
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const uint32_t a0 = lo ? h.lo[2 * s] : 0u, a1 = hi ? h.hi[2 * s] : 0u;
    const uint32_t a2 = lo ? h.lo[2 * s + 1] : 0u, a3 = hi ? h.hi[2 * s + 1] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) mma_16816(acc[i], a0, a1, a2, a3, up.w[i][s][0], up.w[i][s][1]);
  }
}
// Eight neighbouring columns of a row, as far as there are any.
template <bool VEC>
__device__ __forceinline__ uint4 load_row(const bf16* p, int columns, bool there) {
  if (VEC) return load16(p, there && columns > 0);
  uint32_t y[4] = {0u, 0u, 0u, 0u};
  if (there) {
    const uint16_t* s = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < columns) y[i / 2] |= (uint32_t)s[i] << (16 * (i % 2));
  }
  return make_uint4(y[0], y[1], y[2], y[3]);
}
template <bool VEC>
__device__ __forceinline__ void store_row(bf16* p, const float (&acc)[4][4], int h, int columns) {
  if (VEC) {
    if (columns > 0)
      *reinterpret_cast<uint4*>(p) = make_uint4(cvt2(acc[0][2 * h], acc[0][2 * h + 1]), cvt2(acc[1][2 * h], acc[1][2 * h + 1]),
                                                cvt2(acc[2][2 * h], acc[2][2 * h + 1]), cvt2(acc[3][2 * h], acc[3][2 * h + 1]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < columns) p[i] = __float2bfloat16_rn(acc[i / 2][2 * h + i % 2]);
  }
}
__device__ __forceinline__ void unpack_row(float (&acc)[4][4], int h, const uint4& y) {
  const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc[i][2 * h] = bf_lo(w[i]);
    acc[i][2 * h + 1] = bf_hi(w[i]);
  }
}

// ------------------------------------------------------------------ few tokens
// Both products in one kernel: clusters stand for one adapter and their blocks for
// every gridDim.x-th 256 columns. A cluster's blocks share the first product, every
// warp 32 columns of x at a time, add their sums in a fixed order through shared
// memory and have the inner rows in it at once. (With a launch of its own for the
// inner rows 64 tokens of 64 adapters, 4096 to 12288 at rank 16, took 14.4 us and 18.4
// us with the host, now 15.4 and 17.0; one token 18.4 us with the host, now 12.6.)
// Weights and base rows of the second product load meanwhile, and then AHEAD strips
// ahead: one where a block has one strip (one token 6144 to 18432: 6.0 us with four),
// else kAhead. An adapter's second cluster reads `down` again, from L2; grids are
// one wave. Bound by latency: list, first product, cluster and second product follow
// one another.
template <int KS>
struct Few {
  static constexpr int kTile = 16 * 16 * KS;                      // inner values of 16 tokens
  static constexpr int kSteps = KS == 1 ? 4 : KS == 2 ? 2 : 1;    // of the first product whose loads are under way together
  static constexpr int kAhead = KS == 1 ? 4 : KS == 2 ? 2 : KS == 4 ? 3 : 1;
  static constexpr int kLine = KS >= 4 ? 16 * KS + 32 : 16 * KS;  // inner rows side by side in different banks
  static constexpr int kBlocks = KS <= 2 ? 2 : 1;                 // an SM
  static constexpr size_t kSmem = (kWarps + 1) * kTile * 4 + 16 * kLine * 2;
};

template <int KS, int AHEAD, bool VEC>
__global__ void __launch_bounds__(kThreads, Few<KS>::kBlocks) few_kernel(const Args a) {
  using C = Few<KS>;
  constexpr int NR = 2 * KS;
  extern __shared__ float sums[];  // [kWarps][kTile], the block's [kTile], then the inner rows
  __shared__ List list;
  float* block_sums = sums + kWarps * C::kTile;
  bf16* inner_rows = reinterpret_cast<bf16*>(block_sums + C::kTile);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int parts = tc::cluster_size(), part = parts > 1 ? (int)tc::cluster_rank() : 0;
  const int stride = gridDim.x * kThreads;
  const int start = blockIdx.x * kThreads + warp * 32;
  int adapter;
  const int count = list_tokens(a, list, blockIdx.y, adapter);
  // the same in all blocks of the cluster
  if ((int)blockIdx.z * 16 >= count || (adapter < 0 && a.out == a.base && a.out_stride == a.base_stride)) return;
  for (int first = blockIdx.z * 16; first < count; first += gridDim.z * 16) {
    const bool lo = first + g < count, hi = first + 8 + g < count;
    const int64_t t0 = list.token[lo ? first + g : first], t1 = list.token[hi ? first + 8 + g : first];
    // strips of columns under way, a ring
    Up<KS> up[AHEAD];
    uint4 base[AHEAD][2];
    const bf16 *weight = up_of(a, max(adapter, 0)), *b0 = a.base + t0 * a.base_stride, *b1 = a.base + t1 * a.base_stride;
    bf16 *o0 = a.out + t0 * a.out_stride, *o1 = a.out + t1 * a.out_stride;
    const auto load_strip = [&](int s, int column) {
      if (column >= a.outputs) return;
      const int mine = column + 8 * t;
      base[s][0] = load_row<VEC>(b0 + mine, a.outputs - mine, lo);
      base[s][1] = load_row<VEC>(b1 + mine, a.outputs - mine, hi);
      if (adapter >= 0) up[s].load(weight, column, a.outputs, a.rank, g, t);
    };
    if (KS <= 4) {  // else the registers are not there yet
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) load_strip(s, start + s * stride);
    }
    if (adapter >= 0) {
      float acc[NR][4];
#pragma unroll
      for (int i = 0; i < NR * 4; ++i) acc[i / 4][i % 4] = 0.0f;
      const bf16* down = a.down + ((int64_t)adapter * a.rank + g) * a.width;
      const bf16 *x0 = a.x + t0 * a.x_stride, *x1 = a.x + t1 * a.x_stride;
#pragma unroll C::kSteps
      for (int k0 = (part * kWarps + warp) * 32; k0 < a.width; k0 += parts * kWarps * 32) {
        const int k = k0 + 8 * t;
        const bool there = k < a.width;
        uint4 w[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) w[n] = load16(down + (int64_t)(8 * n) * a.width + k, there && 8 * n + g < a.rank);
        const uint4 v0 = load16(x0 + k, there && lo), v1 = load16(x1 + k, there && hi);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          mma_16816(acc[n], v0.x, v1.x, v0.y, v1.y, w[n].x, w[n].y);
          mma_16816(acc[n], v0.z, v1.z, v0.w, v1.w, w[n].z, w[n].w);
        }
      }
      // [register][lane] of each warp: no two lanes in one bank
#pragma unroll
      for (int i = 0; i < NR * 4; ++i) sums[warp * C::kTile + i * 32 + lane] = acc[i / 4][i % 4];
      __syncthreads();
      for (int i = threadIdx.x; i < C::kTile; i += kThreads) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += sums[w * C::kTile + i];
        block_sums[i] = v;
      }
      if (parts > 1) tc::cluster_sync_all(); else __syncthreads();
      const float scale = a.scale ? a.scale[adapter] : 1.0f;
      for (int i = threadIdx.x; i < C::kTile / 2; i += kThreads) {
        // two columns side by side: registers 2 e, 2 e + 1 of a lane
        const int l = i % 32, e = i / 32 % 2, n = i / 64;
        const int at = (n * 4 + 2 * e) * 32 + l;
        float h0 = 0.0f, h1 = 0.0f;
        if (parts > 1) {
#pragma unroll 8
          for (int p = 0; p < parts; ++p) {
            h0 += cluster_load(block_sums + at, p);
            h1 += cluster_load(block_sums + at + 32, p);
          }
        } else {
          h0 = block_sums[at], h1 = block_sums[at + 32];
        }
        // zeros past the rank, once for all columns (where they are read, as the expand kernels do it: 16.0 us for 64 tokens of
        // 64 adapters, here 15.5)
        *reinterpret_cast<uint32_t*>(inner_rows + (8 * e + l / 4) * C::kLine + 8 * n + 2 * (l % 4)) =
            8 * n < a.rank ? cvt2(h0 * scale, h1 * scale) : 0u;
      }
      __syncthreads();
      if (parts > 1) tc::cluster_arrive();  // done with the other blocks' sums
    }
    Inner<KS> inner;
    if (adapter >= 0) inner.load(inner_rows + g * C::kLine, lo, inner_rows + (8 + g) * C::kLine, hi, t, 16 * KS);
    if (KS > 4) load_strip(0, start);
    for (int next = start; next < a.outputs;) {
#pragma unroll
      for (int s = 0; s < AHEAD; ++s, next += stride) {
        if (next >= a.outputs) break;
        const int mine = next + 8 * t;
        float acc[4][4];
        unpack_row(acc, 0, base[s][0]);
        unpack_row(acc, 1, base[s][1]);
        if (adapter >= 0) add_update<KS>(acc, up[s], inner, true, true);
        load_strip(s, next + AHEAD * stride);
        if (lo) store_row<VEC>(o0 + mine, acc, 0, a.outputs - mine);
        if (hi) store_row<VEC>(o1 + mine, acc, 1, a.outputs - mine);
      }
    }
    if (adapter >= 0) {
      __syncthreads();  // the inner rows have been read
      if (parts > 1) tc::cluster_wait();
    }
  }
}

// Many tokens: tiles of 64 neighbours by 32 columns a warp. A warp has a ring of
// tiles of its own in shared memory, which bulk copies fill and empty: nothing but
// bytes in flight, and whole rows, make this kernel fast. 12240 tokens to 24576 at
// rank 32, both products: 223 us, 0.93 of the measured copy rate (this kernel 0.97);
// base rows through registers, the next tile's on their way, 457 us; through the
// rings, but runs of tiles down the columns, 272 us. Blocks therefore take the tiles
// of a row of tiles in turn; where the grid is a multiple of their number a warp
// keeps its columns, and its weights while the adapter stays the same. Rows in
// shared memory are 64 bytes long: two of them fill the banks.
constexpr int kExpandRows = 64;
constexpr int kSlotBytes = kExpandRows * 64;
template <int KS>
struct Expand {
  static constexpr int kBlocks = KS <= 4 ? 2 : 1;  // an SM: at rank 128 the weights alone are 64 registers
  static constexpr int kSlots = KS <= 4 ? 3 : 6;
  static constexpr int kHeld = KS <= 2 ? 4 : 2;  // 16-row tiles whose inner values are loaded together
  static constexpr size_t kSmem = 128 + kWarps * kSlots * (kSlotBytes + 8) + 8;
};

// One row's eight columns in a tile.
__device__ __forceinline__ uint4* tile_at(uint8_t* tile, int row, int t) { return reinterpret_cast<uint4*>(tile + row * 64 + t * 16); }

template <int KS>
__global__ void __launch_bounds__(kThreads, Expand<KS>::kBlocks)
    expand_kernel(const __grid_constant__ CUtensorMap map_base, const __grid_constant__ CUtensorMap map_out, const Args a) {
  using namespace tc;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  constexpr int kSlots = Expand<KS>::kSlots, kHeld = Expand<KS>::kHeld;
  uint8_t* ring = smem + warp * (kSlots * kSlotBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kWarps * kSlots * kSlotBytes) + warp * kSlots;
  uint32_t* abort_flag = reinterpret_cast<uint32_t*>(smem + kWarps * kSlots * (kSlotBytes + 8));
  const Watch watch{abort_flag, &g_adapters_status};
  if (lane == 0) {
    for (int s = 0; s < kSlots; ++s) mbar_init(smem_u32(&full[s]), 1);
    if (warp == 0) {
      *abort_flag = 0u;
      prefetch_map(&map_base);
      prefetch_map(&map_out);
    }
    mbar_init_fence();
  }
  __syncthreads();
  const bool el = elect_one();
  // Items go along the rows and are dealt out in turn, so that the blocks together work on whole rows.
  const int blocks = (a.outputs + kThreads - 1) / kThreads;
  const int64_t items = (int64_t)((a.tokens + kExpandRows - 1) / kExpandRows) * blocks;
  const int count = (int)((items - blockIdx.x + gridDim.x - 1) / gridDim.x);
  const int step_tile = gridDim.x / blocks, step_block = gridDim.x % blocks;
  const auto advance = [&](int& tile, int& block) {
    tile += step_tile;
    block += step_block;
    if (block >= blocks) block -= blocks, ++tile;
  };
  // the next tile to be fetched, and the one in hand
  int fetch_tile = blockIdx.x / blocks, fetch_block = blockIdx.x % blocks, fetched = 0;
  int tile = fetch_tile, block = fetch_block;
  const auto fetch = [&] {
    const int fetch_column = fetch_block * kThreads + warp * 32;
    if (fetched < count && el) {
      const uint32_t s = (uint32_t)fetched % kSlots, bar = smem_u32(&full[s]);
      if (fetch_column < a.outputs) {
        mbar_expect_tx(bar, kSlotBytes);
        tma_load_2d(smem_u32(ring + s * kSlotBytes), &map_base, bar, fetch_column, fetch_tile * kExpandRows);
      } else {
        mbar_arrive(bar);  // nothing to come
      }
    }
    ++fetched;
    advance(fetch_tile, fetch_block);
  };
  for (int s = 0; s < kSlots; ++s) fetch();
  bool ok = true;
  const auto wait_for = [&](int i) {
    const bool landed = warp_wait(smem_u32(&full[i % kSlots]), (uint32_t)(i / kSlots) & 1u, watch, lane);
    __syncwarp();
    return landed;
  };
  Groups<2> groups;
  groups.load(a, tile * kExpandRows, lane);
  wait_for_predecessor();
  Up<KS> up;
  int kept = -1, kept_column = -1;  // whose weights `up` holds
  for (int i = 0; i < count; ++i) {
    const int first = tile * kExpandRows, this_column = block * kThreads + warp * 32;
    Groups<2> now = groups;
    now.check(a);
    advance(tile, block);
    if (i + 1 < count) groups.load(a, tile * kExpandRows, lane);
    uint8_t* rows = ring + i % kSlots * kSlotBytes;
    if (this_column < a.outputs) {  // the last columns' warps may have none
      // Inner values do not depend on whose they are; they load before the base rows are there.
      Inner<KS> inner[kHeld];
      const auto load_inner = [&](int from) {
#pragma unroll
        for (int m = 0; m < kHeld; ++m) {
          const int token = first + 16 * (from + m) + g;
          const bf16* r = a.inner + (int64_t)token * a.padded;
          inner[m].load(r, token < a.tokens, r + 8 * a.padded, token + 8 < a.tokens, t, a.rank);
        }
      };
      load_inner(0);
      int adapter;
      uint32_t members[2];
      bool all = this_column == kept_column && __all_sync(0xffffffffu, now.id[0] == kept && now.id[1] == kept);
      bool any = all || now.next(adapter, members);
      if (all) members[0] = members[1] = 0xffffffffu, adapter = kept;
      bool held = true;  // the first kHeld tiles' inner values
      if (!(ok = wait_for(i))) break;
      while (any) {
        if (adapter != kept || this_column != kept_column) {
          kept = adapter, kept_column = this_column;
          up.load(up_of(a, adapter), this_column, a.outputs, a.rank, g, t);
        }
#pragma unroll
        for (int from = 0; from < kExpandRows / 16; from += kHeld) {
          if (kHeld < kExpandRows / 16 && !(from == 0 && held)) load_inner(from);
#pragma unroll
          for (int m = from; m < from + kHeld; ++m) {
            const uint32_t here = members[m / 2] >> (16 * (m % 2)) & 0xffffu;
            if (here == 0u) continue;
            // rows of other adapters are neither changed nor used
            const bool lo = here >> g & 1, hi = here >> (8 + g) & 1;
            uint4 *r0 = tile_at(rows, 16 * m + g, t), *r1 = tile_at(rows, 16 * m + 8 + g, t);
            float acc[4][4];
            unpack_row(acc, 0, *r0);
            unpack_row(acc, 1, *r1);
            add_update<KS>(acc, up, inner[m - from], lo, hi);
            if (lo) *r0 = make_uint4(cvt2(acc[0][0], acc[0][1]), cvt2(acc[1][0], acc[1][1]), cvt2(acc[2][0], acc[2][1]), cvt2(acc[3][0], acc[3][1]));
            if (hi) *r1 = make_uint4(cvt2(acc[0][2], acc[0][3]), cvt2(acc[1][2], acc[1][3]), cvt2(acc[2][2], acc[2][3]), cvt2(acc[3][2], acc[3][3]));
          }
        }
        held = false;
        any = !all && now.next(adapter, members);
      }
      fence_async_smem();
      __syncwarp();
      if (el) tma_store_2d(&map_out, smem_u32(rows), this_column, first);
    } else if (!(ok = wait_for(i))) {
      break;
    }
    if (el) bulk_commit();
    // The tile before this one has been stored: its slot takes the next.
    if (i > 0) {
      if (el) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      fetch();
    }
    __syncwarp();
  }
  if (el) bulk_wait_all();
  if (!ok) {  // giving up: time for the copies in flight to land before the block can exit
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 100000ull) {
    }
  }
}

// The same for rows that bulk copies cannot address (an odd number of columns, other strides): 32 tokens at a time.
template <int KS>
__global__ void __launch_bounds__(kThreads) expand_odd_kernel(const Args a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int blocks = (a.outputs + kThreads - 1) / kThreads;
  const int first = (int)(blockIdx.x / blocks) * 32, column = (int)(blockIdx.x % blocks) * kThreads + warp * 32;
  const int mine = column + 8 * t;
  Groups<1> groups;
  groups.load(a, first, lane);
  groups.check(a);
  float acc[2][4][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int token = first + 16 * m + 8 * h + g;
      unpack_row(acc[m], h, load_row<false>(a.base + (int64_t)token * a.base_stride + mine, a.outputs - mine, token < a.tokens));
    }
  int adapter;
  uint32_t members[1];
  bool waited = false;
  while (groups.next(adapter, members)) {
    Up<KS> up;
    up.load(up_of(a, adapter), column, a.outputs, a.rank, g, t);
    if (!waited) tc::wait_for_predecessor();
    waited = true;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const bool lo = members[0] >> (16 * m + g) & 1, hi = members[0] >> (16 * m + 8 + g) & 1;
      const bf16* r = a.inner + (int64_t)(first + 16 * m + g) * a.padded;
      float sum[4][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[i / 4][i % 4] = acc[m][i / 4][i % 4];
      Inner<KS> inner;
      inner.load(r, lo, r + 8 * a.padded, hi, t, a.rank);
      add_update<KS>(sum, up, inner, true, true);
#pragma unroll
      for (int i = 0; i < 16; ++i)  // rows of other adapters stay as they were
        if (i % 4 < 2 ? lo : hi) acc[m][i / 4][i % 4] = sum[i / 4][i % 4];
    }
  }
  if (!waited) tc::wait_for_predecessor();
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int token = first + 16 * m + 8 * h + g;
      if (token < a.tokens) store_row<false>(a.out + (int64_t)token * a.out_stride + mine, acc[m], h, a.outputs - mine);
    }
}

// ------------------------------------------------------------------ host
int padded_rank(int64_t rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// Blocks of a cluster that share the columns of `tiles` tiles: as many as give the GPU `blocks`, each at least `columns` wide.
int column_parts(const Args& a, int64_t tiles, int64_t blocks, int columns) {
  int parts = 1;
  while (parts < 8 && 2 * tiles * parts <= blocks && (int64_t)parts * columns < a.width) parts *= 2;
  return parts;
}

// Tokens by their adapters, in one kernel? Neighbours are tiled where an adapter has 64 of them or more on average.
bool few(int64_t tokens, int64_t adapters) { return tokens <= kFew && tokens < 64 * adapters; }
int64_t workspace_bytes(int64_t tokens, int64_t adapters, int64_t rank) {
  return few(tokens, adapters) ? 0 : tokens * padded_rank(rank) * 2;
}

template <int KS>
int launch_few(const Args& a, bool vec, cudaStream_t stream) {
  const int tiles = (a.tokens + 15) / 16, chunks = (tiles + a.groups - 1) / a.groups;
  int blocks = Few<KS>::kBlocks * sm_count() / (a.groups * chunks);  // for one adapter's tile
  if (blocks > (a.outputs + kThreads - 1) / kThreads) blocks = (a.outputs + kThreads - 1) / kThreads;
  int parts = 1;
  while (parts < 8 && 2 * parts <= blocks && (int64_t)parts * kWarps * 32 < a.width) parts *= 2;
  blocks = blocks < 1 ? 1 : blocks / parts * parts;
  const bool one = (int64_t)blocks * kThreads >= a.outputs;
  const auto kernel = one ? (vec ? few_kernel<KS, 1, true> : few_kernel<KS, 1, false>)
                          : (vec ? few_kernel<KS, Few<KS>::kAhead, true> : few_kernel<KS, Few<KS>::kAhead, false>);
  static bool done[2][2][64] = {};
  const int st = tc::configure_smem(kernel, Few<KS>::kSmem, done[one][vec]);
  if (st) return st;
  const dim3 grid((unsigned)blocks, (unsigned)(a.groups + 1), (unsigned)chunks);
  return tc::launch("adapters (few tokens)", kernel, grid, kThreads, Few<KS>::kSmem, stream, (unsigned)parts, false, a);
}

template <int N>
int launch_shrink(const Args& a, cudaStream_t stream) {
  using C = Shrink<N>;
  static bool done[64] = {};
  int st = tc::configure_smem(shrink_kernel<N>, C::kSmem, done);
  if (st) return st;
  CUtensorMap mx, md;
  const cuuint64_t x_dims[2] = {(cuuint64_t)a.width, (cuuint64_t)a.tokens}, x_strides[1] = {(cuuint64_t)a.x_stride * 2};
  const cuuint32_t x_box[2] = {64, kShrinkRows};
  const cuuint64_t d_dims[3] = {(cuuint64_t)a.width, (cuuint64_t)a.rank, (cuuint64_t)a.count};
  const cuuint64_t d_strides[2] = {(cuuint64_t)a.width * 2, (cuuint64_t)a.width * (cuuint64_t)a.rank * 2};
  const cuuint32_t d_box[3] = {64, N, 1};
  if ((st = tc::make_map(&mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.x, x_dims, x_strides, x_box, CU_TENSOR_MAP_SWIZZLE_128B)) ||
      (st = tc::make_map(&md, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.down, d_dims, d_strides, d_box, CU_TENSOR_MAP_SWIZZLE_128B)))
    return st;
  const int64_t tiles = (a.tokens + kShrinkRows - 1) / kShrinkRows;
  LR_REQUIRE(tiles <= 65535, "adapters: too many tokens");
  const int parts = column_parts(a, tiles, C::kBlocks * sm_count(), 256);
  // The ordinary way: the expand kernels read base, the tokens' numbers and weights before they wait for this one.
  return tc::launch("adapters (inner rows)", shrink_kernel<N>, dim3((unsigned)parts, (unsigned)tiles), kShrinkThreads, C::kSmem, stream,
                    (unsigned)parts, false, mx, md, a);
}

template <int KS>
int launch_expand(const Args& a, bool vec, cudaStream_t stream) {
  const int64_t blocks = (a.outputs + kThreads - 1) / kThreads;
  if (!vec) {
    const int64_t all = (int64_t)((a.tokens + 31) / 32) * blocks;
    LR_REQUIRE(all <= INT32_MAX, "adapters: too many blocks");
    return tc::launch("adapters (outputs)", expand_odd_kernel<KS>, dim3((unsigned)all), kThreads, 0, stream, 1, true, a);
  }
  static bool done[64] = {};
  int st = tc::configure_smem(expand_kernel<KS>, Expand<KS>::kSmem, done);
  if (st) return st;
  CUtensorMap mb, mo;
  const cuuint64_t dims[2] = {(cuuint64_t)a.outputs, (cuuint64_t)a.tokens};
  const cuuint64_t base_strides[1] = {(cuuint64_t)a.base_stride * 2}, out_strides[1] = {(cuuint64_t)a.out_stride * 2};
  const cuuint32_t box[2] = {32, kExpandRows};
  if ((st = tc::make_map(&mb, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.base, dims, base_strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)) ||
      (st = tc::make_map(&mo, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.out, dims, out_strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)))
    return st;
  const int64_t items = (int64_t)((a.tokens + kExpandRows - 1) / kExpandRows) * blocks;
  int64_t grid = Expand<KS>::kBlocks * sm_count();
  const int64_t whole = grid / blocks * blocks;  // the same columns for every tile of a block
  if (whole * 8 >= grid * 7) grid = whole;
  if (grid > items) grid = items;
  return tc::launch("adapters (outputs)", expand_kernel<KS>, dim3((unsigned)grid), kThreads, Expand<KS>::kSmem,
                    stream, 1, true, mb, mo, a);
}

template <int KS>
int run(const Args& a, bool vec, cudaStream_t stream) {
  if (few(a.tokens, a.count)) return launch_few<KS>(a, vec, stream);
  const int st = launch_shrink<16 * KS>(a, stream);
  return st ? st : launch_expand<KS>(a, vec, stream);
}

}  // namespace
}  // namespace adapters

int read_status_adapters(unsigned int* bits, int clear) {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_adapters_status, sizeof(v)) != cudaSuccess) return launch_status("reading the device status");
  if (clear) {
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbol(g_adapters_status, &zero, sizeof(zero)) != cudaSuccess)
      return launch_status("clearing the device status");
  }
  *bits |= v;
  return LR_OK;
}

}  // namespace lr

static int check_adapters(int64_t tokens, int64_t width, int64_t outputs, int64_t rank, int64_t adapters) {
  using namespace lr;
  LR_REQUIRE(tokens >= 0 && width > 0 && outputs > 0 && rank > 0 && adapters > 0, "adapters: invalid shape");
  LR_REQUIRE(tokens < (1 << 30) && width < (1 << 30) && outputs < (1 << 30) && adapters < (1 << 30), "adapters: shape too large");
  if (rank % 8 || rank > 128) return set_error(LR_ERR_UNSUPPORTED, "adapters: rank %lld (a multiple of 8 up to 128)", (long long)rank);
  if (width % 8) return set_error(LR_ERR_UNSUPPORTED, "adapters: width %lld (a multiple of 8)", (long long)width);
  return LR_OK;
}

extern "C" int64_t lr_adapters_workspace_bytes(int64_t tokens, int64_t width, int64_t outputs, int64_t rank, int64_t adapters) {
  if (check_adapters(tokens, width, outputs, rank, adapters) || tokens == 0) return 0;
  return lr::adapters::workspace_bytes(tokens, adapters, rank);
}

extern "C" int lr_adapters(const void* x, int64_t x_stride, const void* base, int64_t base_stride, const void* down, const void* up,
                           const float* scale, const int32_t* index, int64_t tokens, int64_t width, int64_t outputs, int64_t rank,
                           int64_t adapters, void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lr;
  int st = check_adapters(tokens, width, outputs, rank, adapters);
  if (st) return st;
  if (tokens == 0) return LR_OK;
  LR_REQUIRE(x && base && down && up && index && out, "adapters: null pointer");
  LR_REQUIRE((x_stride >= width || tokens == 1) && x_stride >= 0 && base_stride >= 0 && out_stride >= outputs, "adapters: strides");
  if (x_stride % 8 || !aligned(x, 16) || !aligned(down, 16) || !aligned(up, 16))
    return set_error(LR_ERR_UNSUPPORTED, "adapters: x, down and up must be 16-byte aligned");
  const int64_t need = adapters::workspace_bytes(tokens, adapters, rank);
  LR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), "adapters: a workspace of %lld bytes is needed",
             (long long)need);
  const adapters::Args a{static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(base),
                         static_cast<const __nv_bfloat16*>(down), static_cast<const __nv_bfloat16*>(up), scale, index,
                         static_cast<__nv_bfloat16*>(out), static_cast<__nv_bfloat16*>(workspace), x_stride, base_stride,
                         out_stride, (int)tokens, (int)width, (int)outputs, (int)rank, (int)adapters,
                         adapters::padded_rank(rank), (int)(adapters < tokens ? adapters : tokens)};
  const bool vec = outputs % 8 == 0 && base_stride >= outputs && base_stride % 8 == 0 && out_stride % 8 == 0 && aligned(base, 16) && aligned(out, 16);
  auto* s = static_cast<cudaStream_t>(stream);
  if (rank <= 16) return adapters::run<1>(a, vec, s);
  if (rank <= 32) return adapters::run<2>(a, vec, s);
  if (rank <= 64) return adapters::run<4>(a, vec, s);
  return adapters::run<8>(a, vec, s);
}
