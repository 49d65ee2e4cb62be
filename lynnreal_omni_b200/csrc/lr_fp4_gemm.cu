// Product of two matrices of 4-bit floating-point rows:
//   out[m, n] = bf16( (sum_k A[m, k] B[n, k]) * row_scale[m] * col_scale[n] + bias[n] )
// with A, B the values of codes and block scales, accumulated in fp32.
//
// The tensor core multiplies the codes and applies the block scales itself
// (tcgen05.mma kind::mxf4nvf4, one e4m3 scale per 16 columns, or kind::mxf4,
// one e8m0 scale per 32): 64 columns of K an instruction, at four times the
// bf16 rate. Codes reach shared memory by TMA with 128-byte swizzle, 256
// columns (128 bytes) a stage. Scales lie in global memory in the order in
// which the tensor core reads them, so a stage's scales are one box of whole
// 512-byte tiles (128 rows x 4 blocks) and go to tensor memory with
// tcgen05.cp, 32 lanes x 16 bytes spread to all four lane quadrants: row
// 32 j + r of a tile is lane r, column j. Copies and MMAs of one thread run in
// order, so no wait stands between them.
//
// Two kernels:
//   * gemm_kernel (more than kFewRows rows): persistent over CTA pairs, 256 x
//     192 H output tiles in H = 1 or 2 units of 192 columns. Two accumulators
//     of 192 columns leave 128 of the 512 TMEM columns for the scales. H = 1
//     alternates between them, so that the epilogue of a tile overlaps the next
//     one's MMAs; H = 2 uses both for one tile, which reads 30 % fewer bytes
//     from L2 a product, and drains each into registers as packed bf16 before
//     it hands it back. Bound by what L2 gives an SM (with the MMAs left out the
//     copies of 256 x 192 tiles take 573 of 777 us) and by power: 12240 x 6144
//     to 24576 in 645-675 us, 5.5-5.7 PFLOP/s, 0.83-0.87 of four times the
//     measured bf16 rate, about 780 us when it runs for seconds. MMAs of 192
//     columns keep two accumulators and the scales in tensor memory.
//   * few_rows_kernel: the weight takes the 128-row side and the few
//     activation rows the narrow side; bound by reading the weight, K is split
//     over a cluster's CTAs and joined through distributed shared memory, in a
//     fixed order. 1 x 6144 to 18432: 13.5 us, 4.7 TB/s. At 128 rows it takes
//     13.6 us (6144 x 6144) where gemm_kernel takes 15.4, hence kFewRows.
#include "lr_fp4.cuh"
#include "lr_tc.cuh"

namespace lr {

static __device__ unsigned int g_fp4_status = 0;

namespace fp4 {
namespace {

using namespace tc;
using bf16 = __nv_bfloat16;

constexpr int KB = 128;          // bytes of codes per row and stage (256 columns)
constexpr int TM = 128;          // rows a CTA
constexpr int TN = 192;          // columns a unit (an accumulator)
constexpr int kGroupWarps = 4;   // epilogue warps a unit, one per TMEM lane quadrant
constexpr int kThreads = 64 + 2 * 32 * kGroupWarps;
constexpr int kFewThreads = 64 + 32 * kGroupWarps;
constexpr int kOutChunk = 32 * 32 * 2;  // a warp's 32 rows x 32 columns of bf16
constexpr int kBarBytes = 1024;
constexpr int kFewRows = 128;
constexpr int kMaxSplits = 8;  // the largest portable cluster

struct Epilogue {
  const float* row_scale;
  const float* col_scale;
  const bf16* bias;
  bf16* out;
  int64_t ldo;
};

template <int FORMAT>
constexpr int kScaleTiles = FORMAT == kNv ? 4 : 2;  // 512-byte scale tiles per 128 rows and stage

// Instruction descriptor: E2M1 operands (1 at bits 7 and 10), N / 8 at 17, scale
// type at 23 (0: e4m3, 1: e8m0), M / 16 at 24.
template <int FORMAT>
constexpr uint32_t idesc(int m, int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n / 8) << 17) | ((FORMAT == kMx ? 1u : 0u) << 23) |
         ((uint32_t)(m / 16) << 24);
}

// Shared-memory descriptor of a 512-byte scale tile: no swizzle, 8 rows of 16 bytes contiguous.
__device__ __forceinline__ uint64_t desc_scales(uint32_t saddr) {
  return (uint64_t)(saddr >> 4) | ((uint64_t)(128u >> 4) << 16) | ((uint64_t)(128u >> 4) << 32) |
         ((uint64_t)1u << 46);
}
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t saddr) {
  if (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc_scales(saddr)) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc_scales(saddr)) : "memory");
}
#define LR_FP4_MMA(GROUP, KIND)                                                                                   \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                                   \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n" ::"r"(d), \
               "l"(a), "l"(b), "r"(desc), "r"(accumulate), "r"(sa), "r"(sb)                                        \
               : "memory")
template <int FORMAT, bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t sa, uint32_t sb,
                                    uint32_t accumulate) {
  if (FORMAT == kNv) {
    if (PAIR)
      LR_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else
      LR_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  } else {
    if (PAIR)
      LR_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
    else
      LR_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
  }
}

// A stage's scales of 128-row tiles to tensor memory: A's to sfa (four columns a
// tile of blocks), B's RB row tiles to sfb (4 RB columns a tile of blocks).
template <int FORMAT, bool PAIR, int RB>
__device__ __forceinline__ void issue_scales(uint32_t sa0, uint32_t sb0, uint32_t sfa, uint32_t sfb) {
  constexpr int CT = kScaleTiles<FORMAT>;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    copy_scales<PAIR>(sfa + c * 4, sa0 + c * 512);
#pragma unroll
    for (int r = 0; r < RB; ++r) copy_scales<PAIR>(sfb + (c * RB + r) * 4, sb0 + (r * CT + c) * 512);
  }
}
// A stage's four MMAs. shift: column at which the unit's first B row stands.
template <int FORMAT, bool PAIR, int RB>
__device__ __forceinline__ void issue_mmas(uint32_t d, uint32_t a0, uint32_t b0, uint32_t sfa, uint32_t sfb,
                                           uint32_t shift, uint32_t desc, bool first) {
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const int c = FORMAT == kNv ? kk : kk / 2;
    // the half of a column's four bytes that this MMA's two mxfp4 scales are
    const uint32_t ids = FORMAT == kNv ? 0u : (uint32_t)((kk & 1) * 2);
    mma<FORMAT, PAIR>(d, desc_kmajor(a0 + kk * 32), desc_kmajor(b0 + kk * 32), desc | (ids << 4) | (ids << 29),
                      sfa + c * 4, sfb + c * 4 * RB + shift, first && kk == 0 ? 0u : 1u);
  }
}

// ------------------------------------------------------------------ many rows
template <int FORMAT, int H>
struct Tile {
  static constexpr int kRows = 2 * TM, kCols = H * TN;
  static constexpr int kRB = H == 1 ? 2 : 3;  // 128-row scale tiles that 192 H rows of B touch
  static constexpr int kA = TM * KB, kB = kCols / 2 * KB;  // a CTA loads its rows of A and half the rows of B
  static constexpr int kSa = kScaleTiles<FORMAT> * 512, kSb = kRB * kScaleTiles<FORMAT> * 512;
  static constexpr int kStage = kA + kB + kSa + kSb;
  static constexpr int kStages = H == 1 ? 5 : 4;
  static constexpr int kOut = 2 * kGroupWarps * kOutChunk;
  static constexpr int kColBytes = 4 * TN * 8;  // (column scale, bias), two units a group
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kOut + kColBytes + kBarBytes;
  static_assert(kStage % 1024 == 0 && kSmem <= 232448, "shared memory");
  // tensor memory: accumulators at 0 and TN, scales of two stages from 2 TN
  static constexpr int kSfCols = kScaleTiles<FORMAT> * 4 * (1 + kRB);
  static_assert(2 * TN + 2 * kSfCols <= 512, "tensor memory");
};

// `group` consecutive row blocks are swept across all column blocks before the
// next group starts, so their codes stay in L2 while B streams through.
__device__ __forceinline__ void tile_coords(int t, int num_m, int num_n, int group, int& mb, int& nb) {
  const int span = group * num_n;
  const int g = t / span, first = g * group;
  const int size = min(num_m - first, group);
  const int r = t - g * span;
  mb = first + r % size;
  nb = r / size;
}

// A staged 32 x 32 chunk to rows of any alignment: a row a store, a column a lane. (Pairs of columns in 4-byte stores
// took half as many and twice the time: the odd rows' pairs straddle the staged words.)
__device__ __forceinline__ void store_rows(const uint8_t* buf, bf16* dst, int64_t ld, int rows, bool inside, int lane) {
  uint16_t* to = reinterpret_cast<uint16_t*>(dst) + lane;
#pragma unroll
  for (int i0 = 0; i0 < 32; i0 += 8) {
    uint16_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[k] = *reinterpret_cast<const uint16_t*>(buf + (i0 + k) * 64 + (((lane >> 3) ^ (((i0 + k) >> 1) & 3)) << 4) + (lane & 7) * 2);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (inside && i0 + k < rows) to[(i0 + k) * ld] = v[k];
  }
}

// The 128 threads of an epilogue group meet; true if every one of them brought `ok`.
__device__ __forceinline__ bool group_barrier(int group, bool ok) {
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.and.pred q, %1, 128, p;\n\t"
               "selp.u32 %0, 1, 0, q;\n\t}\n"
               : "=r"(all)
               : "r"(1 + group), "r"(ok ? 1u : 0u)
               : "memory");
  return all != 0;
}

// TMA_OUT: out's rows start on 16-byte boundaries.
template <int FORMAT, int H, bool TMA_OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                const __grid_constant__ CUtensorMap map_out, int M, int N, int K, int group,
                const Epilogue ep) {
  using C = Tile<FORMAT, H>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* out_stage = smem + C::kStages * C::kStage;
  float2* cols = reinterpret_cast<float2*>(out_stage + C::kOut);
  uint64_t* bars = reinterpret_cast<uint64_t*>(out_stage + C::kOut + C::kColBytes);
  uint64_t* full = bars;                    // the leader's: both CTAs' copies landed
  uint64_t* empty = bars + C::kStages;      // MMAs have read the stage
  uint64_t* tfull = bars + 2 * C::kStages;  // [2] accumulator ready
  uint64_t* tempty = tfull + 2;             // [2] the leader's: accumulator drained
  uint64_t* drain = tfull + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  const Watch watch{tmem_slot + 1, &g_fp4_status};

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int num_m = (M + C::kRows - 1) / C::kRows, num_n = (N + C::kCols - 1) / C::kCols;
  const int tiles = num_m * num_n;
  const int kblocks = (K / 2 + KB - 1) / KB;
  const int first_tile = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&tfull[a]), 1);
      mbar_init(smem_u32(&tempty[a]), 2 * kGroupWarps);
    }
    mbar_init(smem_u32(drain), 1);
    *watch.abort_flag = 0u;
    mbar_init_fence();
    prefetch_map(&map_a);
    prefetch_map(&map_b);
    prefetch_map(&map_sa);
    prefetch_map(&map_sb);
  }
  if (warp == 1) tmem_alloc<2>(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_predecessor();

  if (warp == 0) {
    // -------------------------------------------------------- copies
    const bool el = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = first_tile; t < tiles && ok; t += step) {
      int mb, nb;
      tile_coords(t, num_m, num_n, group, mb, nb);
      const int m0 = mb * C::kRows + (int)rank * TM, n0 = nb * C::kCols;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!warp_wait(smem_u32(&empty[stage]), phase ^ 1u, watch, lane)) {
          ok = false;
          break;
        }
        if (el) {
          const uint32_t a = smem_u32(smem + stage * C::kStage), b = a + C::kA, sa = b + C::kB, sb = sa + C::kSa;
          const uint32_t own = smem_u32(&full[stage]);
          if (rank == 0) mbar_expect_tx(own, 2 * C::kStage);
          const uint32_t bar = map_to_rank(own, 0);
          tma_load_2d_pair(a, &map_a, bar, kb * KB, m0);
          // unit u of B (192 rows): rows [96 rank, +96) of it
#pragma unroll
          for (int u = 0; u < H; ++u)
            tma_load_2d_pair(b + u * (TN / 2) * KB, &map_b, bar, kb * KB, n0 + u * TN + (int)rank * (TN / 2));
          tma_load_3d_pair(sa, &map_sa, bar, 0, kb * kScaleTiles<FORMAT>, m0 / 128);
          tma_load_3d_pair(sb, &map_sb, bar, 0, kb * kScaleTiles<FORMAT>, n0 / 128);
        }
        __syncwarp();
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok) {
      // giving up: time for the copies in flight to land before the CTA can exit
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 100000ull) {
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ------------------------------------------------------ MMAs
      const bool el = elect_one();
      int stage = 0, local = 0;
      uint32_t phase = 0, buffer = 0;
      bool ok = true;
      constexpr uint32_t kDesc = idesc<FORMAT>(C::kRows, TN);
      for (int t = first_tile; t < tiles && ok; t += step, ++local) {
        int mb, nb;
        tile_coords(t, num_m, num_n, group, mb, nb);
        // H = 1: a unit starts at row 0 or 64 of its scale tile. H = 2: unit 1 starts 192 rows in.
        const uint32_t shift = H == 1 ? (uint32_t)(nb * TN % 128 / 32) : 0u;
        const int acc = H == 1 ? local & 1 : 0;
        const uint32_t parity = (H == 1 ? (uint32_t)(local >> 1) & 1u : (uint32_t)local & 1u) ^ 1u;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!warp_wait(smem_u32(&full[stage]), phase, watch, lane) ||
              (kb == 0 && !warp_wait(smem_u32(&tempty[acc]), parity, watch, lane))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_u32(smem + stage * C::kStage), b = a + C::kA, sa = b + C::kB, sb = sa + C::kSa;
          const uint32_t sfa = tmem + 2 * TN + buffer * C::kSfCols, sfb = sfa + kScaleTiles<FORMAT> * 4;
          if (el) {
            issue_scales<FORMAT, true, C::kRB>(sa, sb, sfa, sfb);
            issue_mmas<FORMAT, true, C::kRB>(tmem + acc * TN, a, b, sfa, sfb, shift, kDesc, kb == 0);
          }
          if (H == 2) {
            if (kb == 0) {
              if (!warp_wait(smem_u32(&tempty[1]), parity, watch, lane)) {
                ok = false;
                break;
              }
              tc_fence_after();
            }
            if (el) {
              if (kb == kblocks - 1) mma_commit_pair(smem_u32(&tfull[0]), (uint16_t)3);
              issue_mmas<FORMAT, true, C::kRB>(tmem + TN, a, b + (TN / 2) * KB, sfa, sfb, TN / 32, kDesc, kb == 0);
            }
          }
          if (el) {
            mma_commit_pair(smem_u32(&empty[stage]), (uint16_t)3);
            if (kb == kblocks - 1) mma_commit_pair(smem_u32(&tfull[H == 1 ? acc : 1]), (uint16_t)3);
          }
          __syncwarp();
          buffer ^= 1u;
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        if (el) mma_commit_pair(smem_u32(drain), (uint16_t)1);
        __syncwarp();
        drain_bounded(smem_u32(drain), 0u);
      }
    }
  } else {
    // -------------------------------------------------------- epilogue
    // Group g drains accumulator g: every other tile (H = 1) or unit g of every tile (H = 2).
    const int g = (warp - 2) / kGroupWarps, quad = warp & 3;  // TMEM lanes 32 quad .. + 32
    uint8_t* buf = out_stage + (warp - 2) * kOutChunk;
    int turn = 0;
    for (int t = first_tile + (H == 1 ? g * step : 0); t < tiles; t += H == 1 ? 2 * step : step, ++turn) {
      int mb, nb;
      tile_coords(t, num_m, num_n, group, mb, nb);
      const int n0 = nb * C::kCols + (H == 1 ? 0 : g * TN);
      const int row0 = mb * C::kRows + (int)rank * TM + quad * 32, row = row0 + lane;
      float2* cs = cols + (g * 2 + (turn & 1)) * TN;
      for (int i = quad * 32 + lane; i < TN; i += 32 * kGroupWarps) {
        const int n = n0 + i;
        cs[i] = make_float2(n < N && ep.col_scale ? ep.col_scale[n] : 1.0f,
                            n < N && ep.bias ? __bfloat162float(ep.bias[n]) : 0.0f);
      }
      const float rs = row < M && ep.row_scale ? ep.row_scale[row] : 1.0f;
      const bool ok = warp_wait(smem_u32(&tfull[g]), (uint32_t)turn & 1u, watch, lane);
      if (!group_barrier(g, ok)) break;
      tc_fence_after();
      // 32 columns to this warp's staging buffer (64-byte swizzle: conflict-free 16-byte writes) and out.
      auto store = [&](int c, const uint32_t* y) {
        const int col0 = n0 + c * 32;
        if (col0 >= N) return;
        if (TMA_OUT && lane == 0) bulk_wait_read();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) =
              make_uint4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
        if constexpr (TMA_OUT) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_out, smem_u32(buf), col0, row0);
            bulk_commit();
          }
        } else {  // rows that start off 16-byte boundaries
          __syncwarp();
          store_rows(buf, ep.out + (int64_t)row0 * ep.ldo + col0, ep.ldo, M - row0, col0 + lane < N, lane);
        }
      };
      // The next tile's MMAs wait for this accumulator where H = 2: it is emptied before anything is stored. The last
      // tile's columns are stored as they come (512 x 4096 to 12288: 1.5 of 17 us).
      const bool hold = H == 2 && t + step < tiles;
      uint32_t y[TN / 2];
      const uint32_t tbase = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(g * TN);
#pragma unroll
      for (int c = 0; c < TN / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(tbase + (uint32_t)(c * 32), r);
        if (c == TN / 32 - 1) {  // everything is in registers: hand the accumulator back
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(smem_u32(&tempty[g]), 0u);
        }
        const float4* c4 = reinterpret_cast<const float4*>(cs + c * 32);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float4 f = c4[e];  // two columns' (scale, bias)
          y[c * 16 + e] =
              cvt2(fmaf(__uint_as_float(r[2 * e]) * rs, f.x, f.y), fmaf(__uint_as_float(r[2 * e + 1]) * rs, f.z, f.w));
        }
        if (!hold) store(c, y + c * 16);
      }
      if (hold) {
#pragma unroll
        for (int c = 0; c < TN / 32; ++c) store(c, y + c * 16);
      }
    }
    if (TMA_OUT && lane == 0) bulk_wait_all();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem, 512);
  }
}

// ------------------------------------------------------------------ few rows
template <int FORMAT, int NT>
struct Few {
  static constexpr int kA = TM * KB, kB = NT * KB;
  static constexpr int kS = kScaleTiles<FORMAT> * 512;
  static constexpr int kStage = kA + kB + 2 * kS;
  static constexpr int kStages = NT <= 32 ? 4 : 3;  // two CTAs an SM
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kBarBytes;
  static constexpr int kSfCols = kScaleTiles<FORMAT> * 8;
  static constexpr int kTmem = NT <= 64 ? 128 : 256;
  static_assert(kStage % 1024 == 0 && NT + 2 * kSfCols <= kTmem && 2 * (kSmem + 1024) <= 233472, "two CTAs an SM");
  static_assert(TM * NT * 4 <= kStages * kStage, "the partial tile reuses the stages");
};

// Weight rows [128 x, +128) against the M <= NT activation rows; the cluster's
// CTAs take consecutive slices of K.
template <int FORMAT, int NT>
__global__ void __launch_bounds__(kFewThreads)
    few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                    const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ CUtensorMap map_sx, int M, int N,
                    int K, int splits, const Epilogue ep) {
  using C = Few<FORMAT, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStage);
  uint64_t* full = bars;
  uint64_t* empty = bars + C::kStages;
  uint64_t* done = bars + 2 * C::kStages;
  uint64_t* drain = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  const Watch watch{tmem_slot + 1, &g_fp4_status};

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int n0 = (int)(blockIdx.x / splits) * TM;
  const int kblocks = (K / 2 + KB - 1) / KB;
  const int kb0 = (int)((int64_t)kblocks * rank / splits), kb1 = (int)((int64_t)kblocks * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(done), 1);
    mbar_init(smem_u32(drain), 1);
    *watch.abort_flag = 0u;
    mbar_init_fence();
    prefetch_map(&map_w);
    prefetch_map(&map_x);
    prefetch_map(&map_sw);
    prefetch_map(&map_sx);
  }
  if (warp == 1) tmem_alloc<1>(smem_u32(tmem_slot), C::kTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_predecessor();

  if (warp == 0) {
    const bool el = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_wait(smem_u32(&empty[stage]), phase ^ 1u, watch, lane)) {
        ok = false;
        break;
      }
      if (el) {
        const uint32_t a = smem_u32(smem + stage * C::kStage), b = a + C::kA, sa = b + C::kB, sb = sa + C::kS;
        const uint32_t bar = smem_u32(&full[stage]);
        mbar_expect_tx(bar, C::kStage);
        tma_load_2d(a, &map_w, bar, kb * KB, n0);
        tma_load_2d(b, &map_x, bar, kb * KB, 0);
        tma_load_3d(sa, &map_sw, bar, 0, kb * kScaleTiles<FORMAT>, n0 / 128);
        tma_load_3d(sb, &map_sx, bar, 0, kb * kScaleTiles<FORMAT>, 0);
      }
      __syncwarp();
      if (++stage == C::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (!ok) {
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 100000ull) {
      }
    }
  } else if (warp == 1) {
    const bool el = elect_one();
    int stage = 0;
    uint32_t phase = 0, buffer = 0;
    bool ok = true;
    constexpr uint32_t kDesc = idesc<FORMAT>(TM, NT);
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_wait(smem_u32(&full[stage]), phase, watch, lane)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (el) {
        const uint32_t a = smem_u32(smem + stage * C::kStage), b = a + C::kA, sa = b + C::kB, sb = sa + C::kS;
        const uint32_t sfa = tmem + NT + buffer * C::kSfCols, sfb = sfa + kScaleTiles<FORMAT> * 4;
        issue_scales<FORMAT, false, 1>(sa, sb, sfa, sfb);
        issue_mmas<FORMAT, false, 1>(tmem, a, b, sfa, sfb, 0u, kDesc, kb == kb0);
        mma_commit(smem_u32(&empty[stage]));
        if (kb == kb1 - 1) mma_commit(smem_u32(done));
      }
      __syncwarp();
      buffer ^= 1u;
      if (++stage == C::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (!ok) {
      if (el) mma_commit(smem_u32(drain));
      __syncwarp();
      drain_bounded(smem_u32(drain), 0u);
    }
  } else {
    // The partial tile, [activation row][weight row] fp32, over the stages (every copy into them has been read).
    const int quad = warp & 3;
    if (warp_wait(smem_u32(done), 0u, watch, lane)) {
      tc_fence_after();
      float* part = reinterpret_cast<float*>(smem) + quad * 32 + lane;
      #pragma unroll 1
      for (int c = 0; c < M; c += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)c, r);
#pragma unroll
        for (int e = 0; e < 16; ++e) part[(c + e) * TM] = __uint_as_float(r[e]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync_all();
  if (warp >= 2) {
    // A warp an activation row, a lane four outputs; the slices' sums are fetched together and added in order.
    const int n = n0 + lane * 4;
    float cs[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cs[e] = n + e < N && ep.col_scale ? ep.col_scale[n + e] : 1.0f;
      b[e] = n + e < N && ep.bias ? __bfloat162float(ep.bias[n + e]) : 0.0f;
    }
    const bool whole = n + 4 <= N && ep.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(ep.out) & 7) == 0;
    for (int i = rank + (warp - 2) * splits; i < M; i += kGroupWarps * splits) {
      const uint32_t part = smem_u32(smem) + (uint32_t)(i * TM + lane * 4) * 4;
      float4 v[kMaxSplits];
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s) {
        v[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (s < splits)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[s].x), "=f"(v[s].y), "=f"(v[s].z), "=f"(v[s].w)
                       : "r"(map_to_rank(part, (uint32_t)s))
                       : "memory");
      }
      float y[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
      for (int s = 1; s < kMaxSplits; ++s) y[0] += v[s].x, y[1] += v[s].y, y[2] += v[s].z, y[3] += v[s].w;
      const float rs = ep.row_scale ? ep.row_scale[i] : 1.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(y[e] * rs, cs[e], b[e]);
      bf16* dst = ep.out + (int64_t)i * ep.ldo + n;
      if (whole) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(cvt2(y[0], y[1]), cvt2(y[2], y[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N) dst[e] = __float2bfloat16_rn(y[e]);
      }
    }
  }
  __syncwarp();
  if (splits > 1) cluster_sync_all();  // peers have read this CTA's shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, C::kTmem);
  }
}

// ------------------------------------------------------------------ host
int code_map(CUtensorMap* map, const void* base, int64_t rows, int64_t K, uint32_t box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)(K / 2), (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(K / 2)};
  const cuuint32_t box[2] = {KB, box_rows};
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
template <int FORMAT>
int scale_map(CUtensorMap* map, const void* base, int64_t rows, int64_t K, uint32_t row_tiles) {
  const cuuint64_t ctiles = (cuuint64_t)((K / (FORMAT == kNv ? 16 : 32) + 3) / 4);
  const cuuint64_t dims[3] = {128, ctiles, (cuuint64_t)((rows + 127) / 128)};
  const cuuint64_t strides[2] = {512, 512 * ctiles};
  const cuuint32_t box[3] = {128, (cuuint32_t)kScaleTiles<FORMAT>, row_tiles};
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct Operands {
  const void *a, *as, *b, *bs;
  int M, N, K;
};

template <int FORMAT, int H, bool TMA_OUT>
int launch_many_to(const Operands& o, const Epilogue& ep, cudaStream_t stream) {
  using C = Tile<FORMAT, H>;
  CUtensorMap ma, mb, msa, msb, mo{};
  int st;
  if ((st = code_map(&ma, o.a, o.M, o.K, TM)) || (st = code_map(&mb, o.b, o.N, o.K, TN / 2)) ||
      (st = scale_map<FORMAT>(&msa, o.as, o.M, o.K, 1)) || (st = scale_map<FORMAT>(&msb, o.bs, o.N, o.K, C::kRB)))
    return st;
  if (TMA_OUT) {
    const cuuint64_t dims[2] = {(cuuint64_t)o.N, (cuuint64_t)o.M}, strides[1] = {(cuuint64_t)ep.ldo * 2};
    const cuuint32_t box[2] = {32, 32};
    if ((st = make_map(&mo, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ep.out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B)))
      return st;
  }
  static bool done[64] = {};
  if ((st = configure_smem(gemm_kernel<FORMAT, H, TMA_OUT>, C::kSmem, done))) return st;
  const int num_m = (o.M + C::kRows - 1) / C::kRows, num_n = (o.N + C::kCols - 1) / C::kCols;
  const int tiles = num_m * num_n, pairs = sm_count() / 2;
  int64_t group = (24ll << 20) / ((int64_t)C::kRows * o.K / 2);  // 24 MB of A's codes
  if (group < 1) group = 1;
  return launch("fp4 gemm", gemm_kernel<FORMAT, H, TMA_OUT>, dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs))), kThreads, C::kSmem,
                stream, 1, true, ma, mb, msa, msb, mo, o.M, o.N, o.K, (int)(group < num_m ? group : num_m), ep);
}
template <int FORMAT, int H>
int launch_many(const Operands& o, const Epilogue& ep, cudaStream_t stream) {
  if (ep.ldo % 8 == 0 && aligned(ep.out, 16)) return launch_many_to<FORMAT, H, true>(o, ep, stream);
  return launch_many_to<FORMAT, H, false>(o, ep, stream);
}

template <int FORMAT, int NT>
int launch_few(const Operands& o, const Epilogue& ep, cudaStream_t stream) {
  using C = Few<FORMAT, NT>;
  CUtensorMap mw, mx, msw, msx;
  int st;
  if ((st = code_map(&mw, o.b, o.N, o.K, TM)) || (st = code_map(&mx, o.a, o.M, o.K, NT)) ||
      (st = scale_map<FORMAT>(&msw, o.bs, o.N, o.K, 1)) || (st = scale_map<FORMAT>(&msx, o.as, o.M, o.K, 1)))
    return st;
  static bool done[64] = {};
  if ((st = configure_smem(few_rows_kernel<FORMAT, NT>, C::kSmem, done))) return st;
  const int tiles = (o.N + TM - 1) / TM;
  const int kblocks = (o.K / 2 + KB - 1) / KB;
  // As many slices as fill the GPU with two CTAs an SM and leave each two stages; powers of two, as clusters of 3 or 6 do not
  // pack (1x6144 to 6144 with four slices 8.0 us, with six 11.9).
  int splits = 1;
  while (splits < kMaxSplits && tiles * splits * 2 <= 2 * sm_count() && kblocks >= 4 * splits) splits *= 2;
  return launch("fp4 gemm (few rows)", few_rows_kernel<FORMAT, NT>, dim3((unsigned)(tiles * splits)), kFewThreads, C::kSmem,
                stream, (unsigned)splits, true, mw, mx, msw, msx, o.M, o.N, o.K, splits, ep);
}

template <int FORMAT>
int gemm(const Operands& o, const Epilogue& ep, cudaStream_t stream) {
  if (o.M <= 16) return launch_few<FORMAT, 16>(o, ep, stream);
  if (o.M <= 32) return launch_few<FORMAT, 32>(o, ep, stream);
  if (o.M <= 64) return launch_few<FORMAT, 64>(o, ep, stream);
  if (o.M <= kFewRows) return launch_few<FORMAT, 128>(o, ep, stream);
  // a wide tile takes about 1.4 times a narrow one's time for twice its columns
  const int64_t pairs = sm_count() / 2, num_m = (o.M + 2 * TM - 1) / (2 * TM);
  const int64_t narrow = (num_m * ((o.N + TN - 1) / TN) + pairs - 1) / pairs;
  const int64_t wide = (num_m * ((o.N + 2 * TN - 1) / (2 * TN)) + pairs - 1) / pairs;
  if (wide * 7 <= narrow * 5) return launch_many<FORMAT, 2>(o, ep, stream);
  return launch_many<FORMAT, 1>(o, ep, stream);
}

}  // namespace
}  // namespace fp4

int read_status_fp4(unsigned int* bits, int clear) {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_fp4_status, sizeof(v)) != cudaSuccess) return launch_status("reading the device status");
  if (clear) {
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbol(g_fp4_status, &zero, sizeof(zero)) != cudaSuccess)
      return launch_status("clearing the device status");
  }
  *bits |= v;
  return LR_OK;
}

}  // namespace lr

extern "C" int lr_fp4_gemm(const void* a, const void* a_scales, const void* b, const void* b_scales, int64_t M,
                           int64_t N, int64_t K, int format, const float* row_scale, const float* col_scale,
                           const void* bias, void* out, int64_t ldo, void* stream) {
  using namespace lr;
  LR_REQUIRE(format == LR_FP4_NV || format == LR_FP4_MX, "fp4_gemm: unknown format %d", format);
  LR_REQUIRE(M >= 0 && N > 0 && K > 0 && M < (1ll << 31) - 512 && N < (1ll << 31) - 512 && K <= (1 << 30) &&
                 ((M + 255) / 256) * ((N + 191) / 192) < (1ll << 31),
             "fp4_gemm: invalid shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (K % 32) return set_error(LR_ERR_UNSUPPORTED, "fp4_gemm: K must be a multiple of 32, got %lld", (long long)K);
  if (M == 0) return LR_OK;
  LR_REQUIRE(a && a_scales && b && b_scales && out, "fp4_gemm: null pointer");
  LR_REQUIRE(ldo >= N, "fp4_gemm: ldo %lld < N %lld", (long long)ldo, (long long)N);
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(a_scales, 16) || !aligned(b_scales, 16))
    return set_error(LR_ERR_UNSUPPORTED, "fp4_gemm: codes and scales must be 16-byte aligned");
  const fp4::Operands o{a, a_scales, b, b_scales, (int)M, (int)N, (int)K};
  const fp4::Epilogue ep{row_scale, col_scale, static_cast<const __nv_bfloat16*>(bias), static_cast<__nv_bfloat16*>(out),
                         ldo};
  auto* st = static_cast<cudaStream_t>(stream);
  return format == LR_FP4_NV ? fp4::gemm<fp4::kNv>(o, ep, st) : fp4::gemm<fp4::kMx>(o, ep, st);
}
