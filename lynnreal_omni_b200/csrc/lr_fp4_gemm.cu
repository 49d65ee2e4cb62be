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
//   * gemm_kernel (more than kFewRows rows): persistent, 128 x 192 (a CTA) or
//     256 x 192 (a CTA pair) output tiles, two accumulators of 192 columns, so
//     that the epilogue of a tile overlaps the next one's MMAs; 192 leaves 128
//     of the 512 TMEM columns for the scales, which 256 would not.
//   * few_rows_kernel: the weight takes the 128-row side and the few
//     activation rows the narrow side; bound by reading the weight, K is split
//     over a cluster's CTAs and joined through distributed shared memory, in a
//     fixed order.
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
constexpr int TN = 192;          // columns a tile
constexpr int kEpiWarps = 4;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kOutChunk = 32 * 32 * 2;  // a warp's 32 rows x 32 columns of bf16
constexpr int kBarBytes = 1024;
constexpr int kFewRows = 128;

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
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128u >> 4) << 16) | ((uint64_t)(128u >> 4) << 32) |
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

// One stage: scales to tensor memory, then four MMAs. RB: 128-row scale tiles
// of B; sfa, sfb: their columns in tensor memory; shift: column at which the
// tile's first B row stands.
template <int FORMAT, bool PAIR, int RB>
__device__ __forceinline__ void issue_stage(uint32_t d, uint32_t a0, uint32_t b0, uint32_t sa0, uint32_t sb0,
                                            uint32_t sfa, uint32_t sfb, uint32_t shift, uint32_t desc, bool first) {
  constexpr int CT = kScaleTiles<FORMAT>;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    copy_scales<PAIR>(sfa + c * 4, sa0 + c * 512);
#pragma unroll
    for (int r = 0; r < RB; ++r) copy_scales<PAIR>(sfb + c * 4 * RB + r * 4, sb0 + (r * CT + c) * 512);
  }
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
template <int FORMAT, bool PAIR>
struct Tile {
  static constexpr int kBRows = PAIR ? TN / 2 : TN;
  static constexpr int kA = TM * KB, kB = kBRows * KB;
  static constexpr int kSa = kScaleTiles<FORMAT> * 512, kSb = 2 * kScaleTiles<FORMAT> * 512;
  static constexpr int kStage = kA + kB + kSa + kSb;
  static constexpr int kStages = PAIR ? 6 : 4;
  static constexpr int kOut = kEpiWarps * 2 * kOutChunk;
  static constexpr int kCols = 2 * TN * 8;  // (column scale, bias) of two tiles
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kOut + kCols + kBarBytes;
  static_assert(kStage % 1024 == 0 && kSmem <= 232448, "shared memory");
  // tensor memory: accumulators at 0 and TN, scales of two stages from 2 TN
  static constexpr int kSfCols = kScaleTiles<FORMAT> * 12;
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

// All epilogue warps meet; true if every one of them brought `ok`.
__device__ __forceinline__ bool epilogue_barrier(bool ok) {
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 128, p;\n\t"
               "selp.u32 %0, 1, 0, q;\n\t}\n"
               : "=r"(all)
               : "r"(ok ? 1u : 0u)
               : "memory");
  return all != 0;
}

template <int FORMAT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                const __grid_constant__ CUtensorMap map_out, int M, int N, int K, int group, int tma_out,
                const Epilogue ep) {
  using C = Tile<FORMAT, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* out_stage = smem + C::kStages * C::kStage;
  float2* cols = reinterpret_cast<float2*>(out_stage + C::kOut);
  uint64_t* bars = reinterpret_cast<uint64_t*>(out_stage + C::kOut + C::kCols);
  uint64_t* full = bars;                   // copies landed (the leader's, of both CTAs)
  uint64_t* empty = bars + C::kStages;     // MMAs have read the stage
  uint64_t* tfull = bars + 2 * C::kStages;  // [2] accumulator ready
  uint64_t* tempty = tfull + 2;             // [2] accumulator drained (the leader's)
  uint64_t* drain = tfull + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  const Watch watch{tmem_slot + 1, &g_fp4_status};

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  constexpr int kRows = PAIR ? 2 * TM : TM;
  const int num_m = (M + kRows - 1) / kRows, num_n = (N + TN - 1) / TN;
  const int tiles = num_m * num_n;
  const int kblocks = (K / 2 + KB - 1) / KB;
  const int first_tile = PAIR ? blockIdx.x >> 1 : blockIdx.x;
  const int step = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&tfull[a]), 1);
      mbar_init(smem_u32(&tempty[a]), (PAIR ? 2 : 1) * kEpiWarps);
    }
    mbar_init(smem_u32(drain), 1);
    *watch.abort_flag = 0u;
    mbar_init_fence();
    prefetch_map(&map_a);
    prefetch_map(&map_b);
    prefetch_map(&map_sa);
    prefetch_map(&map_sb);
  }
  if (warp == 1) tmem_alloc<PAIR ? 2 : 1>(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------ copies
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, any = false;
      for (int t = first_tile; t < tiles && ok; t += step) {
        int mb, nb;
        tile_coords(t, num_m, num_n, group, mb, nb);
        const int m0 = mb * kRows + (int)rank * TM, n0 = nb * TN;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!wait_bounded(smem_u32(&empty[stage]), phase ^ 1u, watch)) {
            ok = false;
            break;
          }
          const uint32_t a = smem_u32(smem + stage * C::kStage), b = a + C::kA, sa = b + C::kB, sb = sa + C::kSa;
          uint32_t bar = smem_u32(&full[stage]);
          if (rank == 0) mbar_expect_tx(bar, (PAIR ? 2 : 1) * C::kStage);
          if (PAIR) {
            bar = map_to_rank(bar, 0);
            tma_load_2d_pair(a, &map_a, bar, kb * KB, m0);
            tma_load_2d_pair(b, &map_b, bar, kb * KB, n0 + (int)rank * C::kBRows);
            tma_load_3d_pair(sa, &map_sa, bar, 0, kb * kScaleTiles<FORMAT>, m0 / 128);
            tma_load_3d_pair(sb, &map_sb, bar, 0, kb * kScaleTiles<FORMAT>, n0 / 128);
          } else {
            tma_load_2d(a, &map_a, bar, kb * KB, m0);
            tma_load_2d(b, &map_b, bar, kb * KB, n0);
            tma_load_3d(sa, &map_sa, bar, 0, kb * kScaleTiles<FORMAT>, m0 / 128);
            tma_load_3d(sb, &map_sb, bar, 0, kb * kScaleTiles<FORMAT>, n0 / 128);
          }
          any = true;
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && any) {
        // giving up: time for the copies in flight to land before the CTA can exit
        const unsigned long long t0 = globaltimer();
        while (globaltimer() - t0 < 100000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // ------------------------------------------------------ MMAs
      int stage = 0, local = 0;
      uint32_t phase = 0, buffer = 0;
      bool ok = true;
      constexpr uint32_t kDesc = idesc<FORMAT>(kRows, TN);
      for (int t = first_tile; t < tiles && ok; t += step, ++local) {
        int mb, nb;
        tile_coords(t, num_m, num_n, group, mb, nb);
        const uint32_t shift = (uint32_t)(nb * TN % 128 / 32);  // a tile starts at row 0 or 64 of B's scale tile
        const int acc = local & 1;
        if (!wait_bounded(smem_u32(&tempty[acc]), ((uint32_t)(local >> 1) & 1u) ^ 1u, watch)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!wait_bounded(smem_u32(&full[stage]), phase, watch)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_u32(smem + stage * C::kStage), b = a + C::kA, sa = b + C::kB, sb = sa + C::kSa;
          const uint32_t sf = tmem + 2 * TN + buffer * C::kSfCols;
          issue_stage<FORMAT, PAIR, 2>(tmem + acc * TN, a, b, sa, sb, sf, sf + kScaleTiles<FORMAT> * 4, shift, kDesc,
                                       kb == 0);
          buffer ^= 1u;
          if (PAIR)
            mma_commit_pair(smem_u32(&empty[stage]), (uint16_t)3);
          else
            mma_commit(smem_u32(&empty[stage]));
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) {
          if (PAIR)
            mma_commit_pair(smem_u32(&tfull[acc]), (uint16_t)3);
          else
            mma_commit(smem_u32(&tfull[acc]));
        }
      }
      if (!ok) {
        if (PAIR)
          mma_commit_pair(smem_u32(drain), (uint16_t)1);
        else
          mma_commit(smem_u32(drain));
        drain_bounded(smem_u32(drain), 0u);
      }
    }
  } else {
    // -------------------------------------------------------- epilogue
    const int quad = warp & 3;  // TMEM lanes 32 quad .. + 32
    uint8_t* staging = out_stage + (warp - 2) * 2 * kOutChunk;
    uint32_t chunk = 0;
    int local = 0;
    for (int t = first_tile; t < tiles; t += step, ++local) {
      const int acc = local & 1;
      int mb, nb;
      tile_coords(t, num_m, num_n, group, mb, nb);
      const int n0 = nb * TN;
      const int row0 = mb * kRows + (int)rank * TM + quad * 32, row = row0 + lane;
      float2* cs = cols + acc * TN;
      for (int i = threadIdx.x - 64; i < TN; i += 32 * kEpiWarps) {
        const int n = n0 + i;
        cs[i] = make_float2(n < N && ep.col_scale ? ep.col_scale[n] : 1.0f,
                            n < N && ep.bias ? __bfloat162float(ep.bias[n]) : 0.0f);
      }
      const float rs = row < M && ep.row_scale ? ep.row_scale[row] : 1.0f;
      const bool ok = warp_wait(smem_u32(&tfull[acc]), (uint32_t)(local >> 1) & 1u, watch, lane);
      if (!epilogue_barrier(ok)) break;
      tc_fence_after();
      const uint32_t tbase = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * TN);
#pragma unroll 1
      for (int c = 0; c < TN / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(tbase + (uint32_t)(c * 32), r);
        if (c == TN / 32 - 1) {  // everything is in registers: hand the accumulator back
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR)
              mbar_arrive_cluster(smem_u32(&tempty[acc]), 0u);
            else
              mbar_arrive(smem_u32(&tempty[acc]));
          }
        }
        const int col0 = n0 + c * 32;
        if (col0 >= N) continue;
        uint32_t y[16];
        const float4* c4 = reinterpret_cast<const float4*>(cs + c * 32);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float4 f = c4[e];  // two columns' (scale, bias)
          y[e] = cvt2(fmaf(__uint_as_float(r[2 * e]) * rs, f.x, f.y), fmaf(__uint_as_float(r[2 * e + 1]) * rs, f.z, f.w));
        }
        // rows to this warp's staging buffer, 64-byte swizzle: conflict-free 16-byte writes
        uint8_t* buf = staging + (chunk & 1u) * kOutChunk;
        if (tma_out && lane == 0) bulk_wait_read1();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) =
              make_uint4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
        if (tma_out) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_out, smem_u32(buf), col0, row0);
            bulk_commit();
          }
        } else {  // rows that start off 16-byte boundaries: a row a step, a lane a column
          __syncwarp();
          if (col0 + lane < N)
            for (int i = 0; i < 32 && row0 + i < M; ++i)
              ep.out[(int64_t)(row0 + i) * ep.ldo + col0 + lane] = *reinterpret_cast<const bf16*>(
                  buf + i * 64 + ((((uint32_t)lane >> 3) ^ ((i >> 1) & 3)) << 4) + (lane & 7) * 2);
        }
        ++chunk;
      }
    }
    if (tma_out && lane == 0) bulk_wait_all();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<PAIR ? 2 : 1>(tmem, 512);
  }
}

// ------------------------------------------------------------------ few rows
template <int FORMAT, int NT>
struct Few {
  static constexpr int kA = TM * KB, kB = NT * KB;
  static constexpr int kS = kScaleTiles<FORMAT> * 512;
  static constexpr int kStage = kA + kB + 2 * kS;
  static constexpr int kStages = 4;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kBarBytes;
  static constexpr int kSfCols = kScaleTiles<FORMAT> * 8;
  static constexpr int kTmem = NT <= 64 ? 128 : 256;
  static_assert(kStage % 1024 == 0 && NT + 2 * kSfCols <= kTmem && kSmem <= 232448, "budgets");
  static_assert(TM * NT * 4 <= kStages * kStage, "the partial tile reuses the stages");
};

// Weight rows [128 x, +128) against activation rows [NT y, +NT); the cluster's
// CTAs take consecutive slices of K.
template <int FORMAT, int NT>
__global__ void __launch_bounds__(kThreads)
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
  const int n0 = (int)(blockIdx.x / splits) * TM, m0 = (int)blockIdx.y * NT;
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

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!wait_bounded(smem_u32(&empty[stage]), phase ^ 1u, watch)) {
          ok = false;
          break;
        }
        const uint32_t a = smem_u32(smem + stage * C::kStage), b = a + C::kA, sa = b + C::kB, sb = sa + C::kS;
        const uint32_t bar = smem_u32(&full[stage]);
        mbar_expect_tx(bar, C::kStage);
        tma_load_2d(a, &map_w, bar, kb * KB, n0);
        tma_load_2d(b, &map_x, bar, kb * KB, m0);
        tma_load_3d(sa, &map_sw, bar, 0, kb * kScaleTiles<FORMAT>, n0 / 128);
        tma_load_3d(sb, &map_sx, bar, 0, kb * kScaleTiles<FORMAT>, m0 / 128);
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
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, buffer = 0;
      constexpr uint32_t kDesc = idesc<FORMAT>(TM, NT);
      const uint32_t shift = (uint32_t)(m0 % 128 / 32);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!wait_bounded(smem_u32(&full[stage]), phase, watch)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = smem_u32(smem + stage * C::kStage), b = a + C::kA, sa = b + C::kB, sb = sa + C::kS;
        const uint32_t sf = tmem + NT + buffer * C::kSfCols;
        issue_stage<FORMAT, false, 1>(tmem, a, b, sa, sb, sf, sf + kScaleTiles<FORMAT> * 4, shift, kDesc, kb == kb0);
        buffer ^= 1u;
        mma_commit(smem_u32(&empty[stage]));
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) {
        mma_commit(smem_u32(done));
      } else {
        mma_commit(smem_u32(drain));
        drain_bounded(smem_u32(drain), 0u);
      }
    }
  } else {
    // The partial tile, [activation row][weight row] fp32, over the stages (every copy into them has been read).
    const int quad = warp & 3;
    ok = warp_wait(smem_u32(done), 0u, watch, lane);
    if (ok) {
      tc_fence_after();
      float* part = reinterpret_cast<float*>(smem) + quad * 32 + lane;
      const int live = min(NT, M - m0);
#pragma unroll 1
      for (int c = 0; c < live; c += 16) {
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
    // Activation rows rank, rank + splits, ...: the slices' sums added in order.
    const int quad = warp & 3, n = n0 + quad * 32 + lane;
    const float cs = n < N && ep.col_scale ? ep.col_scale[n] : 1.0f;
    const float b = n < N && ep.bias ? __bfloat162float(ep.bias[n]) : 0.0f;
    const uint32_t part = smem_u32(smem) + (uint32_t)(quad * 32 + lane) * 4;
    for (int i = rank; i < NT && m0 + i < M; i += splits) {
      float y = 0.0f;
      for (int s = 0; s < splits; ++s) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                     : "=f"(v)
                     : "r"(map_to_rank(part + (uint32_t)i * TM * 4, (uint32_t)s))
                     : "memory");
        y += v;
      }
      if (ep.row_scale) y *= ep.row_scale[m0 + i];
      if (n < N) ep.out[(int64_t)(m0 + i) * ep.ldo + n] = __float2bfloat16_rn(fmaf(y, cs, b));
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

template <int FORMAT, bool PAIR>
int launch_many(const Operands& o, const Epilogue& ep, cudaStream_t stream) {
  using C = Tile<FORMAT, PAIR>;
  CUtensorMap ma, mb, msa, msb, mo{};
  int st;
  if ((st = code_map(&ma, o.a, o.M, o.K, TM)) || (st = code_map(&mb, o.b, o.N, o.K, C::kBRows)) ||
      (st = scale_map<FORMAT>(&msa, o.as, o.M, o.K, 1)) || (st = scale_map<FORMAT>(&msb, o.bs, o.N, o.K, 2)))
    return st;
  const int tma_out = ep.ldo % 8 == 0 && aligned(ep.out, 16);
  if (tma_out) {
    const cuuint64_t dims[2] = {(cuuint64_t)o.N, (cuuint64_t)o.M}, strides[1] = {(cuuint64_t)ep.ldo * 2};
    const cuuint32_t box[2] = {32, 32};
    if ((st = make_map(&mo, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ep.out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B)))
      return st;
  }
  static bool done[64] = {};
  if ((st = configure_smem(gemm_kernel<FORMAT, PAIR>, C::kSmem, done))) return st;
  constexpr int kRows = PAIR ? 2 * TM : TM;
  const int num_m = (o.M + kRows - 1) / kRows, num_n = (o.N + TN - 1) / TN;
  const int64_t tiles = (int64_t)num_m * num_n;
  const int workers = PAIR ? sm_count() / 2 : sm_count();
  const int grid = (PAIR ? 2 : 1) * (int)(tiles < workers ? tiles : workers);
  int64_t group = (24ll << 20) / ((int64_t)kRows * o.K / 2);  // 24 MB of A's codes
  if (group < 1) group = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {PAIR ? 2u : 1u, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, gemm_kernel<FORMAT, PAIR>, ma, mb, msa, msb, mo, o.M, o.N, o.K,
                     (int)(group < num_m ? group : num_m), tma_out, ep);
  return launch_status("fp4 gemm");
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
  const int tiles = ((o.N + TM - 1) / TM) * ((o.M + NT - 1) / NT);
  const int kblocks = (o.K / 2 + KB - 1) / KB;
  // as many slices as fill the GPU with two CTAs an SM and leave each two stages
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= 2 * sm_count() && kblocks >= 4 * splits) splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((o.N + TM - 1) / TM * splits), (unsigned)((o.M + NT - 1) / NT));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)splits, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, few_rows_kernel<FORMAT, NT>, mw, mx, msw, msx, o.M, o.N, o.K, splits, ep);
  return launch_status("fp4 gemm (few rows)");
}

template <int FORMAT>
int gemm(const Operands& o, const Epilogue& ep, cudaStream_t stream) {
  if (o.M <= 16) return launch_few<FORMAT, 16>(o, ep, stream);
  if (o.M <= 32) return launch_few<FORMAT, 32>(o, ep, stream);
  if (o.M <= 64) return launch_few<FORMAT, 64>(o, ep, stream);
  if (o.M <= kFewRows) return launch_few<FORMAT, 128>(o, ep, stream);
  return launch_many<FORMAT, true>(o, ep, stream);
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
