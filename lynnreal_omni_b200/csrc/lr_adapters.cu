// Low-rank adapters of many requests beside a shared projection:
//   out[t, :] = base[t, :] + scale[e] * up[e] (down[e] x[t, :]),  e = index[t]
// (e < 0: out[t, :] = base[t, :]), where base is the shared projection's output.
//
// Two kernels: shrink_kernel makes the few values down[e] x[t] of every token
// (fp32, in parts over the columns), expand_kernel adds up[e] times them to the
// base row. Both are bound by memory: per byte of x or base a rank of 16 to 128
// gives the tensor core 8 to 64 products, so mma.sync is fast enough, and its
// operands come straight from global memory, 16 bytes a load: a sum over columns
// does not mind their order, and neither do the outputs of a tile, so what a
// thread loads at once are the columns that it stands for. Nothing but the small
// inner rows passes through shared memory.
//
// Tokens are taken in tiles, whatever their adapters: for each adapter that
// occurs in a tile the rows of the others are zeros, and their sums are put back
// afterwards (an infinity in one request's row or adapter reaches no other).
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
  bf16* out;
  int64_t x_stride, base_stride, out_stride;
  int tokens, width, outputs, rank, count;
  int splits;    // parts of the columns
  int padded;    // columns of an inner row
  float* inner;  // [splits][tokens][padded]
};

constexpr int kWarps = 8;

// The adapters of a tile of up to 64 tokens, one after another, in every warp alike.
struct Groups {
  int id[2];  // of tokens lane and lane + 32; -1: none, or had already
  uint64_t none;

  __device__ __forceinline__ Groups(const Args& a, int first, int tile, int lane) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = lane + 32 * i;
      id[i] = at < tile && first + at < a.tokens ? a.index[first + at] : -1;
      bad |= id[i] >= a.count;
      if (id[i] >= a.count) id[i] = -1;
    }
    if (bad) atomicOr(&g_adapters_status, (unsigned)kDevErrAdapter);
    none = ~((uint64_t)__ballot_sync(0xffffffffu, id[0] >= 0) | (uint64_t)__ballot_sync(0xffffffffu, id[1] >= 0) << 32);
  }
  // The next adapter and the tokens that have it; false at the end.
  __device__ __forceinline__ bool next(int& adapter, uint64_t& members) {
    const unsigned b0 = __ballot_sync(0xffffffffu, id[0] >= 0), b1 = __ballot_sync(0xffffffffu, id[1] >= 0);
    if ((b0 | b1) == 0u) return false;
    adapter = b0 ? __shfl_sync(0xffffffffu, id[0], __ffs(b0) - 1) : __shfl_sync(0xffffffffu, id[1], __ffs(b1) - 1);
    members = (uint64_t)__ballot_sync(0xffffffffu, id[0] == adapter) |
              (uint64_t)__ballot_sync(0xffffffffu, id[1] == adapter) << 32;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (id[i] == adapter) id[i] = -1;
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

// ------------------------------------------------------------------ shrink
// MT tiles of 16 tokens, NR tiles of 8 rank rows. The warps of a block, and the
// blocks of a tile (blockIdx.y), each take a run of columns; the warps' sums are
// added in a fixed order, the blocks' by expand_kernel. Blocks of blockIdx.z take
// every gridDim.z-th adapter of the tile.
template <int MT, int NR>
__global__ void __launch_bounds__(32 * kWarps) shrink_kernel(const Args a) {
  constexpr int kRegs = MT * NR * 4;
  extern __shared__ float sums[];  // [kWarps / 2][kRegs][32]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int first = blockIdx.x * (16 * MT);
  tc::allow_dependent();
  Groups groups(a, first, 16 * MT, lane);
  const int steps = (a.width + 31) / 32;
  const int each = (steps + kWarps * a.splits - 1) / (kWarps * a.splits);
  const int k0 = min((int)(blockIdx.y * kWarps + warp) * each, steps) * 32, k1 = min(k0 + each * 32, a.width);

  int adapter;
  uint64_t members;
  for (int number = 0; groups.next(adapter, members); ++number) {
    if (number % gridDim.z != blockIdx.z) continue;
    float acc[MT][NR][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.0f;
    const bf16* down = a.down + (int64_t)adapter * a.rank * a.width;
#pragma unroll 2
    for (int k = k0 + 8 * t; k < k1 + 8 * t; k += 32) {
      const bool there = k < k1;
      uint4 w[NR], x[MT][2];
#pragma unroll
      for (int n = 0; n < NR; ++n) w[n] = load16(down + (int64_t)(8 * n + g) * a.width + k, there && 8 * n + g < a.rank);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = 16 * m + 8 * h + g;
          x[m][h] = load16(a.x + (int64_t)(first + row) * a.x_stride + k, there && (members >> row & 1));
        }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          mma_16816(acc[m][n], x[m][0].x, x[m][1].x, x[m][0].y, x[m][1].y, w[n].x, w[n].y);
          mma_16816(acc[m][n], x[m][0].z, x[m][1].z, x[m][0].w, x[m][1].w, w[n].z, w[n].w);
        }
    }
#pragma unroll
    for (int half = kWarps / 2; half >= 1; half /= 2) {
      __syncthreads();
      if (warp >= half && warp < 2 * half) {
        float* dst = sums + (warp - half) * kRegs * 32 + lane;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) dst[i * 32] = acc[i / (NR * 4)][i / 4 % NR][i % 4];
      }
      __syncthreads();
      if (warp < half) {
        const float* src = sums + warp * kRegs * 32 + lane;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) acc[i / (NR * 4)][i / 4 % NR][i % 4] += src[i * 32];
      }
    }
    if (warp == 0) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = 16 * m + 8 * h + g;
          if (!(members >> row & 1)) continue;
          float* dst = a.inner + ((int64_t)blockIdx.y * a.tokens + first + row) * a.padded + 2 * t;
#pragma unroll
          for (int n = 0; n < NR; ++n)
            if (8 * n < a.padded) *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(acc[m][n][2 * h], acc[m][n][2 * h + 1]);
        }
    }
  }
}

// ------------------------------------------------------------------ expand
// MT tiles of 16 tokens, 32 columns a warp, rank up to 16 KS. The base values
// are the products' accumulators. A thread's eight columns lie side by side:
// column n of the tile's i-th product stands for column 8 (n / 2) + 2 i + n % 2.
// The inner values, scaled, are rounded to bf16 for the product (2^-9 of the
// update, as every factor of it is rounded already); sums and base stay in fp32
// and are rounded once.
template <int MT, int KS, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) expand_kernel(const Args a) {
  constexpr int kPad = KS > 1 ? 16 * KS : 16;
  constexpr int kLine = kPad >= 64 ? kPad + 32 : kPad;  // rows side by side in different banks
  __shared__ __align__(16) bf16 inner[16 * MT * kLine];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int column_blocks = (a.outputs + 32 * kWarps - 1) / (32 * kWarps);
  const int first = (int)(blockIdx.x / column_blocks) * (16 * MT);
  const int column = (int)(blockIdx.x % column_blocks) * (32 * kWarps) + warp * 32;
  Groups groups(a, first, 16 * MT, lane);

  // The rows of this block: those of its adapters, and, in the first one, those of none.
  uint64_t owned = blockIdx.z == 0 ? groups.none : 0;
  {
    Groups all = groups;
    int adapter;
    uint64_t members;
    for (int number = 0; all.next(adapter, members); ++number)
      if (number % gridDim.z == blockIdx.z) owned |= members;
  }
  const int rows = min(16 * MT, a.tokens - first);
  if (rows < 64) owned &= (1ull << rows) - 1;
  if (owned == 0) {  // the same in every thread
    tc::wait_for_predecessor();
    return;
  }
  const int mine = column + 8 * t;
  float acc[MT][4][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 16 * m + 8 * h + g;
      const bf16* src = a.base + (int64_t)(first + row) * a.base_stride + mine;
      uint32_t y[4] = {0u, 0u, 0u, 0u};
      if (owned >> row & 1) {
        if (VEC) {
          if (mine < a.outputs) {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
          }
        } else {
          const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (mine + i < a.outputs) y[i / 2] |= (uint32_t)s[i] << (16 * (i % 2));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[m][i][2 * h] = bf_lo(y[i]);
        acc[m][i][2 * h + 1] = bf_hi(y[i]);
      }
    }
  bool waited = false;
  int adapter;
  uint64_t members;
  for (int number = 0; groups.next(adapter, members); ++number) {
    if (number % gridDim.z != blockIdx.z) continue;
    uint32_t up[4][KS][2];
    const bf16* weight = a.up + (int64_t)adapter * a.outputs * a.rank;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = column + 8 * (g >> 1) + 2 * i + (g & 1);
      const bf16* src = weight + (int64_t)n * a.rank;
      if (KS == 1) {
        const uint2 w = n < a.outputs && 4 * t < a.rank ? *reinterpret_cast<const uint2*>(src + 4 * t) : make_uint2(0u, 0u);
        up[i][0][0] = w.x, up[i][0][1] = w.y;
      } else {
#pragma unroll
        for (int s = 0; s < KS / 2; ++s) {
          const uint4 w = load16(src + 32 * s + 8 * t, n < a.outputs && 32 * s + 8 * t < a.rank);
          up[i][2 * s][0] = w.x, up[i][2 * s][1] = w.y;
          up[i][(2 * s + 1) % KS][0] = w.z, up[i][(2 * s + 1) % KS][1] = w.w;
        }
      }
    }
    if (!waited) {
      waited = true;
      tc::wait_for_predecessor();
      // The inner rows: parts added in order, scaled.
      for (int at = threadIdx.x; at < 16 * MT * (kPad / 4); at += 32 * kWarps) {
        const int row = at / (kPad / 4), c = at % (kPad / 4) * 4;
        const int token = first + row;
        uint2 packed = make_uint2(0u, 0u);
        int e = token < a.tokens ? a.index[token] : -1;
        if (e >= 0 && e < a.count && (owned >> row & 1) && c < a.rank) {
          float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const float* src = a.inner + (int64_t)token * a.padded + c;
          for (int s = 0; s < a.splits; ++s, src += (int64_t)a.tokens * a.padded) {
            const float4 part = __ldcg(reinterpret_cast<const float4*>(src));
            v[0] += part.x, v[1] += part.y, v[2] += part.z, v[3] += part.w;
          }
          const float scale = a.scale ? a.scale[e] : 1.0f;
          packed = make_uint2(cvt2(v[0] * scale, v[1] * scale), cvt2(v[2] * scale, v[3] * scale));
        }
        *reinterpret_cast<uint2*>(inner + row * kLine + c) = packed;
      }
      __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (!(members >> (16 * m) & 0xffff)) continue;
      float before[4][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) before[i / 4][i % 4] = acc[m][i / 4][i % 4];
      const bool lo = members >> (16 * m + g) & 1, hi = members >> (16 * m + 8 + g) & 1;
      const bf16 *r0 = inner + (16 * m + g) * kLine, *r1 = r0 + 8 * kLine;
      if (KS == 1) {
        uint2 h0 = *reinterpret_cast<const uint2*>(r0 + 4 * t), h1 = *reinterpret_cast<const uint2*>(r1 + 4 * t);
        if (!lo) h0 = make_uint2(0u, 0u);
        if (!hi) h1 = make_uint2(0u, 0u);
#pragma unroll
        for (int i = 0; i < 4; ++i) mma_16816(acc[m][i], h0.x, h1.x, h0.y, h1.y, up[i][0][0], up[i][0][1]);
      } else {
#pragma unroll
        for (int s = 0; s < KS / 2; ++s) {
          const uint4 h0 = load16(r0 + 32 * s + 8 * t, lo), h1 = load16(r1 + 32 * s + 8 * t, hi);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mma_16816(acc[m][i], h0.x, h1.x, h0.y, h1.y, up[i][2 * s][0], up[i][2 * s][1]);
            mma_16816(acc[m][i], h0.z, h1.z, h0.w, h1.w, up[i][(2 * s + 1) % KS][0], up[i][(2 * s + 1) % KS][1]);
          }
        }
      }
      // rows of other adapters stay as they were, whatever this one's values
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(e < 2 ? lo : hi)) acc[m][i][e] = before[i][e];
    }
  }
  if (!waited) tc::wait_for_predecessor();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 16 * m + 8 * h + g;
      if (!(owned >> row & 1)) continue;
      bf16* dst = a.out + (int64_t)(first + row) * a.out_stride + mine;
      if (VEC) {
        if (mine < a.outputs)
          *reinterpret_cast<uint4*>(dst) =
              make_uint4(cvt2(acc[m][0][2 * h], acc[m][0][2 * h + 1]), cvt2(acc[m][1][2 * h], acc[m][1][2 * h + 1]),
                         cvt2(acc[m][2][2 * h], acc[m][2][2 * h + 1]), cvt2(acc[m][3][2 * h], acc[m][3][2 * h + 1]));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (mine + i < a.outputs) dst[i] = __float2bfloat16_rn(acc[m][i / 2][2 * h + i % 2]);
      }
    }
}

// ------------------------------------------------------------------ host
struct Plan {
  bool few;  // tiles of 16 tokens, a block for each adapter of a tile
  int splits, padded;
  int64_t bytes;
};
Plan plan(int64_t tokens, int64_t width, int64_t rank) {
  Plan p{};
  p.few = tokens <= 512;
  p.padded = (int)((rank + 15) / 16 * 16);
  const int64_t tiles = p.few ? (tokens + 15) / 16 : (tokens + 63) / 64;
  int64_t splits = (2 * sm_count() + tiles - 1) / tiles;
  const int64_t most = (width + 64 * kWarps - 1) / (64 * kWarps);  // two steps a warp at least
  if (splits > most) splits = most;
  if (splits > 16) splits = 16;
  p.splits = (int)splits;
  p.bytes = splits * tokens * p.padded * 4;
  return p;
}

template <int MT, int NR>
int launch_shrink(const Args& a, unsigned groups, cudaStream_t stream) {
  constexpr size_t smem = kWarps / 2 * MT * NR * 4 * 32 * 4;
  static bool done[64] = {};
  if (smem > 48 * 1024) {
    const int st = tc::configure_smem(shrink_kernel<MT, NR>, smem, done);
    if (st) return st;
  }
  const dim3 grid((unsigned)((a.tokens + 16 * MT - 1) / (16 * MT)), (unsigned)a.splits, groups);
  shrink_kernel<MT, NR><<<grid, 32 * kWarps, smem, stream>>>(a);
  return launch_status("adapters (inner rows)");
}

template <int MT, int KS>
int launch_expand(const Args& a, unsigned groups, bool vec, cudaStream_t stream) {
  const int64_t blocks = (int64_t)((a.tokens + 16 * MT - 1) / (16 * MT)) * ((a.outputs + 32 * kWarps - 1) / (32 * kWarps));
  LR_REQUIRE(blocks <= INT32_MAX, "adapters: too many blocks");
  const dim3 grid((unsigned)blocks, 1, groups);
  return tc::launch("adapters (outputs)", vec ? expand_kernel<MT, KS, true> : expand_kernel<MT, KS, false>, grid, 32 * kWarps, 0,
                    stream, 1, true, a);
}

template <int MT_SHRINK, int NR, int MT_EXPAND>
int launch_both(const Args& a, unsigned groups, bool vec, cudaStream_t stream) {
  const int st = launch_shrink<MT_SHRINK, NR>(a, groups, stream);
  return st ? st : launch_expand<MT_EXPAND, (NR + 1) / 2>(a, groups, vec, stream);
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
  return lr::adapters::plan(tokens, width, rank).bytes;
}

extern "C" int lr_adapters(const void* x, int64_t x_stride, const void* base, int64_t base_stride, const void* down, const void* up,
                           const float* scale, const int32_t* index, int64_t tokens, int64_t width, int64_t outputs, int64_t rank,
                           int64_t adapters, void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lr;
  int st = check_adapters(tokens, width, outputs, rank, adapters);
  if (st) return st;
  if (tokens == 0) return LR_OK;
  LR_REQUIRE(x && base && down && up && index && out, "adapters: null pointer");
  LR_REQUIRE(x_stride >= 0 && base_stride >= 0 && out_stride >= outputs, "adapters: strides");
  if (x_stride % 8 || !aligned(x, 16) || !aligned(down, 16) || !aligned(up, 16))
    return set_error(LR_ERR_UNSUPPORTED, "adapters: x, down and up must be 16-byte aligned");
  const adapters::Plan p = adapters::plan(tokens, width, rank);
  LR_REQUIRE(workspace && workspace_bytes >= p.bytes && aligned(workspace, 16), "adapters: a workspace of %lld bytes is needed",
             (long long)p.bytes);
  const adapters::Args a{static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(base),
                         static_cast<const __nv_bfloat16*>(down), static_cast<const __nv_bfloat16*>(up), scale, index,
                         static_cast<__nv_bfloat16*>(out), x_stride, base_stride, out_stride, (int)tokens, (int)width,
                         (int)outputs, (int)rank, (int)adapters, p.splits, p.padded, static_cast<float*>(workspace)};
  const bool vec = outputs % 8 == 0 && base_stride % 8 == 0 && out_stride % 8 == 0 && aligned(base, 16) && aligned(out, 16);
  auto* s = static_cast<cudaStream_t>(stream);
  if (p.few) {
    const unsigned groups = (unsigned)(adapters < 16 ? adapters : 16);
    if (rank <= 16) return adapters::launch_both<1, 2, 1>(a, groups, vec, s);
    if (rank <= 32) return adapters::launch_both<1, 4, 1>(a, groups, vec, s);
    if (rank <= 64) return adapters::launch_both<1, 8, 1>(a, groups, vec, s);
    return adapters::launch_both<1, 16, 1>(a, groups, vec, s);
  }
  if (rank <= 16) return adapters::launch_both<4, 2, 4>(a, 1, vec, s);
  if (rank <= 32) return adapters::launch_both<4, 4, 4>(a, 1, vec, s);
  if (rank <= 64) return adapters::launch_both<2, 8, 4>(a, 1, vec, s);
  return adapters::launch_both<2, 16, 4>(a, 1, vec, s);
}
