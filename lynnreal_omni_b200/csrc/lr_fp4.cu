// Quantisation of bf16 rows to 4-bit floating point, and back.
//
// nvfp4, row r, blocks b of 16 columns:
//   A = max(max_k |x_k|, 1e-8),  row scale s = A / 2688           (2688 = 6 * 448)
//   e_b = e4m3(448 max_{k in b} |x_k| / A),  code = e2m1(x_k * (2688 / (e_b A)))
// so that x ~ code * e_b * s with the row's largest block at e4m3's largest
// scale. The two quotients are IEEE divisions, one a block: 448 max and e_b A
// are short numbers, so ties between two codes mostly come out as ties.
// mxfp4, blocks of 32 columns: e = floor(log2(max |x|)) - 2 (2 = the largest
// exponent of e2m1), code = e2m1(x 2^-e); the exponent is read off the bits.
// Both round to the nearest code, ties to even, and saturate at 6. A row
// (nvfp4) or block (mxfp4) that holds an infinity or a NaN gets a NaN scale, so
// that a product with it is NaN and not a number that looks right.
//
// Bound by memory: 2 bytes in, 0.5 + 1/16 (1/32) bytes out a value; a row's
// values stay in registers between the pass for A and the rounding. A thread
// holds units of 16 columns, consecutive units in consecutive threads (32-byte
// loads, 8-byte stores); the two halves of an mxfp4 block are two lanes. Rows of
// up to 1024 columns take a warp, up to 6144 a block of 128, longer ones of 512
// threads, so that a thread holds at most three units. 12240 x 6144 nvfp4: 30 us,
// 6.4 TB/s, 0.98 of the measured copy rate; back 31 us.
#include "lr_fp4.cuh"
#include "lr_host.h"
#include "lr_tc.cuh"

namespace lr {
namespace fp4 {
namespace {

using bf16 = __nv_bfloat16;

struct Unit {
  uint4 lo, hi;
};

__device__ __forceinline__ Unit load_unit(const bf16* p) { return {ld_stream(p), ld_stream(p + 8)}; }

// Largest magnitude of a unit as bf16 bits, NaN kept.
__device__ __forceinline__ float unit_absmax(const Unit& u) {
  const uint32_t w[8] = {u.lo.x, u.lo.y, u.lo.z, u.lo.w, u.hi.x, u.hi.y, u.hi.z, u.hi.w};
  __nv_bfloat162 m = as_bf2(w[0] & 0x7fff7fffu);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, as_bf2(w[i] & 0x7fff7fffu));
  const __nv_bfloat16 r = __hmax_nan(__low2bfloat16(m), __high2bfloat16(m));
  return __bfloat162float(r);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ uint2 encode_unit(const Unit& u, float factor) {
  float f[8];
  uint2 r;
  unpack8(u.lo, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __fmul_rn(f[e], factor);
  r.x = pack_e2m1(f);
  unpack8(u.hi, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __fmul_rn(f[e], factor);
  r.y = pack_e2m1(f);
  return r;
}

// Scale byte and the factor that takes values to code units, of one nvfp4 block.
__device__ __forceinline__ float nv_factor(float block_max, float row_max, uint32_t& byte) {
  // rows beyond 2^110 are scaled down by a power of two, so that 448 max and e A stay finite
  const float g = row_max > 0x1p110f ? 0x1p-20f : 1.0f;
  const float a = __fmul_rn(row_max, g);
  byte = to_e4m3(__fdiv_rn(__fmul_rn(__fmul_rn(block_max, g), 448.0f), a));
  const float e = from_e4m3(byte);
  return e == 0.0f ? 0.0f : __fmul_rn(__fdiv_rn(2688.0f, __fmul_rn(e, a)), g);
}
__device__ __forceinline__ float mx_factor(float block_max, uint32_t& byte) {
  const uint32_t ex = __float_as_uint(block_max) >> 23;
  byte = ex == 255u ? 255u : (uint32_t)max((int)ex - 2, 0);
  return __uint_as_float((254u - min(byte, 253u)) << 23);  // 2^(127 - byte)
}

// TPR threads a row, NB units a thread (columns past TPR * NB * 16 are read
// again in a second pass when NB == 0). One row a TPR-thread group.
template <int FORMAT, int TPR, int NB>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
    quantize_kernel(const bf16* __restrict__ x, int rows, int width, int64_t row_stride, uint8_t* __restrict__ codes,
                    uint8_t* __restrict__ scales, float* __restrict__ row_scales) {
  constexpr int kThreads = TPR < 128 ? 128 : TPR;
  __shared__ float red[kThreads / 32];
  const int t = threadIdx.x % TPR;
  const int row = blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
  // A product that follows may set itself up: at once beside a grid that leaves room (two blocks on each of the 148 SMs),
  // else when this one ends.
  const bool early = gridDim.x <= 296;
  if (early) tc::allow_dependent();
  const bool live = row < rows;
  const int units = width / 16;
  const int blocks = FORMAT == kNv ? units : units / 2;
  const int64_t ctiles = (blocks + 3) / 4;
  const bf16* src = x + (int64_t)(live ? row : 0) * row_stride;
  constexpr int N = NB > 0 ? NB : 1;
  const int passes = NB > 0 ? 1 : (units + TPR - 1) / TPR;

  Unit u[N];
  float row_max = 0.0f;
  if (NB > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int unit = i * TPR + t;
      u[i] = live && unit < units ? load_unit(src + unit * 16) : Unit{};
    }
    if (FORMAT == kNv) {
#pragma unroll
      for (int i = 0; i < N; ++i) row_max = max_nan(row_max, unit_absmax(u[i]));
    }
  } else if (FORMAT == kNv && live) {
    for (int unit = t; unit < units; unit += TPR) row_max = max_nan(row_max, unit_absmax(load_unit(src + (int64_t)unit * 16)));
  }
  if (FORMAT == kNv) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) row_max = max_nan(row_max, __shfl_xor_sync(0xffffffffu, row_max, off));
    if (TPR > 32) {
      if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = row_max;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < TPR / 32; ++w) row_max = max_nan(row_max, red[w]);
    }
    row_max = row_max < 1.0e-8f ? 1.0e-8f : row_max;  // keeps NaN
    if (live && t == 0) row_scales[row] = __fmul_rn(row_max, (float)(1.0 / 2688.0));
  }
  for (int pass = 0; pass < passes; ++pass) {
    if (NB == 0) {
      const int unit = pass * TPR + t;
      u[0] = live && unit < units ? load_unit(src + (int64_t)unit * 16) : Unit{};
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int unit = (NB > 0 ? i : pass) * TPR + t;
      float m = unit_absmax(u[i]);
      uint32_t byte;
      float factor;
      if (FORMAT == kNv) {
        factor = nv_factor(m, row_max, byte);
      } else {
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
        factor = mx_factor(m, byte);
      }
      if (live && unit < units) {
        *reinterpret_cast<uint2*>(codes + (int64_t)row * (width / 2) + unit * 8) = encode_unit(u[i], factor);
        if (FORMAT == kNv)
          scales[scale_offset(row, unit, ctiles)] = (uint8_t)byte;
        else if ((unit & 1) == 0)
          scales[scale_offset(row, unit / 2, ctiles)] = (uint8_t)byte;
      }
    }
  }
  if (!early) tc::allow_dependent();
  // zeros in the last tile's blocks past the row (they meet zero codes)
  if (live && t < (int)(ctiles * 4 - blocks)) scales[scale_offset(row, blocks + t, ctiles)] = 0;
}

// A warp a row and kUnits units a lane, 32 apart; a block eight rows, whose scales
// lie in the same 32-byte sectors.
constexpr int kUnits = 2;
template <int FORMAT, bool WIDE>
__global__ void __launch_bounds__(256)
    dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                      const float* __restrict__ row_scales, int rows, int width, bf16* __restrict__ out) {
  const int units = width / 16, lane = threadIdx.x & 31;
  const int64_t ctiles = ((FORMAT == kNv ? units : units / 2) + 3) / 4;
  const int unit0 = blockIdx.x * (32 * kUnits) + lane;
  for (int64_t row = (int64_t)blockIdx.y * 8 + (threadIdx.x >> 5); row < rows; row += (int64_t)gridDim.y * 8) {
    uint2 c[kUnits];
    uint32_t byte[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int unit = unit0 + 32 * i;
      if (unit < units) {
        c[i] = __ldcs(reinterpret_cast<const uint2*>(codes + row * (width / 2) + unit * 8));
        byte[i] = scales[scale_offset(row, FORMAT == kNv ? unit : unit / 2, ctiles)];
      }
    }
    const float rs = row_scales != nullptr ? row_scales[row] : 1.0f;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int unit = unit0 + 32 * i;
      if (unit >= units) break;
      const float s = __fmul_rn(scale_value<FORMAT>(byte[i]), rs);
      float lo[8], hi[8];
      unpack_e2m1(c[i].x, lo);
      unpack_e2m1(c[i].y, hi);
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[e] = __fmul_rn(lo[e], s), hi[e] = __fmul_rn(hi[e], s);
      const uint4 u = pack8(lo), v = pack8(hi);
      bf16* dst = out + row * width + unit * 16;
      if (WIDE) {
        asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(u.x), "r"(u.y), "r"(u.z),
                     "r"(u.w), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                     : "memory");
      } else {
        reinterpret_cast<uint4*>(dst)[0] = u;
        reinterpret_cast<uint4*>(dst)[1] = v;
      }
    }
  }
}

template <int FORMAT, int TPR, int NB>
int launch_quantize(const bf16* x, int rows, int width, int64_t stride, uint8_t* codes, uint8_t* scales, float* rs,
                    cudaStream_t st) {
  constexpr int per = TPR < 128 ? 128 / TPR : 1;
  quantize_kernel<FORMAT, TPR, NB><<<(rows + per - 1) / per, TPR < 128 ? 128 : TPR, 0, st>>>(x, rows, width, stride,
                                                                                            codes, scales, rs);
  return launch_status("fp4 quantize");
}

template <int FORMAT>
int quantize(const bf16* x, int rows, int width, int64_t stride, uint8_t* codes, uint8_t* scales, float* rs,
             cudaStream_t st) {
  const int units = width / 16;
  if (units <= 32) return launch_quantize<FORMAT, 32, 1>(x, rows, width, stride, codes, scales, rs, st);
  if (units <= 64) return launch_quantize<FORMAT, 32, 2>(x, rows, width, stride, codes, scales, rs, st);
  if (units <= 128) return launch_quantize<FORMAT, 128, 1>(x, rows, width, stride, codes, scales, rs, st);
  if (units <= 256) return launch_quantize<FORMAT, 128, 2>(x, rows, width, stride, codes, scales, rs, st);
  if (units <= 384) return launch_quantize<FORMAT, 128, 3>(x, rows, width, stride, codes, scales, rs, st);
  if (units <= 512) return launch_quantize<FORMAT, 512, 1>(x, rows, width, stride, codes, scales, rs, st);
  if (units <= 1024) return launch_quantize<FORMAT, 512, 2>(x, rows, width, stride, codes, scales, rs, st);
  if (units <= 1536) return launch_quantize<FORMAT, 512, 3>(x, rows, width, stride, codes, scales, rs, st);
  return launch_quantize<FORMAT, 512, 0>(x, rows, width, stride, codes, scales, rs, st);
}

int check_rows(const char* who, int64_t rows, int64_t width, int format) {
  LR_REQUIRE(format == LR_FP4_NV || format == LR_FP4_MX, "%s: unknown format %d", who, format);
  LR_REQUIRE(rows >= 0 && rows <= INT32_MAX - 512 && width > 0 && width <= (1 << 30), "%s: invalid shape %lld x %lld",
             who, (long long)rows, (long long)width);
  if (width % 32)
    return set_error(LR_ERR_UNSUPPORTED, "%s: the width must be a multiple of 32, got %lld", who, (long long)width);
  return LR_OK;
}

}  // namespace
}  // namespace fp4
}  // namespace lr

extern "C" int lr_fp4_quantize_rows(const void* x, int64_t rows, int64_t width, int64_t row_stride, int format,
                                    void* codes, void* scales, float* row_scales, void* stream) {
  using namespace lr;
  int st = fp4::check_rows("fp4_quantize_rows", rows, width, format);
  if (st) return st;
  if (rows == 0) return LR_OK;
  LR_REQUIRE(x && codes && scales && (format == LR_FP4_MX || row_scales), "fp4_quantize_rows: null pointer");
  LR_REQUIRE(rows == 1 || row_stride >= width, "fp4_quantize_rows: row stride %lld smaller than the width",
             (long long)row_stride);
  if (!aligned(x, 16) || (rows > 1 && row_stride % 8) || !aligned(codes, 16))
    return set_error(LR_ERR_UNSUPPORTED, "fp4_quantize_rows: rows must start on 16-byte boundaries");
  auto* s = static_cast<cudaStream_t>(stream);
  auto* src = static_cast<const __nv_bfloat16*>(x);
  auto* c = static_cast<uint8_t*>(codes);
  auto* sc = static_cast<uint8_t*>(scales);
  if (format == LR_FP4_NV) return fp4::quantize<fp4::kNv>(src, (int)rows, (int)width, row_stride, c, sc, row_scales, s);
  return fp4::quantize<fp4::kMx>(src, (int)rows, (int)width, row_stride, c, sc, row_scales, s);
}

extern "C" int lr_fp4_dequantize_rows(const void* codes, const void* scales, const float* row_scales, int64_t rows,
                                      int64_t width, int format, void* out, void* stream) {
  using namespace lr;
  int st = fp4::check_rows("fp4_dequantize_rows", rows, width, format);
  if (st) return st;
  if (rows == 0) return LR_OK;
  LR_REQUIRE(codes && scales && out, "fp4_dequantize_rows: null pointer");
  if (!aligned(codes, 16) || !aligned(out, 16))
    return set_error(LR_ERR_UNSUPPORTED, "fp4_dequantize_rows: rows must start on 16-byte boundaries");
  const int64_t blocks = (rows + 7) / 8;
  const dim3 grid((unsigned)((width / 16 + 32 * fp4::kUnits - 1) / (32 * fp4::kUnits)), (unsigned)(blocks < 65535 ? blocks : 65535));
  const auto kernel = format == LR_FP4_NV ? aligned(out, 32) ? fp4::dequantize_kernel<fp4::kNv, true>
                                                             : fp4::dequantize_kernel<fp4::kNv, false>
                      : aligned(out, 32)  ? fp4::dequantize_kernel<fp4::kMx, true>
                                          : fp4::dequantize_kernel<fp4::kMx, false>;
  kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), row_scales, (int)rows, (int)width,
      static_cast<__nv_bfloat16*>(out));
  return launch_status("fp4 dequantize");
}
