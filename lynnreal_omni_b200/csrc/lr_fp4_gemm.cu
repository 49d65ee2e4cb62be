// Product of two matrices of 4-bit floating-point rows:
//   out[m, n] = bf16( (sum_k A[m, k] B[n, k]) * row_scale[m] * col_scale[n] + bias[n] )
// with A, B the values of codes and block scales, accumulated in fp32.
#include "lr_fp4.cuh"
#include "lr_host.h"

namespace lr {
namespace fp4 {
namespace {

constexpr int T = 64, KT = 32;

template <int FORMAT>
__global__ void __launch_bounds__(256)
    gemm_kernel(const uint8_t* __restrict__ a, const uint8_t* __restrict__ as, const uint8_t* __restrict__ b,
                const uint8_t* __restrict__ bs, int M, int N, int K, const float* __restrict__ row_scale,
                const float* __restrict__ col_scale, const __nv_bfloat16* __restrict__ bias,
                __nv_bfloat16* __restrict__ out, int64_t ldo) {
  __shared__ float sa[KT][T + 1], sb[KT][T + 1];
  const int m0 = blockIdx.y * T, n0 = blockIdx.x * T;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t ctiles = (K / (FORMAT == kNv ? 16 : 32) + 3) / 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += KT) {
    // 64 rows x 4 groups of 8 columns each
    for (int side = 0; side < 2; ++side) {
      const int r = threadIdx.x / 4, g = threadIdx.x % 4;
      const int row = (side ? n0 : m0) + r;
      float f[8] = {};
      if (row < (side ? N : M)) {
        const int col = k0 + g * 8;
        unpack_e2m1(*reinterpret_cast<const uint32_t*>((side ? b : a) + (int64_t)row * (K / 2) + col / 2), f);
        const float s = scale_value<FORMAT>((side ? bs : as)[scale_offset(row, col / (FORMAT == kNv ? 16 : 32), ctiles)]);
        for (int e = 0; e < 8; ++e) f[e] *= s;
      }
      for (int e = 0; e < 8; ++e) (side ? sb : sa)[g * 8 + e][r] = f[e];
    }
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= M || n >= N) continue;
      float y = acc[i][j];
      if (row_scale) y *= row_scale[m];
      if (col_scale) y *= col_scale[n];
      if (bias) y += __bfloat162float(bias[n]);
      out[m * ldo + n] = __float2bfloat16_rn(y);
    }
}

}  // namespace
}  // namespace fp4
}  // namespace lr

extern "C" int lr_fp4_gemm(const void* a, const void* a_scales, const void* b, const void* b_scales, int64_t M,
                           int64_t N, int64_t K, int format, const float* row_scale, const float* col_scale,
                           const void* bias, void* out, int64_t ldo, void* stream) {
  using namespace lr;
  LR_REQUIRE(format == LR_FP4_NV || format == LR_FP4_MX, "fp4_gemm: unknown format %d", format);
  LR_REQUIRE(M >= 0 && N > 0 && K > 0 && M < (1ll << 31) - 512 && N < (1ll << 31) - 512 && K <= (1 << 30),
             "fp4_gemm: invalid shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (K % 32) return set_error(LR_ERR_UNSUPPORTED, "fp4_gemm: K must be a multiple of 32, got %lld", (long long)K);
  if (M == 0) return LR_OK;
  LR_REQUIRE(a && a_scales && b && b_scales && out, "fp4_gemm: null pointer");
  LR_REQUIRE(ldo >= N, "fp4_gemm: ldo %lld < N %lld", (long long)ldo, (long long)N);
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(a_scales, 16) || !aligned(b_scales, 16))
    return set_error(LR_ERR_UNSUPPORTED, "fp4_gemm: codes and scales must be 16-byte aligned");
  const dim3 grid((unsigned)((N + fp4::T - 1) / fp4::T), (unsigned)((M + fp4::T - 1) / fp4::T));
  LR_REQUIRE(grid.y <= 65535, "fp4_gemm: too many rows");
  auto* st = static_cast<cudaStream_t>(stream);
  const auto kernel = format == LR_FP4_NV ? fp4::gemm_kernel<fp4::kNv> : fp4::gemm_kernel<fp4::kMx>;
  kernel<<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(a_scales),
                               static_cast<const uint8_t*>(b), static_cast<const uint8_t*>(b_scales), (int)M, (int)N,
                               (int)K, row_scale, col_scale, static_cast<const __nv_bfloat16*>(bias),
                               static_cast<__nv_bfloat16*>(out), ldo);
  return launch_status("fp4 gemm");
}
