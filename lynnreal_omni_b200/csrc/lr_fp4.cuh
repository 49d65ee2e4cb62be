// Device helpers of the 4-bit floating-point formats: e2m1 codes (two a byte,
// the even column in the low nibble) under one scale a block.
//   nvfp4: blocks of 16 columns, e4m3 scales, one fp32 scale a row on top;
//   mxfp4: blocks of 32 columns, e8m0 scales (powers of two).
// Scales are stored in the order in which the tensor core reads them: tiles of
// 128 rows x 4 blocks, 512 bytes each, byte [row % 32][row / 32][block].
#pragma once

#include "lr_common.cuh"

namespace lr {
namespace fp4 {

enum Format : int { kNv = 0, kMx = 1 };

// Byte offset of the scale of (row, block) for `ctiles` tiles across a row.
__host__ __device__ __forceinline__ int64_t scale_offset(int64_t row, int64_t block, int64_t ctiles) {
  return ((row >> 7) * ctiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// Eight fp32 values -> eight e2m1 codes, nearest even, values beyond 6 -> 6.
__device__ __forceinline__ uint32_t pack_e2m1(const float (&f)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}

// Eight codes -> their values (exact in f16).
__device__ __forceinline__ void unpack_e2m1(uint32_t w, float (&f)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}"
        : "=f"(f[2 * i]), "=f"(f[2 * i + 1])
        : "r"(h[i]));
}

// fp32 -> e4m3 byte, nearest even, beyond 448 -> 448, NaN -> 0x7f.
__device__ __forceinline__ uint32_t to_e4m3(float x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(x));
  return r & 0xffu;
}
__device__ __forceinline__ float from_e4m3(uint32_t byte) {
  float f;
  asm("{\n\t.reg .b32 h;\n\t.reg .b16 l, u;\n\t"
      "cvt.rn.f16x2.e4m3x2 h, %1;\n\tmov.b32 {l, u}, h;\n\tcvt.f32.f16 %0, l;\n\t}"
      : "=f"(f)
      : "h"((uint16_t)byte));
  return f;
}
// e8m0 byte -> 2^(byte - 127); 255 is NaN.
__device__ __forceinline__ float from_e8m0(uint32_t byte) {
  return byte == 0 ? __uint_as_float(0x00400000u) : byte == 255 ? __uint_as_float(0x7fc00000u)
                                                                : __uint_as_float(byte << 23);
}

template <int FORMAT>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return FORMAT == kNv ? from_e4m3(byte) : from_e8m0(byte);
}

}  // namespace fp4
}  // namespace lr
