// Rotary position embedding of queries and keys with tables computed on the fly.
//
// Token n at position p turns the pair (a, b) of rotary frequency f_i by the
// angle p f_i:  (a c - b s, b c + a s),  c = factor cos(p f_i), s = factor
// sin(p f_i). Pairs are (x_i, x_{i + R/2}) (half layout) or (x_2i, x_{2i+1})
// (interleaved); the columns from R on are copied.
//
// The angle of a far position is a large number of radians, of which fp32
// keeps few digits after the point. It is therefore formed in turns,
// p f / 2 pi, as an unevaluated sum of two floats: the whole turns fall away
// exactly and sincospi sees an argument within [-2, 2] that is right to about
// 1e-7, whatever the position.
//
// Bound by memory: every value is read and written once (4 bytes a value).
// Angles are computed once a token and kept in shared memory for all heads.
#include "lr_common.cuh"
#include "lr_host.h"

namespace lr {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kThreads = 256;

struct RopeArgs {
  const bf16* src[2];  // query, key
  bf16* dst[2];        // [tokens, heads, head_dim]
  int64_t token_stride[2], head_stride[2];
  int heads[2];
  const void* positions;
  int positions_64;
  const float* inv_freq;  // [rotary / 2], radians per position
  float factor;
  int tokens, head_dim, rotary;
};

__device__ __forceinline__ float fraction(float x) { return x - rintf(x); }  // exact

// (cos, sin) of p f, times the factor. f / 2 pi is held in three floats and p in
// two (p = ph + pl); every product is split into its rounded value and its
// exact error, and each part sheds its whole turns before they are added.
__device__ __forceinline__ float2 rotation(int64_t p, float f, float factor) {
  constexpr double kTurn = 0.15915494309189535;  // 1 / 2 pi = kHi + kMid + kLo
  constexpr float kHi = (float)kTurn, kMid = (float)(kTurn - (double)kHi);
  constexpr float kLo = (float)(kTurn - (double)kHi - (double)kMid) - 9.8393e-18f;  // 1 / 2 pi - kTurn
  const float fh = __fmul_rn(f, kHi), e1 = __fmaf_rn(f, kHi, -fh);
  const float m = __fmul_rn(f, kMid), e2 = __fmaf_rn(f, kMid, -m);
  const float fm = __fadd_rn(e1, m), bb = __fsub_rn(fm, e1);
  const float e3 = __fadd_rn(__fsub_rn(e1, __fsub_rn(fm, bb)), __fsub_rn(m, bb));
  const float fl = __fadd_rn(__fadd_rn(e3, e2), __fmul_rn(f, kLo));
  const float ph = (float)(p >> 12) * 4096.0f, pl = (float)(int)(p & 4095);  // exact for |p| < 2^36
  const float x = __fmul_rn(ph, fh), y = __fmul_rn(pl, fh), z = __fmul_rn(ph, fm);
  const float turns = (fraction(x) + fraction(y)) + fraction(__fmaf_rn(ph, fh, -x)) + fraction(z) +
                      (__fmaf_rn(pl, fh, -y) + __fmaf_rn(ph, fm, -z) + __fmul_rn(pl, fm) + __fmul_rn(ph, fl));
  float s, c;
  sincospif(2.0f * turns, &s, &c);
  return make_float2(c * factor, s * factor);
}

// Tokens blockIdx.x * tpb .. + tpb. VEC: eight values (16 bytes) an access.
// An item is one access of each half of the pairs (half layout) or one access
// (interleaved, copied columns).
template <bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeArgs a, int tpb) {
  extern __shared__ float2 turn[];  // [tpb][rotary / 2]
  const int half = a.rotary / 2;
  const int64_t token0 = (int64_t)blockIdx.x * tpb;
  const int here = (int)min((int64_t)tpb, a.tokens - token0);
  for (int i = threadIdx.x; i < here * half; i += kThreads) {
    const int64_t n = token0 + i / half;
    const int64_t p = a.positions_64 ? static_cast<const int64_t*>(a.positions)[n]
                                     : (int64_t) static_cast<const int32_t*>(a.positions)[n];
    turn[i] = rotation(p, a.inv_freq[i % half], a.factor);
  }
  __syncthreads();
  constexpr int W = VEC ? 8 : 1;
  const int rot_items = INTERLEAVED ? a.rotary / (VEC ? 8 : 2) : half / W;
  const int items = rot_items + (a.head_dim - a.rotary) / W;
  const int heads = a.heads[0] + a.heads[1];
  const int total = here * heads * items;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int row = i / items, item = i - row * items;
    const int t = row / heads, h = row - t * heads;
    const int which = h >= a.heads[0];
    const int head = which ? h - a.heads[0] : h;
    const bf16* src = a.src[which] + (token0 + t) * a.token_stride[which] + head * a.head_stride[which];
    bf16* dst = a.dst[which] + ((token0 + t) * a.heads[which] + head) * (int64_t)a.head_dim;
    const float2* tt = turn + t * half;
    if (item >= rot_items) {
      const int col = a.rotary + (item - rot_items) * W;
      if (VEC)
        *reinterpret_cast<uint4*>(dst + col) = ld_stream(src + col);
      else
        dst[col] = src[col];
    } else if (INTERLEAVED) {
      if (VEC) {
        float f[8];
        unpack8(ld_stream(src + item * 8), f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 r = tt[item * 4 + e];
          const float x = f[2 * e], y = f[2 * e + 1];
          f[2 * e] = x * r.x - y * r.y;
          f[2 * e + 1] = y * r.x + x * r.y;
        }
        *reinterpret_cast<uint4*>(dst + item * 8) = pack8(f);
      } else {
        const float2 r = tt[item];
        const float x = __bfloat162float(src[2 * item]), y = __bfloat162float(src[2 * item + 1]);
        dst[2 * item] = __float2bfloat16_rn(x * r.x - y * r.y);
        dst[2 * item + 1] = __float2bfloat16_rn(y * r.x + x * r.y);
      }
    } else {
      if (VEC) {
        float x[8], y[8];
        unpack8(ld_stream(src + item * 8), x);
        unpack8(ld_stream(src + half + item * 8), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 r = tt[item * 8 + e];
          const float u = x[e], v = y[e];
          x[e] = u * r.x - v * r.y;
          y[e] = v * r.x + u * r.y;
        }
        *reinterpret_cast<uint4*>(dst + item * 8) = pack8(x);
        *reinterpret_cast<uint4*>(dst + half + item * 8) = pack8(y);
      } else {
        const float2 r = tt[item];
        const float x = __bfloat162float(src[item]), y = __bfloat162float(src[half + item]);
        dst[item] = __float2bfloat16_rn(x * r.x - y * r.y);
        dst[half + item] = __float2bfloat16_rn(y * r.x + x * r.y);
      }
    }
  }
}

}  // namespace
}  // namespace lr

extern "C" int lr_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads, const void* k,
                       int64_t k_token_stride, int64_t k_head_stride, int64_t k_heads, const void* positions,
                       int positions_64, const float* inv_freq, float factor, int64_t tokens, int64_t head_dim,
                       int64_t rotary_dim, int interleaved, void* q_out, void* k_out, void* stream) {
  using namespace lr;
  LR_REQUIRE(tokens >= 0 && tokens <= INT32_MAX && q_heads >= 0 && k_heads >= 0 && q_heads + k_heads > 0 &&
                 q_heads + k_heads <= 65536 && head_dim > 0 && head_dim <= 4096,
             "rope: invalid shape");
  LR_REQUIRE(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
             "rope: rotary dimensions must be even and fit the head");
  if (tokens == 0) return LR_OK;
  LR_REQUIRE((q_heads == 0 || (q && q_out)) && (k_heads == 0 || (k && k_out)) && positions &&
                 (rotary_dim == 0 || inv_freq),
             "rope: null pointer");
  LR_REQUIRE(q_token_stride >= 0 && q_head_stride >= 0 && k_token_stride >= 0 && k_head_stride >= 0,
             "rope: negative strides");
  RopeArgs a{};
  a.src[0] = static_cast<const bf16*>(q);
  a.src[1] = static_cast<const bf16*>(k);
  a.dst[0] = static_cast<bf16*>(q_out);
  a.dst[1] = static_cast<bf16*>(k_out);
  a.token_stride[0] = q_token_stride, a.token_stride[1] = k_token_stride;
  a.head_stride[0] = q_head_stride, a.head_stride[1] = k_head_stride;
  a.heads[0] = (int)q_heads, a.heads[1] = (int)k_heads;
  a.positions = positions;
  a.positions_64 = positions_64;
  a.inv_freq = inv_freq;
  a.factor = factor;
  a.tokens = (int)tokens, a.head_dim = (int)head_dim, a.rotary = (int)rotary_dim;
  bool vec = head_dim % 8 == 0 && (interleaved ? rotary_dim % 8 == 0 : rotary_dim % 16 == 0);
  for (int w = 0; w < 2; ++w)
    if (a.heads[w])
      vec = vec && a.token_stride[w] % 8 == 0 && a.head_stride[w] % 8 == 0 && aligned(a.src[w], 16) &&
            aligned(a.dst[w], 16);
  // Four tokens a block share the launch of their angles (one angle a thread
  // at 128 columns); fewer while the blocks would not fill the GPU twice.
  const int tpb = tokens >= 8 * sm_count() && rotary_dim <= 1024 ? 4 : 1;
  const unsigned grid = (unsigned)((tokens + tpb - 1) / tpb);
  const size_t smem = (size_t)tpb * (rotary_dim / 2) * sizeof(float2);
  auto* st = static_cast<cudaStream_t>(stream);
  if (vec && interleaved)
    rope_kernel<true, true><<<grid, kThreads, smem, st>>>(a, tpb);
  else if (vec)
    rope_kernel<true, false><<<grid, kThreads, smem, st>>>(a, tpb);
  else if (interleaved)
    rope_kernel<false, true><<<grid, kThreads, smem, st>>>(a, tpb);
  else
    rope_kernel<false, false><<<grid, kThreads, smem, st>>>(a, tpb);
  return launch_status("rope");
}
