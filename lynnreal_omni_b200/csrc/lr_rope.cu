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
// exactly and what is left, below about 2 turns, is right to about 1e-7 of a turn;
// sincospi's argument is twice that (below 4, right to 2e-7), whatever the position.
//
// Bound by memory: every value is read and written once (4 bytes a value).
// Angles are computed once a token and kept in shared memory for all heads. 16384
// tokens of 32 + 8 heads x 128 take 51 us in either layout, the floor at the
// measured copy rate (51.3 us); with 16-byte accesses 66 us, with the angles of
// a head's items in the same banks 65 us (half layout).
#include "lr_common.cuh"
#include "lr_host.h"

namespace lr {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kMaxThreads = 512;

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

// W columns as they lie in memory.
template <int W>
struct Columns {
  uint4 v[W / 8];
};
template <>
struct Columns<1> {
  uint16_t v;
};
__device__ __forceinline__ Columns<16> load(const bf16* p, Columns<16>) {
  Columns<16> c;
  asm volatile("ld.global.cs.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(c.v[0].x), "=r"(c.v[0].y), "=r"(c.v[0].z), "=r"(c.v[0].w), "=r"(c.v[1].x), "=r"(c.v[1].y),
                 "=r"(c.v[1].z), "=r"(c.v[1].w)
               : "l"(p));
  return c;
}
__device__ __forceinline__ Columns<8> load(const bf16* p, Columns<8>) { return {{ld_stream(p)}}; }
__device__ __forceinline__ Columns<1> load(const bf16* p, Columns<1>) { return {*reinterpret_cast<const uint16_t*>(p)}; }
__device__ __forceinline__ void store(bf16* p, const Columns<16>& c) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(c.v[0].x), "r"(c.v[0].y),
               "r"(c.v[0].z), "r"(c.v[0].w), "r"(c.v[1].x), "r"(c.v[1].y), "r"(c.v[1].z), "r"(c.v[1].w)
               : "memory");
}
__device__ __forceinline__ void store(bf16* p, const Columns<8>& c) { *reinterpret_cast<uint4*>(p) = c.v[0]; }
__device__ __forceinline__ void store(bf16* p, const Columns<1>& c) { *reinterpret_cast<uint16_t*>(p) = c.v; }

// Place of angle n: 16 bytes stay free behind each 16 angles, so that the items of a head, 64 or 128 bytes of angles
// apart, read from different banks.
__host__ __device__ __forceinline__ int padded(int n) { return n + (n >> 4) * 2; }

// (a, b) turned by r.
__device__ __forceinline__ void turn_pair(float& a, float& b, float2 r) {
  const float u = a, v = b;
  a = u * r.x - v * r.y;
  b = v * r.x + u * r.y;
}

// TPB consecutive tokens. An item is what one thread moves of one head: W
// columns (16 in 32-byte accesses, 8, or 1) of each half of the pairs (half
// layout), W columns of pairs side by side (interleaved; 2 where W is 1), or W
// copied columns. Rotated
// items come first, so that few warps hold both kinds; a thread keeps its item
// over the block's tokens and has all their loads under way before the first
// product, and the first ones before the angles.
template <int W, bool INTERLEAVED, int TPB>
__global__ void __launch_bounds__(kMaxThreads) rope_kernel(const RopeArgs a) {
  extern __shared__ float2 turn[];  // [TPB][padded(rotary / 2)]
  using V = Columns<W>;
  const int half = a.rotary / 2, row = padded(half);
  const int64_t token0 = (int64_t)blockIdx.x * TPB;
  const int here = (int)min((int64_t)TPB, a.tokens - token0);
  const int heads = a.heads[0] + a.heads[1];
  constexpr int kStep = INTERLEAVED && W == 1 ? 2 : W;  // columns from one item to the next
  const int rot_items = (INTERLEAVED ? a.rotary : half) / kStep, copy_items = (a.head_dim - a.rotary) / W;
  const int rotated = heads * rot_items, total = rotated + heads * copy_items;

  bool first = true;
  for (int i = threadIdx.x; first || i < total; i += blockDim.x) {
    const bool any = i < total, turned = i < rotated;
    const int j = turned ? i : i - rotated, per = turned ? rot_items : copy_items;
    int h = any ? j / per : 0;
    const int item = any ? j - h * per : 0;
    const int which = h >= a.heads[0];
    h -= which ? a.heads[0] : 0;
    const int col = turned ? item * kStep : a.rotary + item * W;
    const int second = INTERLEAVED ? 1 : half;  // column distance of a pair, where a thread loads both apart
    const int64_t src_stride = which ? a.token_stride[1] : a.token_stride[0];
    const int64_t dst_stride = (int64_t)(which ? a.heads[1] : a.heads[0]) * a.head_dim;
    const bf16* src = (which ? a.src[1] : a.src[0]) + token0 * src_stride + h * (which ? a.head_stride[1] : a.head_stride[0]) + col;
    bf16* dst = (which ? a.dst[1] : a.dst[0]) + token0 * dst_stride + h * (int64_t)a.head_dim + col;
    const bool two = turned && !(INTERLEAVED && W > 1);
    V x[TPB], y[TPB];
#pragma unroll
    for (int t = 0; t < TPB; ++t)
      if (any && t < here) {
        x[t] = load(src + t * src_stride, V{});
        if (two) y[t] = load(src + t * src_stride + second, V{});
      }
    if (first) {
      for (int n = threadIdx.x; n < here * half; n += blockDim.x) {
        const int64_t at = token0 + n / half;
        const int64_t p = a.positions_64 ? static_cast<const int64_t*>(a.positions)[at]
                                         : (int64_t) static_cast<const int32_t*>(a.positions)[at];
        turn[n / half * row + padded(n % half)] = rotation(p, a.inv_freq[n % half], a.factor);
      }
      __syncthreads();
      first = false;
      if (!any) break;
    }
#pragma unroll
    for (int t = 0; t < TPB; ++t) {
      if (t >= here) break;
      bf16* to = dst + t * dst_stride;
      if constexpr (W > 1) {
        if (turned) {
          // angles of the item: W / 2 (interleaved) or W of them
          const float4* r4 = reinterpret_cast<const float4*>(turn + t * row + padded(item * (INTERLEAVED ? W / 2 : W)));
#pragma unroll
          for (int q = 0; q < W / 8; ++q) {
            float u[8], v[8];
            unpack8(x[t].v[q], u);
            if (!INTERLEAVED) unpack8(y[t].v[q], v);
#pragma unroll
            for (int e = 0; e < (INTERLEAVED ? 4 : 8); e += 2) {
              const float4 r = r4[(q * (INTERLEAVED ? 4 : 8) + e) / 2];
              if (INTERLEAVED) {
                turn_pair(u[2 * e], u[2 * e + 1], make_float2(r.x, r.y));
                turn_pair(u[2 * e + 2], u[2 * e + 3], make_float2(r.z, r.w));
              } else {
                turn_pair(u[e], v[e], make_float2(r.x, r.y));
                turn_pair(u[e + 1], v[e + 1], make_float2(r.z, r.w));
              }
            }
            x[t].v[q] = pack8(u);
            if (!INTERLEAVED) y[t].v[q] = pack8(v);
          }
          if (!INTERLEAVED) store(to + half, y[t]);
        }
        store(to, x[t]);
      } else {
        if (turned) {
          float u = bf_bits(x[t].v), v = bf_bits(y[t].v);
          turn_pair(u, v, turn[t * row + padded(item)]);
          x[t].v = f2bf_bits(u);
          y[t].v = f2bf_bits(v);
          store(to + second, y[t]);
        }
        store(to, x[t]);
      }
    }
  }
}

template <int W, bool INTERLEAVED>
int launch_rope(const RopeArgs& a, cudaStream_t stream) {
  // As many tokens a block as keep two accesses of each under way for all (interleaved: 51.4 us at 16384 tokens against
  // 52.5 with two and 58.1 with one), where the blocks fill the GPU and their angles fit.
  constexpr int kMany = INTERLEAVED ? 4 : 2;
  const int tpb = a.tokens >= 8 * sm_count() && a.rotary <= 1024 ? kMany : 1;
  const int64_t items = (int64_t)(a.heads[0] + a.heads[1]) * (a.head_dim / W);
  const int64_t threads = (items / (a.rotary > 0 && !(W > 1 && INTERLEAVED) ? 2 : 1) + 31) / 32 * 32;
  const unsigned block = (unsigned)(threads < 128 ? 128 : threads > kMaxThreads ? kMaxThreads : threads);
  const size_t smem = (size_t)tpb * padded(a.rotary / 2) * sizeof(float2);
  if (tpb == kMany)
    rope_kernel<W, INTERLEAVED, kMany><<<(unsigned)((a.tokens + kMany - 1) / kMany), block, smem, stream>>>(a);
  else
    rope_kernel<W, INTERLEAVED, 1><<<(unsigned)a.tokens, block, smem, stream>>>(a);
  return launch_status("rope");
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
  // The widest access that divides the head, the rotary part and every row's start.
  auto fits = [&](int64_t w) {
    bool ok = head_dim % w == 0 && rotary_dim % (interleaved ? w : 2 * w) == 0;
    for (int i = 0; i < 2; ++i)
      if (a.heads[i])
        ok = ok && a.token_stride[i] % w == 0 && a.head_stride[i] % w == 0 && aligned(a.src[i], 2 * w) && aligned(a.dst[i], 2 * w);
    return ok;
  };
  auto* st = static_cast<cudaStream_t>(stream);
  if (fits(16)) return interleaved ? launch_rope<16, true>(a, st) : launch_rope<16, false>(a, st);
  if (fits(8)) return interleaved ? launch_rope<8, true>(a, st) : launch_rope<8, false>(a, st);
  return interleaved ? launch_rope<1, true>(a, st) : launch_rope<1, false>(a, st);
}
