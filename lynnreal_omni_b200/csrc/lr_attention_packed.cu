// Attention over packed sequences of different lengths, causal or full, with
// query heads sharing key/value heads in groups:
//   out[i, h, :] = sum_j softmax_j(scale * q[i, h, :] . k[j, h / group, :]) v[j, h / group, :]
// over the keys j of query i's own sequence (causal: the queries are the last
// ones of their sequence, and query i of Lq sees keys j <= i + Lk - Lq).
#include "lr_common.cuh"
#include "lr_host.h"

namespace lr {

static __device__ unsigned int g_packed_status = 0;

namespace packed {
namespace {

using bf16 = __nv_bfloat16;

struct Args {
  const bf16 *q, *k, *v;
  bf16* out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const int32_t *cu_q, *cu_k;
  int seqs, total_q, total_k, group, heads, causal;
  float scale_log2;
};

// Raise the status bit unless both offset arrays start at 0, never go down and
// end within their tensors (the threads of one block look at all of them).
__device__ void check_offsets(const Args& a) {
  bool bad = false;
  for (int i = threadIdx.x; i <= a.seqs; i += blockDim.x) {
    const int q = a.cu_q[i], k = a.cu_k[i];
    bad |= q < (i ? a.cu_q[i - 1] : 0) || k < (i ? a.cu_k[i - 1] : 0) || q > a.total_q || k > a.total_k;
    bad |= i == 0 && (q | k) != 0;
  }
  if (bad) atomicOr(&g_packed_status, (unsigned)kDevErrOffsets);
}

// One warp a query token and head; a lane holds D / 32 columns.
template <int D>
__global__ void __launch_bounds__(128) attention_kernel(const Args a) {
  constexpr int E = D / 32;
  if (blockIdx.x == 0) check_offsets(a);
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (item >= (int64_t)a.total_q * a.heads) return;
  const int tok = (int)(item / a.heads), h = (int)(item % a.heads);
  int lo = 0, hi = a.seqs;  // the last sequence that starts at or before the token
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.cu_q[mid] <= tok) lo = mid; else hi = mid;
  }
  float o[E] = {}, q[E];
  float m = -INFINITY, l = 0.0f;
  const int q1 = min(a.cu_q[lo + 1], a.total_q);
  if (tok >= a.cu_q[lo] && tok < q1) {
    const int k0 = max(a.cu_k[lo], 0), k1 = min(a.cu_k[lo + 1], a.total_k);
    const int last = a.causal ? k1 - (q1 - tok) : k1 - 1;
    for (int e = 0; e < E; ++e) q[e] = __bfloat162float(a.q[tok * a.q_ts + h * a.q_hs + lane * E + e]);
    for (int j = k0; j <= last; ++j) {
      float s = 0.0f;
      for (int e = 0; e < E; ++e)
        s = fmaf(q[e], __bfloat162float(a.k[j * a.k_ts + (h / a.group) * a.k_hs + lane * E + e]), s);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      s *= a.scale_log2;
      const float mn = fmaxf(m, s), alpha = exp2f(m - mn), p = exp2f(s - mn);
      l = l * alpha + p;
      for (int e = 0; e < E; ++e)
        o[e] = o[e] * alpha + p * __bfloat162float(a.v[j * a.v_ts + (h / a.group) * a.v_hs + lane * E + e]);
      m = mn;
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  for (int e = 0; e < E; ++e) a.out[item * D + lane * E + e] = __float2bfloat16_rn(o[e] * inv);
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

extern "C" int lr_attention_packed(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                   int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                   int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_q,
                                   const int32_t* cu_k, int64_t seqs, int64_t total_q, int64_t total_k, int64_t heads,
                                   int64_t kv_heads, int64_t head_dim, int causal, float scale, void* out,
                                   void* stream) {
  using namespace lr;
  LR_REQUIRE(seqs > 0 && total_q >= 0 && total_k >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
             "attention_packed: invalid shape");
  if (head_dim != 64 && head_dim != 128)
    return set_error(LR_ERR_UNSUPPORTED, "attention_packed: head_dim %lld (64 or 128)", (long long)head_dim);
  if (total_q == 0) return LR_OK;
  LR_REQUIRE(q && out && cu_q && cu_k && (total_k == 0 || (k && v)), "attention_packed: null pointer");
  packed::Args a{static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(k),
                 static_cast<const __nv_bfloat16*>(v), static_cast<__nv_bfloat16*>(out), q_token_stride, q_head_stride,
                 k_token_stride, k_head_stride, v_token_stride, v_head_stride, cu_q, cu_k, (int)seqs, (int)total_q,
                 (int)total_k, (int)(heads / kv_heads), (int)heads, causal, (float)((double)scale * 1.4426950408889634)};
  const unsigned grid = (unsigned)((total_q * heads + 3) / 4);
  auto* st = static_cast<cudaStream_t>(stream);
  if (head_dim == 64)
    packed::attention_kernel<64><<<grid, 128, 0, st>>>(a);
  else
    packed::attention_kernel<128><<<grid, 128, 0, st>>>(a);
  return launch_status("attention_packed");
}
