// Attention over the paged 8-bit cache.
//
//   x_j = scale * q . k_j + bias_j over the visible keys j,  out = sum_j e^(x_j - max) v_j / sum_j e^(x_j - max),
//   k_j = k_scale[block, head] * e4m3, v_j likewise
//
// A warp per (token, query head): a lane forms the score of one of 32 keys, then all lanes share the sum over the values.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math_constants.h>

#include <algorithm>

#include "fdma_internal.h"

namespace fdma {
namespace {

constexpr int kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  fdma_cache_attention_params p;
  int shift;
  float scale_log2;
};

__device__ __forceinline__ float e4m3_to_f(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}
template <typename T>
__device__ __forceinline__ float load_f(const void* p, int64_t i) {
  return static_cast<float>(static_cast<const T*>(p)[i]);
}
// In units of log2. The lowest finite number of a type stays finite, so that a row of nothing else is an average and not empty.
__device__ __forceinline__ float bias_log2(float b) {
  const float x = b * kLog2e;
  return fabsf(x) > 3.0e38f && fabsf(b) != CUDART_INF_F ? copysignf(3.0e38f, b) : x;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) attend_kernel(const AttnArgs a) {
  __shared__ float s_q[kThreads / 32][256];
  const fdma_cache_attention_params& p = a.p;
  const fdma_cache& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + warp;
  if (w >= static_cast<int64_t>(c.tokens) * p.h) return;
  const int t = static_cast<int>(w / p.h), h = static_cast<int>(w - static_cast<int64_t>(t) * p.h), hk = h / (p.h / c.h_k);
  T* out = static_cast<T*>(p.out) + t * p.out_row_stride + h * p.out_head_stride;
  int lo = 0, hi = c.requests;  // first request whose tokens end behind t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c.cu_seqlens[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  float o[8], m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.f;
  if (lo < c.requests && c.cu_chunks[lo + 1] > c.cu_chunks[lo]) {
    for (int i = lane; i < c.d; i += 32) s_q[warp][i] = load_f<T>(p.query, t * p.query_row_stride + h * p.query_head_stride + i) * a.scale_log2;
    __syncwarp();
    const int n = c.cu_seqlens[lo + 1] - c.cu_seqlens[lo], length = min(min(c.lengths[lo], p.max_seqlen_k), c.width << a.shift);
    const int newest = p.is_causal ? c.lengths[lo] - n + t - c.cu_seqlens[lo] : length;
    const int32_t* list = p.kept_pos ? p.kept_pos + lo * p.kept_batch_stride + hk * p.kept_head_stride : nullptr;
    int slots = length;
    if (list) slots = p.kept_count ? min(p.kept_count[lo * p.count_batch_stride + hk * p.count_head_stride], p.kept_capacity) : p.kept_capacity;
    const int hb = p.h_bias == p.h ? h : p.h_bias == c.h_k ? hk : 0;
    for (int base = 0; base < slots; base += 32) {
      const int slot = base + lane;
      int pos = slot < slots ? (list ? list[slot] : slot) : -1;
      if (pos < 0 || pos >= length || pos > newest) pos = -1;
      int block = pos < 0 ? -1 : c.table[static_cast<int64_t>(lo) * c.width + (pos >> a.shift)];
      if (block < 0 || block >= c.num_blocks) block = -1;
      float x = -CUDART_INF_F, vs = 0.f;
      int64_t row = 0;
      if (block >= 0) {
        const int64_t at = static_cast<int64_t>(block) * c.h_k + hk;
        row = ((at << a.shift) + (pos & ((1 << a.shift) - 1))) * c.d;
        const uint4* k = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(c.k) + row);
        float s = 0.f;
        for (int i = 0; i < c.d / 16; ++i) {
          const uint4 v = k[i];
          const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 16; ++j) s = fmaf(s_q[warp][16 * i + j], e4m3_to_f((words[j / 4] >> (8 * (j % 4))) & 0xFF), s);
        }
        x = s * c.k_scale[at];
        if (p.bias && pos < p.bias_keys) x += bias_log2(load_f<T>(p.bias, lo * p.bias_batch_stride + hb * p.bias_head_stride + pos));
        vs = c.v_scale[at];
      }
      float mx = x;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float m_new = fmaxf(m, mx), m_use = m_new == -CUDART_INF_F ? 0.f : m_new;
      const float corr = m == -CUDART_INF_F ? 0.f : exp2f(m - m_use);
      m = m_new;
      const float e = x == -CUDART_INF_F ? 0.f : exp2f(x - m_use);
      l = l * corr + e;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] *= corr;
      for (int j = 0; j < 32; ++j) {
        const float pj = __shfl_sync(0xffffffffu, e, j), vj = __shfl_sync(0xffffffffu, vs, j);
        const int bj = __shfl_sync(0xffffffffu, block, j);
        const int64_t rj = __shfl_sync(0xffffffffu, row, j);
        if (bj < 0) continue;
        const uint8_t* v = static_cast<const uint8_t*>(c.v) + rj;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i * 32 + lane < c.d) o[i] = fmaf(pj, vj * e4m3_to_f(v[i * 32 + lane]), o[i]);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 + lane < c.d) out[i * 32 + lane] = static_cast<T>(l == 0.f ? 0.f : o[i] / l);
}

}  // namespace

int check_cache(const fdma_cache& c);

}  // namespace fdma

using namespace fdma;

extern "C" size_t fdma_cache_attention_workspace_bytes(const fdma_cache_attention_params*) { return 0; }

extern "C" int fdma_cache_attention(const fdma_cache_attention_params* pp, void* stream) {
  if (!pp) return FDMA_ERR_BAD_ARG;
  const fdma_cache_attention_params& p = *pp;
  const int st = check_cache(p.c);
  if (st) return st;
  if (p.c.tokens == 0) return FDMA_OK;
  if (!p.query || !p.out || p.h <= 0 || p.h % p.c.h_k || p.max_seqlen_q < 0 || p.max_seqlen_k < 0) return FDMA_ERR_BAD_ARG;
  if (p.bias && ((p.h_bias != 1 && p.h_bias != p.c.h_k && p.h_bias != p.h) || p.bias_keys <= 0)) return FDMA_ERR_BAD_ARG;
  if (p.kept_pos && p.kept_capacity <= 0) return FDMA_ERR_BAD_ARG;
  if (p.dtype != FDMA_BF16 && p.dtype != FDMA_FP16) return FDMA_ERR_UNSUPPORTED;
  AttnArgs a;
  a.p = p;
  a.shift = p.c.block_size == 16 ? 4 : p.c.block_size == 32 ? 5 : p.c.block_size == 64 ? 6 : 7;
  a.scale_log2 = p.softmax_scale * kLog2e;
  const int64_t ctas = (static_cast<int64_t>(p.c.tokens) * p.h + 3) / 4;
  if (ctas > 0x7FFFFFFF) return FDMA_ERR_UNSUPPORTED;
  if (p.dtype == FDMA_BF16) attend_kernel<__nv_bfloat16><<<static_cast<unsigned>(ctas), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  else attend_kernel<__half><<<static_cast<unsigned>(ctas), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return static_cast<int>(cudaGetLastError());
}
