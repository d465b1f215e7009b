// Attention of prompt parts over the paged 8-bit cache: requests with many new tokens at once.
//
// Tensor-bound: with n queries per key the keys are worth converting once. One kernel turns the requests' blocks into 16-bit keys and
// values, packed request after request; the packed-sequence forward kernel does the rest with tcgen05. The conversion is
// memory-bound, 6 d bytes per key and kv head (read 2 d, write 4 d). 8-bit numbers times a power of two are exact in bf16. In fp16 they
// are rounded to multiples of 2^-24 where they are that small, which is no coarser than fp16 keys and values are before they
// enter the cache. What fp16 cannot hold is left to the other kernel (PromptFound): the rows are then computed again from the 8 bits. So
// are NaN in values: in the forward kernel one of them reaches the queries of its tile that do not see it. (In a key it does not: scores
// are masked, not multiplied by 0.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cstddef>

#include "fdma_internal.h"

namespace fdma {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 64;
constexpr int kMostRequests = 8192;
constexpr int64_t kMostRows = 1 << 20;               // keys of all requests, what the forward kernel's tables hold
constexpr int64_t kMostBytes = int64_t{1} << 32;     // of scratch

// What the conversion comes upon. In fp16, V scales may be up to 2^8 apart: the forward kernel's probabilities are fp16 then, multiples
// of 2^-24 when small, and values that such a probability meets must not be large beside those of the likely keys (scales 2^8 apart
// add up to 2^-11 of a result over 64 large keys, 2^16 apart 2^-3).
struct PromptFound {
  int32_t again;               // not 0: the rows are to be computed from the 8 bits
  uint32_t largest, smallest;  // bits of the V scales, the latter inverted
};
constexpr int kMostApart = 8;

struct UnpackArgs {
  fdma_cache c;
  int32_t* cu_k;
  PromptFound* found;  // zeros before
  void *k, *v;  // (rows, h_k, d)
  int shift, max_keys, max_queries, rows, heads;
};

template <bool kBf16>
__device__ __forceinline__ uint32_t pack_scaled(uint16_t two, float scale) {
  const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3));
  float2 f = __half22float2(h);
  f.x *= scale;
  f.y *= scale;
  if (kBf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ bool has_nan(uint2 x) {
  return ((((x.x & 0x7F7F7F7Fu) + 0x01010101u) | ((x.y & 0x7F7F7F7Fu) + 0x01010101u)) & 0x80808080u) != 0;
}
// Whether eight 8-bit numbers times the scale are in fp16's range.
__device__ __forceinline__ bool fits_fp16(uint2 x, float scale) {
  bool fits = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t two = static_cast<uint16_t>((i < 2 ? x.x : x.y) >> (16 * (i & 1)));
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
    fits &= fabsf(f.x * scale) <= 65504.f && fabsf(f.y * scale) <= 65504.f;
  }
  return fits;
}

// A CTA converts a 64-key chunk of a request, all heads of K and V, at a time. 2 x 16 048 keys, 8 heads, d = 128 (197 MB): 42 us, of which
// a plain copy would take 31; the rest is the start, the sums over the requests and the look-up of the blocks.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const __grid_constant__ UnpackArgs a) {
  extern __shared__ int s_pre[];  // chunks, then rows, of the requests before
  __shared__ long long s_warp[kThreads / 32], s_pairs[kThreads / 32];
  __shared__ int s_block[4], s_longest[kThreads / 32];
  __shared__ uint32_t s_scales[2];
  __shared__ bool s_beyond;  // a request is beyond the caller's bounds, which this path does not cut as the other one does: none are converted
  const fdma_cache& c = a.c;
  const int R = c.requests, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int *pre_chunks = s_pre, *pre_rows = s_pre + R + 1;
  long long carry = 0, pairs = 0;  // carry: rows << 32 | chunks; pairs: of a new token and a key, see prompt_pays
  int longest = 0;
  if (tid == 0) s_beyond = false;
  __syncthreads();
  for (int base = 0; base < R; base += kThreads) {
    const int r = base + tid;
    long long x = 0;
    long long my_pairs = 0;
    int my_length = 0;
    if (r < R && c.cu_chunks[r + 1] > c.cu_chunks[r] && c.cu_seqlens[r + 1] - c.cu_seqlens[r] >= kPromptTokens) {
      const int n = max(0, min(min(c.lengths[r], a.max_keys), c.width << a.shift));
      x = (static_cast<long long>(n) << 32) | ((n + kChunk - 1) / kChunk);
      my_length = n;
      const int queries = c.cu_seqlens[r + 1] - c.cu_seqlens[r];
      my_pairs = static_cast<long long>(n + kTileKeys) * queries;
      if (c.lengths[r] > a.max_keys || queries > a.max_queries) s_beyond = true;
    }
    my_length = __reduce_max_sync(0xffffffffu, my_length);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) my_pairs += __shfl_xor_sync(0xffffffffu, my_pairs, o);
    if (lane == 0) {
      s_pairs[warp] = my_pairs;
      s_longest[warp] = my_length;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    long long before = carry;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) before += s_warp[i];
      carry += s_warp[i];
      pairs += s_pairs[i];
      longest = max(longest, s_longest[i]);
    }
    x += before;
    if (r < R) {
      pre_chunks[r + 1] = static_cast<int>(x & 0xFFFFFFFF);
      pre_rows[r + 1] = static_cast<int>(min(x >> 32, static_cast<long long>(a.rows)));
    }
    __syncthreads();
  }
  if (tid == 0) pre_chunks[0] = pre_rows[0] = 0;
  __syncthreads();
  const int total_rows = pre_rows[R];
  const bool taken = total_rows > 0 && !s_beyond && prompt_pays(pairs * a.heads, longest, c.d);
  if (blockIdx.x == 0)
    for (int r = tid; r <= R; r += kThreads) a.cu_k[r] = taken ? pre_rows[r] : 0;
  const int total = taken ? pre_chunks[R] : 0;
  bool fits = true;
  uint32_t largest = 0, smallest = 0;  // bits of V scales, the latter inverted
  // A thread keeps its eight columns and walks rows, and heads within a row: the loads of eight do not wait for one another.
  const int pieces = c.d / 8, row_step = kThreads / pieces, my_row = tid / pieces, column = (tid - my_row * pieces) * 8;
  for (int w = blockIdx.x; w < total; w += gridDim.x) {
    int lo = 0, hi = R - 1;  // first request whose chunks end behind w
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (pre_chunks[mid + 1] > w) hi = mid;
      else lo = mid + 1;
    }
    const int pos0 = (w - pre_chunks[lo]) * kChunk, row0 = pre_rows[lo] + pos0, n = min(kChunk, pre_rows[lo + 1] - row0);
    if (tid < 4) {
      const int pos = pos0 + tid * 16;
      int block = tid * 16 < n ? c.table[static_cast<int64_t>(lo) * c.width + (pos >> a.shift)] : -1;
      s_block[tid] = block >= c.num_blocks ? -1 : block;
    }
    __syncthreads();
    for (int row = my_row < row_step ? my_row : n; row < n; row += row_step) {
      const int block = s_block[row >> 4], place = (pos0 + row) & ((1 << a.shift) - 1);
      const int64_t to = static_cast<int64_t>(row0 + row) * c.h_k * c.d + column, at = static_cast<int64_t>(block) * c.h_k;
      const int64_t from = ((at << a.shift) + place) * c.d + column, head_step = static_cast<int64_t>(c.d) << a.shift;
#pragma unroll 4
      for (int head = 0; head < c.h_k; ++head) {
        uint4 y[2] = {};
        if (block >= 0) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(v ? c.v : c.k) + from + head * head_step));
            const float scale = __ldg((v ? c.v_scale : c.k_scale) + at + head);
            fits &= !(v && has_nan(x)) && scale <= 0x1p119f;
            if (!kBf16 && scale > 65504.f / 448.f) fits &= fits_fp16(x, scale);
            if (!kBf16 && v && scale > 0x1p-100f) {
              largest = max(largest, __float_as_uint(scale));
              smallest = max(smallest, ~__float_as_uint(scale));
            }
            y[v] = make_uint4(pack_scaled<kBf16>(static_cast<uint16_t>(x.x), scale), pack_scaled<kBf16>(static_cast<uint16_t>(x.x >> 16), scale),
                              pack_scaled<kBf16>(static_cast<uint16_t>(x.y), scale), pack_scaled<kBf16>(static_cast<uint16_t>(x.y >> 16), scale));
          }
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(v ? a.v : a.k) + to + head * c.d) = y[v];
      }
    }
    __syncthreads();
  }
  if (!fits || (!taken && blockIdx.x == 0 && tid == 0)) atomicOr(&a.found->again, 1);
  if (!kBf16 && total > 0) {
    if (tid == 0) s_scales[0] = s_scales[1] = 0;
    __syncthreads();
    largest = __reduce_max_sync(0xffffffffu, largest);
    smallest = __reduce_max_sync(0xffffffffu, smallest);
    if (lane == 0) {
      atomicMax(&s_scales[0], largest);
      atomicMax(&s_scales[1], smallest);
    }
    __syncthreads();
    if (tid == 0) {  // of two CTAs whose scales are too far apart, the one that looks later sees both
      atomicMax(&a.found->largest, s_scales[0]);
      atomicMax(&a.found->smallest, s_scales[1]);
      __threadfence();
      const uint32_t high = atomicMax(&a.found->largest, 0u), low = ~atomicMax(&a.found->smallest, 0u);
      if (static_cast<int>(high >> 23) - static_cast<int>(low >> 23) > kMostApart) atomicOr(&a.found->again, 1);
    }
  }
}

// At most so many keys: requests that have kPromptTokens new ones each, of the longest length.
int64_t most_rows(const fdma_cache_attention_params& p) {
  const int64_t requests = std::min<int64_t>(p.c.requests, p.c.tokens / kPromptTokens);
  return requests * std::min<int64_t>(p.max_seqlen_k, static_cast<int64_t>(p.c.width) * p.c.block_size);
}
struct Scratch {
  size_t v, lse, found, cu_k, total;
};
Scratch scratch(const fdma_cache_attention_params& p) {
  Scratch s;
  const size_t kv = align256(static_cast<size_t>(most_rows(p)) * p.c.h_k * p.c.d * 2);
  s.v = kv;
  s.lse = 2 * kv;
  s.found = s.lse + align256(static_cast<size_t>(p.h) * p.c.tokens * sizeof(float));
  s.cu_k = s.found + align256(sizeof(PromptFound));
  s.total = s.cu_k + align256((static_cast<size_t>(p.c.requests) + 1) * sizeof(int32_t));
  return s;
}
fdma_fwd_params forward_params(const fdma_cache_attention_params& p, char* ws) {
  const Scratch s = scratch(p);
  fdma_fwd_params f = {};
  f.q = p.query;
  f.k = ws;
  f.v = ws + s.v;
  f.out = p.out;
  f.lse = reinterpret_cast<float*>(ws + s.lse);
  f.q_row_stride = p.query_row_stride; f.q_head_stride = p.query_head_stride;
  f.k_row_stride = f.v_row_stride = static_cast<int64_t>(p.c.h_k) * p.c.d;
  f.k_head_stride = f.v_head_stride = p.c.d;
  f.o_row_stride = p.out_row_stride; f.o_head_stride = p.out_head_stride;
  f.b = 1;
  f.seqlen_q = p.c.tokens;
  f.seqlen_k = static_cast<int32_t>(most_rows(p));
  f.h = p.h; f.h_k = p.c.h_k; f.h_mask = f.h_bias = 1; f.d = p.c.d;
  f.dtype = p.dtype;
  f.is_causal = p.is_causal;
  f.softmax_scale = p.softmax_scale;
  return f;
}

}  // namespace

bool cache_prompt_taken(const fdma_cache_attention_params& p) {
  if (std::min(p.max_seqlen_q, p.c.tokens) < kPromptTokens || p.bias || p.kept_pos || p.c.requests > kMostRequests) return false;
  const int64_t keys = std::min<int64_t>(p.max_seqlen_k, static_cast<int64_t>(p.c.width) * p.c.block_size);
  if (!prompt_pays(static_cast<int64_t>(p.c.tokens) * p.h * (keys + kTileKeys), keys, p.c.d)) return false;
  const int64_t rows = most_rows(p);
  if (rows <= 0 || rows > kMostRows || scratch(p).total > static_cast<size_t>(kMostBytes)) return false;
  if (p.c.tokens > (1 << 19)) return false;
  // the workspace is 256-byte aligned wherever it lies
  return tc_fwd_supported(forward_params(p, reinterpret_cast<char*>(uintptr_t{256})));
}
size_t cache_prompt_workspace_bytes(const fdma_cache_attention_params& p) { return scratch(p).total; }
size_t cache_prompt_again(const fdma_cache_attention_params& p) { return scratch(p).found + offsetof(PromptFound, again); }

int cache_prompt(const fdma_cache_attention_params& p, int shift, void* workspace, cudaStream_t stream) {
  char* ws = static_cast<char*>(workspace);
  const Scratch s = scratch(p);
  UnpackArgs a;
  a.c = p.c;
  a.cu_k = reinterpret_cast<int32_t*>(ws + s.cu_k);
  a.found = reinterpret_cast<PromptFound*>(ws + s.found);
  a.k = ws;
  a.v = ws + s.v;
  a.shift = shift;
  a.max_keys = p.max_seqlen_k;
  a.max_queries = p.max_seqlen_q;
  a.rows = static_cast<int>(most_rows(p));
  a.heads = p.h;
  const size_t smem = (static_cast<size_t>(p.c.requests) + 1) * 8;
  const bool bf16 = p.dtype == FDMA_BF16;
  if (smem > 40 * 1024) {
    static std::atomic<uint64_t> prepared[2] = {};
    const void* kern = bf16 ? reinterpret_cast<const void*>(unpack_kernel<true>) : reinterpret_cast<const void*>(unpack_kernel<false>);
    const int st = allow_smem_once(kern, (kMostRequests + 1) * 8, prepared[bf16]);
    if (st) return st;
  }
  const int64_t most_chunks = a.rows / kChunk + std::min<int64_t>(p.c.requests, p.c.tokens / kPromptTokens);
  const int ctas = static_cast<int>(std::min<int64_t>(most_chunks, 8 * sm_count()));
  cudaError_t e = cudaMemsetAsync(a.found, 0, sizeof(PromptFound), stream);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (bf16) unpack_kernel<true><<<ctas, kThreads, smem, stream>>>(a);
  else unpack_kernel<false><<<ctas, kThreads, smem, stream>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  return tc_fwd(forward_params(p, ws), stream, PackedSeqs{p.c.cu_seqlens, a.cu_k, p.c.requests});
}

}  // namespace fdma
