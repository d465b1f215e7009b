// The paged 8-bit cache: block tables and slot maps from request lengths, and the writer of keys and values.
#include <cuda_fp8.h>

#include "fdma_internal.h"
#include "fdma_rotary.cuh"

namespace fdma {
namespace {

// ---- block tables -----------------------------------------------------------------------------------------------
// Whole numbers and a few kilobytes: the time is that of a launch and of a chain of dependent loads. So extending is ONE launch.
// Every CTA sums up the lengths of all requests itself (one scan over up to 1024 of them at a time) and then fills
// its share of the tokens; what other CTAs still read (lengths, the free list's count) is updated by the CTA that arrives last.
constexpr int kTableThreads = 1024;
constexpr int kMaxRequests = 8192;

// Inclusive scan of K numbers per thread over the CTA, and their totals. s_warp: K * 33 words; ends with all threads past their
// reads of it.
template <int K>
__device__ __forceinline__ void scan(long long (&x)[K], long long (&total)[K], long long* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long y = __shfl_up_sync(0xffffffffu, x[k], o);
      if (lane >= o) x[k] += y;
    }
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < K; ++k) s_warp[k * 33 + warp] = x[k];
  __syncthreads();
  if (warp < K) {  // a warp each
    long long w = lane < warps ? s_warp[warp * 33 + lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    s_warp[warp * 33 + lane] = w;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (warp > 0) x[k] += s_warp[k * 33 + warp - 1];
    total[k] = s_warp[k * 33 + 31];
  }
  __syncthreads();
}

__device__ __forceinline__ int ceil_div(long long x, int shift) { return static_cast<int>((x + (1ll << shift) - 1) >> shift); }

__global__ void __launch_bounds__(kTableThreads) extend_kernel(const fdma_tables_params p, const int shift) {
  // per request: end of its tokens; tokens held before; place of its first new block among the step's (-1: refused)
  extern __shared__ int32_t s_req[];
  __shared__ long long s_warp[3 * 33];
  __shared__ bool s_last;
  int32_t *s_end = s_req, *s_have = s_req + p.requests, *s_first = s_req + 2 * p.requests;
  const int tid = threadIdx.x, threads = blockDim.x;
  const int R = p.requests;
  const int n_free = max(0, min(*p.free_count, p.num_blocks));
  const bool lead = blockIdx.x == 0;
  long long tokens = 0, blocks = 0, units = 0;  // sums over the requests before; units: chunks << 32 | touched blocks
  long long taken = 0;                          // blocks that leave the free list
  for (int base = 0; base < R; base += threads) {
    const int r = base + tid;
    const bool in = r < R;
    const int have = in ? max(0, p.lengths[r]) : 0, n = in ? max(0, p.new_lengths[r]) : 0;
    const long long length = static_cast<long long>(have) + n;
    const long long old = ceil_div(have, shift), want = (length + (1ll << shift) - 1) >> shift;
    const bool fits = n > 0 && want <= p.width;
    int need = fits ? static_cast<int>(want - old) : 0;
    const long long work = (static_cast<long long>(ceil_div(length, 6)) << 32) | static_cast<int>(want - (have >> shift));
    // all sums at once, as if tokens and blocks were enough; where they are not, one after the other
    long long x[3] = {n, need, fits ? work : 0}, sum[3];
    scan(x, sum, s_warp);
    long long end = tokens + x[0], upto = blocks + x[1], both = units + x[2];
    bool granted = n == 0 || fits;
    if (tokens + sum[0] > p.tokens || blocks + sum[1] > n_free) {
      const bool may = fits && end <= p.tokens;
      need = may ? need : 0;
      long long y[1] = {need}, t[1];
      scan(y, t, s_warp);
      upto = blocks + y[0];
      sum[1] = t[0];
      granted = n == 0 || (may && (need == 0 || upto <= n_free));
      long long z[2] = {granted && n > 0 ? work : 0, granted ? need : 0}, u[2];
      scan(z, u, s_warp);
      both = units + z[0];
      sum[2] = u[0];
      taken += u[1];
    } else {
      taken += sum[1];
    }
    tokens += sum[0];
    blocks += sum[1];
    units += sum[2];
    if (in) {
      const int e = static_cast<int>(min(end, static_cast<long long>(p.tokens)));
      s_end[r] = e;
      s_have[r] = have;
      s_first[r] = granted ? static_cast<int>(upto - need) : -1;
      if (lead) {
        p.cu_seqlens[r + 1] = e;
        p.lengths_after[r] = granted ? static_cast<int>(length) : have;
        p.granted[r] = granted ? 1 : 0;
        p.cu_blocks[r + 1] = static_cast<int>(both & 0xFFFFFFFF);
        p.cu_chunks[r + 1] = static_cast<int>(both >> 32);
        if (r == 0) p.cu_seqlens[0] = p.cu_blocks[0] = p.cu_chunks[0] = 0;
      }
    }
  }
  __syncthreads();
  const int mask = (1 << shift) - 1;
  const int last_end = s_end[R - 1];
  for (int t = blockIdx.x * threads + tid; t < p.tokens; t += gridDim.x * threads) {
    int pos = 0;
    int64_t slot = -1;
    if (t < last_end) {
      int lo = 0, hi = R - 1;  // first request whose tokens end behind t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_end[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int start = lo ? s_end[lo - 1] : 0, have = s_have[lo], first = s_first[lo];
      pos = have + t - start;
      if (first >= 0) {
        const int page = pos >> shift, old = ceil_div(have, shift);
        int32_t* entry = p.table + static_cast<int64_t>(lo) * p.width + page;
        const int block = page < old ? *entry : p.free_list[n_free - 1 - (first + page - old)];
        // a new block's first token enters it (nobody reads that entry in this launch)
        if (page >= old && (t == start || (pos & mask) == 0)) *entry = block;
        if (block >= 0) slot = (static_cast<int64_t>(block) << shift) + (pos & mask);
      }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
  // the last CTA: nobody reads lengths and free_count any more
  if (gridDim.x > 1) {
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      s_last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
    }
    __syncthreads();
    if (!s_last) return;
  } else {
    __syncthreads();
  }
  for (int r = tid; r < R; r += threads)
    if (s_first[r] >= 0) p.lengths[r] = s_have[r] + s_end[r] - (r ? s_end[r - 1] : 0);
  if (tid == 0) {
    *p.free_count = n_free - static_cast<int>(taken);
    *p.ticket = 0;
  }
}

__global__ void __launch_bounds__(kTableThreads) truncate_kernel(const fdma_tables_params p, const int shift) {
  extern __shared__ int32_t s_req[];  // per request: blocks kept, place of its first freed block
  __shared__ long long s_warp[33];
  const int threads = blockDim.x;
  int32_t *s_keep = s_req, *s_first = s_req + p.requests;
  const int tid = threadIdx.x, R = p.requests;
  const int n_free = max(0, min(*p.free_count, p.num_blocks));
  long long gone = 0;
  for (int base = 0; base < R; base += threads) {
    const int r = base + tid;
    const int have = r < R ? max(0, p.lengths[r]) : 0, keep = r < R ? min(have, max(0, p.new_lengths[r])) : 0;
    const int held = min(ceil_div(have, shift), p.width), left = min(ceil_div(keep, shift), p.width);
    long long x[1] = {held - left}, sum[1];
    scan(x, sum, s_warp);
    const long long upto = gone + x[0];
    gone += sum[0];
    if (r < R) {
      s_keep[r] = left;
      s_first[r] = static_cast<int>(upto - (held - left));
      p.lengths[r] = keep;
    }
  }
  __syncthreads();
  const long long total = n_free + gone;
  for (int i = tid; i < gone; i += threads) {
    int below = 0, above = R - 1;  // last request whose first freed block is no later: it has freed this one
    while (below < above) {
      const int mid = (below + above + 1) >> 1;
      if (s_first[mid] <= i) below = mid;
      else above = mid - 1;
    }
    int32_t* entry = p.table + static_cast<int64_t>(below) * p.width + s_keep[below] + i - s_first[below];
    const long long at = total - 1 - i;
    if (at < p.num_blocks) p.free_list[at] = *entry;
    *entry = -1;
  }
  if (tid == 0) *p.free_count = static_cast<int>(min(total, static_cast<long long>(p.num_blocks)));
}

int block_shift(int block_size) {
  switch (block_size) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    default: return -1;
  }
}

int check_tables(const fdma_tables_params* p) {
  if (!p || !p->table || !p->lengths || !p->free_list || !p->free_count || !p->ticket || !p->new_lengths) return FDMA_ERR_BAD_ARG;
  if (p->requests < 0 || p->width <= 0 || p->num_blocks <= 0 || p->tokens < 0) return FDMA_ERR_BAD_ARG;
  const int shift = block_shift(p->block_size);
  if (shift < 0 || p->requests > kMaxRequests) return FDMA_ERR_UNSUPPORTED;
  if ((static_cast<int64_t>(p->width) << shift) > 0x7FFFFFFF || (static_cast<int64_t>(p->requests) * p->width << shift >> 6) > 0x7FFFFFFF)
    return FDMA_ERR_UNSUPPORTED;
  return 0;
}

// a thread per request in whole warps, at least as many warps as there are sums
int table_threads(int64_t n) { return static_cast<int>(std::min<int64_t>(kTableThreads, std::max<int64_t>(128, (n + 31) / 32 * 32))); }

template <typename K>
int table_smem(K kernel, int requests, std::atomic<uint64_t>& prepared, size_t* bytes) {
  *bytes = static_cast<size_t>(requests) * 12;
  return *bytes <= 40 * 1024 ? 0 : allow_smem_once(reinterpret_cast<const void*>(kernel), kMaxRequests * 12, prepared);
}

// ---- the writer ---------------------------------------------------------------------------------------------------
// Memory-bound by its bytes: keys and values are read twice (the second time from cache) and written once. A CTA takes one block and a
// few kv heads of K or of V: head by head it looks for the largest magnitude, fixes the scale and writes. It waits for loads and at
// the barrier between the two passes most of the time, so CTAs that turn queries are spread among those.
// 6 prompts of up to 2700 tokens (8 300 in all), 32 + 8 heads, d = 128 (176 MB): 49 us; without the queries 29, the queries alone 28.
constexpr int kAppendThreads = kRotaryWarps * 32;
constexpr int kAppendCtas = 4;  // per SM
constexpr int kMaxBlock = 128, kMaxDim = 256;  // tokens of a block, head dimension
struct AppendArgs {
  fdma_cache_append_params p;
  RotaryUnits key_units;    // of keys that are turned
  RotaryUnits plain_units;  // of values, and keys that are not: two vectors, half a row apart
  RotaryArgs query;
  int shift, most_units;
  int heads;  // of K or V that a CTA writes, one after the other
  int64_t cache_ctas;
};

// N numbers times f, rounded; beyond 448 they become 448
template <int N>
__device__ __forceinline__ Vec<uint8_t, N> to_e4m3(const float (&x)[N], float f) {
  Vec<uint8_t, N> v;
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int j = 0; j < N; j += 2)
      *reinterpret_cast<uint16_t*>(&v.x[j]) = __nv_cvt_float2_to_fp8x2(make_float2(x[j] * f, x[j + 1] * f), __NV_SATFINITE, __NV_E4M3);
  } else {
    v.x[0] = __nv_cvt_float_to_fp8(x[0] * f, __NV_SATFINITE, __NV_E4M3);
  }
  return v;
}
__device__ __forceinline__ uint8_t to_e4m3(float x) { return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float from_e4m3(uint8_t x) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3)));
}

// 2^e, e the smallest (from -100 on) with x <= 448 * 2^e: x and 448 = 1.75 * 2^8 by exponent and mantissa
__device__ __forceinline__ float block_scale(float x) {
  const uint32_t u = __float_as_uint(x);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7FFFFF) > 0x600000 ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, -100) + 127) << 23);
}

template <typename T, int N, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) append_kernel(const __grid_constant__ AppendArgs a) {
  extern __shared__ __align__(16) float2 s_factors[];  // of the block's new tokens, or rotate_tokens' own
  __shared__ float s_max[2][kAppendThreads / 32];
  __shared__ int s_found[5];
  const fdma_cache_append_params& p = a.p;
  const fdma_cache& c = p.c;
  const int tid = threadIdx.x;
  // the CTAs that write and those that turn queries are spread over the launch evenly: the former wait for loads most of the time
  const int64_t before_me = blockIdx.x * a.cache_ctas / gridDim.x;
  if ((blockIdx.x + int64_t{1}) * a.cache_ctas / gridDim.x == before_me) {
    const int warp = tid >> 5;
    rotate_tokens<T, N, kInterleaved>(a.query, (blockIdx.x - before_me) * kRotaryWarps + warp, s_factors + warp * rotary_warp_pairs<N>(a.query));
    return;
  }
  // K of a block's next few heads, or V
  const int id = static_cast<int>(before_me), groups = (c.h_k + a.heads - 1) / a.heads;
  const bool is_v = id & 1;
  const int unit = (id >> 1) / groups, head0 = ((id >> 1) - unit * groups) * a.heads, head_end = min(head0 + a.heads, c.h_k);
  if (tid == 0) s_found[0] = -1;
  __syncthreads();
  for (int r = tid; r < c.requests; r += kAppendThreads) {
    const int first = c.cu_blocks[r], end = c.cu_blocks[r + 1], token = c.cu_seqlens[r], token_end = c.cu_seqlens[r + 1], length = c.lengths[r];
    if (first <= unit && unit < end) {
      s_found[0] = r;
      s_found[1] = token;
      s_found[2] = token_end - token;
      s_found[3] = length;
      s_found[4] = unit - first;
    }
  }
  __syncthreads();
  const int r = s_found[0];
  if (r < 0) return;
  const int bs = 1 << a.shift;
  const int token0 = s_found[1], n_new = s_found[2], length = s_found[3], before = length - n_new;
  const int page = (before >> a.shift) + s_found[4];
  if (token0 < 0 || n_new < 0 || token0 + n_new > c.tokens || before < 0 || page >= c.width) return;
  const int begin = page << a.shift;
  const int lo = max(before - begin, 0), hi = min(length - begin, bs);  // places of the new tokens in the block
  const int n = hi - lo;
  if (n <= 0) return;
  const int first = token0 + begin + lo - before;  // the token at place lo
  const int block = c.table[static_cast<int64_t>(r) * c.width + page];

  const bool turn = !is_v && p.turns;
  const RotaryUnits& ru = turn ? a.key_units : a.plain_units;
  const int half = turn ? ru.half : 0;
  const int64_t row_stride = is_v ? p.value_row_stride : p.key_row_stride, head_stride = is_v ? p.value_head_stride : p.key_head_stride;
  // A thread keeps its unit and walks the tokens. The first kHold of its vectors are asked for a head ahead, and stay in registers
  // between the two passes.
  using V = Vec<T, N>;
  constexpr int kHold = 1;
  const int abreast = kAppendThreads / ru.units;  // units <= 256
  const int t_first = tid / ru.units, u = tid - t_first * ru.units;
  const int t_begin = t_first < abreast ? t_first : n;
  const bool pair = u < ru.pair_units;
  const int2 at = unit_offsets<N, kInterleaved>(ru, u);
  V hx[kHold], hy[kHold] = {};  // y: zeros where the unit has one vector
  const T* src = static_cast<const T*>(is_v ? p.value : p.key) + first * row_stride + head0 * head_stride;
  auto hold = [&](const T* from) {
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      const int t = t_begin + k * abreast;
      if (t < n) {
        hx[k] = *reinterpret_cast<const V*>(from + t * row_stride + at.x);
        if (pair) hy[k] = *reinterpret_cast<const V*>(from + t * row_stride + at.y);
      }
    }
  };
  hold(src);
  if (turn) {
    const int t_step = kAppendThreads / half, f_step = kAppendThreads - t_step * half;
    for (int t = tid / half, f = tid - t * half; t < n; t += t_step, f += f_step) {
      if (f >= half) {
        f -= half;
        if (++t >= n) break;
      }
      s_factors[t * factor_pitch<N>(half) + factor_at<N>(f)] = rotary_factors(before + (first - token0) + t, p.turns[f], p.amplitude, false);
    }
  }
  if (block < 0 || block >= c.num_blocks) return;
  __syncthreads();  // the factors
  auto values = [&](const V& vx, const V& vy, int t, float (&x)[N], float (&y)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      x[j] = to_f(vx.x[j]);
      y[j] = to_f(vy.x[j]);
    }
    if (turn && pair) rotate_unit<N, kInterleaved>(x, y, s_factors + t * factor_pitch<N>(half) + u * kFactorUnit<N>);
  };
  for (int head = head0; head < head_end; ++head, src += head_stride) {
    const int64_t at_scale = static_cast<int64_t>(block) * c.h_k + head;
    uint8_t* dst = static_cast<uint8_t*>(is_v ? c.v : c.k) + (at_scale * bs) * c.d;
    float* scale = (is_v ? c.v_scale : c.k_scale) + at_scale;
    const float old_scale = lo > 0 ? *scale : 0.f;
    float most = 0.f;
    auto look = [&](const V& vx, const V& vy, int t) {
      float x[N], y[N];
      values(vx, vy, t, x, y);
#pragma unroll
      for (int j = 0; j < N; ++j) most = fmaxf(fmaxf(most, fabsf(x[j])), fabsf(y[j]));  // (NaN does not count)
    };
    auto rest = [&](int t, auto&& use) {  // the vectors that are not held: from token t on
      for (; t < n; t += abreast) {
        const V vx = *reinterpret_cast<const V*>(src + t * row_stride + at.x);
        V vy = {};
        if (pair) vy = *reinterpret_cast<const V*>(src + t * row_stride + at.y);
        use(vx, vy, t);
      }
    };
    auto of_all = [&] {  // (two rows: the next head's maxima must not overtake readers of these)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if ((tid & 31) == 0) s_max[head & 1][tid >> 5] = most;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kAppendThreads / 32; ++w) most = fmaxf(most, s_max[head & 1][w]);
    };
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      const int t = t_begin + k * abreast;
      if (t < n) look(hx[k], hy[k], t);
    }
    rest(t_begin + kHold * abreast, look);
    of_all();
    if (most > 3.402823466e38f) {  // infinities do not count: once more without them, in every thread
      __syncthreads();
      most = 0.f;
      rest(t_begin, [&](const V& vx, const V& vy, int t) {
        float x[N], y[N];
        values(vx, vy, t, x, y);
        for (int j = 0; j < N; ++j)
          for (const float v : {fabsf(x[j]), fabsf(y[j])})
            if (v <= 3.402823466e38f) most = fmaxf(most, v);
      });
      of_all();
    }
    const float now = fmaxf(block_scale(most), old_scale), inv = __frcp_rn(now);
    if (tid == 0) *scale = now;
    auto write = [&](const V& vx, const V& vy, int t) {
      float x[N], y[N];
      values(vx, vy, t, x, y);
      uint8_t* row = dst + (lo + t) * c.d;
      *reinterpret_cast<Vec<uint8_t, N>*>(row + at.x) = to_e4m3<N>(x, inv);
      if (pair) *reinterpret_cast<Vec<uint8_t, N>*>(row + at.y) = to_e4m3<N>(y, inv);
    };
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      const int t = t_begin + k * abreast;
      if (t < n) write(hx[k], hy[k], t);
    }
    rest(t_begin + kHold * abreast, write);
    if (head + 1 < head_end) hold(src + head_stride);
    if (lo > 0 && now > old_scale) {  // the tokens that were there, at the new scale
      const float f = old_scale * inv;
      for (int i = tid; i < lo * c.d / 16; i += kAppendThreads) {
        Vec<uint8_t, 16>& v = *reinterpret_cast<Vec<uint8_t, 16>*>(dst + i * 16);
        Vec<uint8_t, 16> x = v;
#pragma unroll
        for (int j = 0; j < 16; ++j) x.x[j] = to_e4m3(from_e4m3(x.x[j]) * f);
        v = x;
      }
    }
  }
}

template <typename T, int N, bool kInterleaved>
int launch_append(AppendArgs a, cudaStream_t stream) {
  const fdma_cache_append_params& p = a.p;
  const fdma_cache& c = p.c;
  const bool turn = p.turns != nullptr;
  a.key_units = rotary_units(c.d, turn ? p.rotary_dim : c.d, N);
  a.plain_units = rotary_units(c.d, c.d, N);
  size_t smem = turn ? static_cast<size_t>(std::min(1 << a.shift, c.tokens)) * factor_pitch<N>(a.key_units.half) * sizeof(float2) : 0;
  int64_t query_ctas = 0;
  a.query = RotaryArgs{};
  if (turn && p.query) {
    fdma_rotary_params q = {};
    q.q = p.query; q.q_out = p.query_out;
    q.turns = p.turns;
    q.positions = c.positions; q.position_bits = 32; q.pos_row_stride = 1;
    q.q_row_stride = p.query_row_stride; q.q_head_stride = p.query_head_stride;
    q.qo_row_stride = p.out_row_stride; q.qo_head_stride = p.out_head_stride;
    q.b = 1; q.seqlen = c.tokens; q.h = p.h; q.d = c.d; q.rotary_dim = p.rotary_dim;
    q.interleaved = p.interleaved; q.dtype = p.dtype; q.amplitude = p.amplitude;
    a.query = rotary_args(q, N);
    query_ctas = (a.query.groups + kRotaryWarps - 1) / kRotaryWarps;
    smem = std::max(smem, rotary_smem<N>(a.query));
  }
  auto kern = append_kernel<T, N, kInterleaved>;
  if (smem > 40 * 1024) {
    static std::atomic<uint64_t> prepared{0};
    const int most = kMaxBlock * factor_pitch<N>(kMaxDim / 2) * static_cast<int>(sizeof(float2));  // (what queries need is less)
    const int st = allow_smem_once(reinterpret_cast<const void*>(kern), most, prepared);
    if (st) return st;
  }
  const int64_t ctas = a.cache_ctas + query_ctas;
  if (ctas > 0x7FFFFFFF) return FDMA_ERR_UNSUPPORTED;
  kern<<<static_cast<unsigned>(ctas), kAppendThreads, smem, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int launch_append_t(const AppendArgs& a, cudaStream_t stream) {
  const fdma_cache_append_params& p = a.p;
  uint64_t x = reinterpret_cast<uintptr_t>(p.key) | reinterpret_cast<uintptr_t>(p.value);
  uint64_t strides = static_cast<uint64_t>(p.key_row_stride | p.key_head_stride | p.value_row_stride | p.value_head_stride);
  if (p.turns && p.query) {
    x |= reinterpret_cast<uintptr_t>(p.query) | reinterpret_cast<uintptr_t>(p.query_out);
    strides |= static_cast<uint64_t>(p.query_row_stride | p.query_head_stride | p.out_row_stride | p.out_head_stride);
  }
  const bool vec = (x | strides * sizeof(T)) % 16 == 0 && rotary_units_fit(p.c.d, p.turns ? p.rotary_dim : p.c.d, 8);
  if (vec) return p.interleaved ? launch_append<T, 8, true>(a, stream) : launch_append<T, 8, false>(a, stream);
  return p.interleaved ? launch_append<T, 1, true>(a, stream) : launch_append<T, 1, false>(a, stream);
}

}  // namespace

int check_cache(const fdma_cache& c) {
  if (!c.k || !c.v || !c.k_scale || !c.v_scale || !c.table || !c.cu_seqlens || !c.lengths || !c.cu_blocks || !c.cu_chunks) return FDMA_ERR_BAD_ARG;
  if (c.requests < 0 || c.width <= 0 || c.num_blocks <= 0 || c.tokens < 0 || c.h_k <= 0 || c.d <= 0) return FDMA_ERR_BAD_ARG;
  if (block_shift(c.block_size) < 0 || c.d % 16 || c.d > 256) return FDMA_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15) return FDMA_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(c.width) * c.block_size > 0x7FFFFFFF) return FDMA_ERR_UNSUPPORTED;
  return 0;
}

}  // namespace fdma

using namespace fdma;

extern "C" int fdma_tables_extend(const fdma_tables_params* p, void* stream) {
  int st = check_tables(p);
  if (st) return st;
  if (!p->cu_seqlens || !p->cu_blocks || !p->cu_chunks || (p->tokens && (!p->positions || !p->slots))) return FDMA_ERR_BAD_ARG;
  if (p->requests == 0 || !p->lengths_after || !p->granted) return FDMA_ERR_BAD_ARG;
  size_t smem;
  static std::atomic<uint64_t> prepared{0};
  st = table_smem(extend_kernel, p->requests, prepared, &smem);
  if (st) return st;
  // a CTA for 2048 tokens: beyond that filling takes longer than another CTA's sums
  const int ctas = std::max(1, std::min(sm_count(), p->tokens / 2048));
  extend_kernel<<<ctas, table_threads(std::max(p->requests, p->tokens)), smem, static_cast<cudaStream_t>(stream)>>>(*p, block_shift(p->block_size));
  return static_cast<int>(cudaGetLastError());
}

extern "C" int fdma_tables_truncate(const fdma_tables_params* p, void* stream) {
  int st = check_tables(p);
  if (st) return st;
  if (p->requests == 0) return FDMA_OK;
  size_t smem;
  static std::atomic<uint64_t> prepared{0};
  st = table_smem(truncate_kernel, p->requests, prepared, &smem);
  if (st) return st;
  truncate_kernel<<<1, kTableThreads, smem, static_cast<cudaStream_t>(stream)>>>(*p, block_shift(p->block_size));
  return static_cast<int>(cudaGetLastError());
}

extern "C" int fdma_cache_append(const fdma_cache_append_params* p, void* stream_) {
  if (!p) return FDMA_ERR_BAD_ARG;
  const int st = check_cache(p->c);
  if (st) return st;
  if (p->c.tokens == 0 || p->c.requests == 0) return FDMA_OK;
  if (!p->key || !p->value || !p->c.positions) return FDMA_ERR_BAD_ARG;
  if (p->turns && (p->rotary_dim <= 0 || p->rotary_dim % 2 || p->rotary_dim > p->c.d)) return FDMA_ERR_BAD_ARG;
  if (p->turns && p->query && (!p->query_out || p->h <= 0)) return FDMA_ERR_BAD_ARG;
  AppendArgs a = {};
  a.p = *p;
  a.shift = block_shift(p->c.block_size);
  a.most_units = static_cast<int>(std::min<int64_t>(p->c.tokens, (static_cast<int64_t>(p->c.tokens) >> a.shift) + 2 * static_cast<int64_t>(p->c.requests)));
  // Heads of a CTA: as many as leave two CTAs for each place on the GPU. They share the look-ups and the factors; CTAs that turn keys
  // take longer than those of values, which a second one evens out (the prompts above: one for each place 51.0 us, two 49.3, three 49.2).
  const int64_t places = static_cast<int64_t>(kAppendCtas) * sm_count();
  const int64_t groups = std::max<int64_t>(1, std::min<int64_t>(p->c.h_k, places / a.most_units));
  a.heads = static_cast<int>((p->c.h_k + groups - 1) / groups);
  a.cache_ctas = 2 * static_cast<int64_t>(a.most_units) * ((p->c.h_k + a.heads - 1) / a.heads);
  if (a.cache_ctas > 0x7FFFFFFF) return FDMA_ERR_UNSUPPORTED;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  switch (p->dtype) {
    case FDMA_BF16: return launch_append_t<__nv_bfloat16>(a, stream);
    case FDMA_FP16: return launch_append_t<__half>(a, stream);
    default: return FDMA_ERR_UNSUPPORTED;
  }
}
