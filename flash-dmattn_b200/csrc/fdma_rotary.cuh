// Rotary positions: what the rotation kernel and the cache's writer share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>

#include "fdma_internal.h"

namespace fdma {

// cos and sin of position * frequency, times the amplitude. The frequency is in turns per position as a 64-bit fraction, so that
// the product modulo 2^64 IS the angle modulo a turn, without rounding: an angle at position 10^6 is as exact as one at 1, and no
// 64-bit floating-point arithmetic or table over positions is needed. (fp32 angles are off by 0.06 at 10^6.)
__device__ __forceinline__ float2 rotary_factors(int64_t position, int64_t turns, float amplitude, bool inverse) {
  const int64_t phase = static_cast<int64_t>(static_cast<uint64_t>(position) * static_cast<uint64_t>(turns));
  float s, c;
  sincospif(__ll2float_rn(phase) * 0x1p-63f, &s, &c);  // half turns in [-1, 1]
  return make_float2(c * amplitude, inverse ? -s * amplitude : s * amplitude);
}

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T x[N];
};

// A row is handled in units: N pairs each (2 N elements) for the rotated part, then N elements each for the rest. In the half
// layout the two elements of a pair are rotary_dim / 2 apart, in the interleaved one they are neighbours.
struct RotaryUnits {
  int d, half, pair_units, units;  // half = rotary_dim / 2 (0: nothing rotated)
  bool interleaved;
};
inline RotaryUnits rotary_units(int d, int rotary_dim, bool interleaved, int n) {
  RotaryUnits u;
  u.d = d;
  u.half = rotary_dim / 2;
  u.pair_units = u.half / n;
  u.units = u.pair_units + (d - rotary_dim) / n;
  u.interleaved = interleaved;
  return u;
}
// whether units of n elements fit: otherwise n = 1
inline bool rotary_units_fit(int d, int rotary_dim, int n) { return rotary_dim / 2 % n == 0 && (d - rotary_dim) % n == 0; }

// The two vectors of unit u of a row in memory (the second is the first for a unit of the rest).
template <int N>
__device__ __forceinline__ int2 unit_offsets(const RotaryUnits& ru, int u) {
  if (u >= ru.pair_units) {
    const int at = 2 * ru.half + (u - ru.pair_units) * N;
    return make_int2(at, at);
  }
  return ru.interleaved ? make_int2(2 * u * N, 2 * u * N + N) : make_int2(u * N, ru.half + u * N);
}

// Rotates the 2 N values of unit u in place, given the N factors of its pairs.
template <int N>
__device__ __forceinline__ void rotate_unit(float (&a)[N], float (&b)[N], const float2* factors, bool interleaved) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 f = factors[i];
    if (interleaved) {  // pair i: elements 2 i, 2 i + 1 of a followed by b
      float& x1 = 2 * i < N ? a[(2 * i) % N] : b[(2 * i) % N];
      float& x2 = 2 * i + 1 < N ? a[(2 * i + 1) % N] : b[(2 * i + 1) % N];
      const float y1 = x1 * f.x - x2 * f.y;
      x2 = x2 * f.x + x1 * f.y;
      x1 = y1;
    } else {
      const float y1 = a[i] * f.x - b[i] * f.y;
      b[i] = b[i] * f.x + a[i] * f.y;
      a[i] = y1;
    }
  }
}

constexpr int kRotaryThreads = 256;

struct RotaryArgs {
  fdma_rotary_params p;
  RotaryUnits ru;
  int tokens_per_cta;
  int64_t tokens;
};
// What CTA `cta` of a rotation does; s_factors holds tokens_per_cta * half pairs.
template <typename T, int N>
__device__ __forceinline__ void rotate_tokens(const RotaryArgs& a, int64_t cta, float2* s_factors) {
  const fdma_rotary_params& p = a.p;
  const RotaryUnits& ru = a.ru;
  const int64_t token0 = cta * a.tokens_per_cta;
  const int n = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_cta), a.tokens - token0));
  for (int i = threadIdx.x; i < n * ru.half; i += kRotaryThreads) {
    const int64_t token = token0 + i / ru.half;
    const int64_t b = token / p.seqlen, s = token - b * p.seqlen;
    int64_t pos = s;
    if (p.positions) {
      const int64_t at = b * p.pos_batch_stride + s * p.pos_row_stride;
      pos = p.position_bits == 64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
    }
    s_factors[i] = rotary_factors(pos, p.turns[i % ru.half], p.amplitude, p.inverse != 0);
  }
  __syncthreads();
  const int per_token = (p.h + p.h_k) * ru.units;
  for (int i = threadIdx.x; i < n * per_token; i += kRotaryThreads) {
    const int t = i / per_token, rest = i - t * per_token;
    const int head = rest / ru.units, u = rest - head * ru.units;
    const int64_t token = token0 + t;
    const int64_t b = token / p.seqlen, s = token - b * p.seqlen;
    const T* src;
    T* dst;
    if (head < p.h) {
      src = static_cast<const T*>(p.q) + b * p.q_batch_stride + s * p.q_row_stride + head * p.q_head_stride;
      dst = static_cast<T*>(p.q_out) + b * p.qo_batch_stride + s * p.qo_row_stride + head * p.qo_head_stride;
    } else {
      src = static_cast<const T*>(p.k) + b * p.k_batch_stride + s * p.k_row_stride + (head - p.h) * p.k_head_stride;
      dst = static_cast<T*>(p.k_out) + b * p.ko_batch_stride + s * p.ko_row_stride + (head - p.h) * p.ko_head_stride;
    }
    const int2 at = unit_offsets<N>(ru, u);
    using V = Vec<T, N>;
    V x = *reinterpret_cast<const V*>(src + at.x);
    if (u < ru.pair_units) {
      V y = *reinterpret_cast<const V*>(src + at.y);
      float fa[N], fb[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        fa[j] = to_f(x.x[j]);
        fb[j] = to_f(y.x[j]);
      }
      rotate_unit<N>(fa, fb, s_factors + t * ru.half + u * N, ru.interleaved);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x.x[j] = from_f<T>(fa[j]);
        y.x[j] = from_f<T>(fb[j]);
      }
      *reinterpret_cast<V*>(dst + at.y) = y;
    }
    *reinterpret_cast<V*>(dst + at.x) = x;
  }
}


// Whether every row of the given tensors can be accessed in 16-byte vectors.
inline bool rotary_aligned16(const fdma_rotary_params& p, int bytes) {
  uint64_t x = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.q_out);
  uint64_t strides = static_cast<uint64_t>(p.q_batch_stride | p.q_row_stride | p.q_head_stride | p.qo_batch_stride | p.qo_row_stride | p.qo_head_stride);
  if (p.h_k) {
    x |= reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.k_out);
    strides |= static_cast<uint64_t>(p.k_batch_stride | p.k_row_stride | p.k_head_stride | p.ko_batch_stride | p.ko_row_stride | p.ko_head_stride);
  }
  return (x | strides * bytes) % 16 == 0;
}
inline RotaryArgs rotary_args(const fdma_rotary_params& p, int n) {
  RotaryArgs a;
  a.p = p;
  a.ru = rotary_units(p.d, p.rotary_dim, p.interleaved != 0, n);
  a.tokens = static_cast<int64_t>(p.b) * p.seqlen;
  const int64_t per_token = static_cast<int64_t>(p.h + p.h_k) * a.ru.units;
  int64_t t = std::max<int64_t>(1, 4 * kRotaryThreads / per_token);
  t = std::min<int64_t>(t, std::max(1, 4096 / a.ru.half));  // 32 KB of factors
  a.tokens_per_cta = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(t, a.tokens / (4 * sm_count()))));
  return a;
}

}  // namespace fdma
