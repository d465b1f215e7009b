// Rotary positions: what the rotation kernel and the cache's writer share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "fdma_internal.h"

namespace fdma {

// sin and cos of pi x for |x| <= 1/4, by their Taylor series (remainders 1.7e-9 and 4.6e-10 at the ends); pi in two parts, so that
// its rounding does not count.
__device__ __forceinline__ void sincos_quarter(float x, float* s, float* c) {
  const float z = x * x;
  float p = 0.08214588661112823f;           // pi^9 / 9!
  p = fmaf(p, z, -0.5992645293207921f);     // -pi^7 / 7!
  p = fmaf(p, z, 2.550164039877345f);       // pi^5 / 5!
  p = fmaf(p, z, -5.16771278004997f);       // -pi^3 / 3!
  p = fmaf(p, z, -8.742277657347586e-8f);   // pi - (its first part)
  *s = fmaf(p, x, 3.1415927410125732f * x);
  float q = -0.02580689139001406f;          // -pi^10 / 10!
  q = fmaf(q, z, 0.23533063035889312f);     // pi^8 / 8!
  q = fmaf(q, z, -1.3352627688545893f);     // -pi^6 / 6!
  q = fmaf(q, z, 4.058712126416768f);       // pi^4 / 4!
  q = fmaf(q, z, -4.934802200544679f);      // -pi^2 / 2!
  *c = fmaf(q, z, 1.f);
}

// cos and sin of position * frequency, times the amplitude. The frequency is in turns per position as a 64-bit fraction, so that
// the product modulo 2^64 IS the angle modulo a turn of that frequency, without rounding, and no 64-bit floating-point arithmetic or
// table over positions is needed. The frequency itself is off by at most 2^-65 turn, an angle at position 10^6 by 2^-45. (fp32
// angles are off by 0.06 at 10^6.)
__device__ __forceinline__ float2 rotary_factors(int64_t position, int64_t turns, float amplitude, bool inverse) {
  const uint64_t phase = static_cast<uint64_t>(position) * static_cast<uint64_t>(turns);
  // the nearest quarter turn, and what is left of it in units of 2^-32 turn: less than one of them is lost, 1.5e-9 of a result
  const uint32_t top = static_cast<uint32_t>(phase >> 32), quarter = top + (1u << 29);
  const int32_t left = static_cast<int32_t>(top - (quarter & (3u << 30)));
  float s, c;
  sincos_quarter(static_cast<float>(left) * 0x1p-31f, &s, &c);
  const uint32_t n = quarter >> 30;
  float cn = n & 1 ? -s : c, sn = n & 1 ? c : s;
  if (n & 2) {
    cn = -cn;
    sn = -sn;
  }
  return make_float2(cn * amplitude, inverse ? -sn * amplitude : sn * amplitude);
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
// N numbers rounded to T, two at a time where the type has an instruction for that
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> round_to(const float (&f)[N]) {
  Vec<T, N> v;
  if constexpr (N % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) *reinterpret_cast<__nv_bfloat162*>(&v.x[j]) = __floats2bfloat162_rn(f[j], f[j + 1]);
      else *reinterpret_cast<__half2*>(&v.x[j]) = __floats2half2_rn(f[j], f[j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v.x[j] = from_f<T>(f[j]);
  }
  return v;
}

// A row is handled in units: N pairs each (2 N elements) for the rotated part, then N elements each for the rest. In the half
// layout the two elements of a pair are rotary_dim / 2 apart, in the interleaved one they are neighbours.
struct RotaryUnits {
  int half, pair_units, units;  // half = rotary_dim / 2 (0: nothing rotated)
};
inline RotaryUnits rotary_units(int d, int rotary_dim, int n) {
  RotaryUnits u;
  u.half = rotary_dim / 2;
  u.pair_units = u.half / n;
  u.units = u.pair_units + (d - rotary_dim) / n;
  return u;
}
// whether units of n elements fit: otherwise n = 1
inline bool rotary_units_fit(int d, int rotary_dim, int n) { return rotary_dim / 2 % n == 0 && (d - rotary_dim) % n == 0; }

// The two vectors of unit u of a row in memory (the second is the first for a unit of the rest).
template <int N, bool kInterleaved>
__device__ __forceinline__ int2 unit_offsets(const RotaryUnits& ru, int u) {
  if (u >= ru.pair_units) {
    const int at = 2 * ru.half + (u - ru.pair_units) * N;
    return make_int2(at, at);
  }
  return kInterleaved ? make_int2(2 * u * N, 2 * u * N + N) : make_int2(u * N, ru.half + u * N);
}

// Rotates the 2 N values of a unit in place, given the factors of its pairs.
template <int N, bool kInterleaved>
__device__ __forceinline__ void rotate_unit(float (&a)[N], float (&b)[N], const float2* factors) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 f = factors[i];
    if (kInterleaved) {  // pair i: elements 2 i, 2 i + 1 of a followed by b
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

// Factors in shared memory: those of a unit side by side, units 16 bytes apart from one another, so that eight lanes on neighbouring
// units read different banks. factor_pitch: of a token.
template <int N>
constexpr int kFactorUnit = N > 1 ? N + 2 : 1;
template <int N>
__host__ __device__ __forceinline__ int factor_pitch(int half) { return half / N * kFactorUnit<N>; }
template <int N>
__device__ __forceinline__ int factor_at(int f) { return f / N * kFactorUnit<N> + f % N; }

// A warp takes one token (`abreast` of them where they are small), computes its factors, and goes over the heads of q and k: a lane
// keeps its unit, and with it the factors in registers, and takes every so many heads. Nothing is shared between warps.
// 2 x 4096 tokens of 32 + 8 heads, d = 128 (168 MB): 35 us (4.8 TB/s; a plain copy between the same buffers takes 33). Asking for
// two or four heads at a time instead needs the registers of half the warps and took 42 and 44 us; going over the units of all
// heads as one row, with the factors read for each vector, 42 us.
constexpr int kRotaryWarps = 8;  // per CTA
struct RotaryArgs {
  fdma_rotary_params p;
  RotaryUnits ru;
  int abreast;
  int64_t groups;  // a warp each
};

// Units [first, first + units) of `heads` heads of n tokens.
template <typename T, int N, bool kInterleaved, bool kPair>
__device__ __forceinline__ void rotate_heads(const T* src, T* dst, int64_t src_row, int64_t dst_row, int64_t src_head, int64_t dst_head, int heads,
                                             int n, const RotaryUnits& ru, const float2* s_factors) {
  using V = Vec<T, N>;
  const int lane = threadIdx.x & 31;
  const int units = kPair ? ru.pair_units : ru.units - ru.pair_units;
  for (int u0 = 0; u0 < units; u0 += 32) {
    const int across = min(units - u0, 32);           // lanes of a head
    const int place = lane / across, u = u0 + lane - place * across;
    const int hs = min(32 / across, heads), ts = 32 / (across * hs);  // heads and tokens side by side
    const int tsub = place / hs, hsub = place - tsub * hs;
    if (tsub >= ts) continue;
    const int2 at = unit_offsets<N, kInterleaved>(ru, kPair ? u : ru.pair_units + u);
    const int64_t src_step = hs * src_head, dst_step = hs * dst_head;
    for (int t = tsub; t < n; t += ts) {
      float2 f[N];
      if (kPair) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = s_factors[t * factor_pitch<N>(ru.half) + u * kFactorUnit<N> + j];
      }
      const T* from = src + t * src_row + hsub * src_head + at.x;
      T* to = dst + t * dst_row + hsub * dst_head + at.x;
      const int apart = at.y - at.x;
      for (int h = hsub; h < heads; h += hs) {
        V x = *reinterpret_cast<const V*>(from);
        if (kPair) {
          const V y = *reinterpret_cast<const V*>(from + apart);
          float fa[N], fb[N];
#pragma unroll
          for (int j = 0; j < N; ++j) {
            fa[j] = to_f(x.x[j]);
            fb[j] = to_f(y.x[j]);
          }
          rotate_unit<N, kInterleaved>(fa, fb, f);
          x = round_to<T, N>(fa);
          *reinterpret_cast<V*>(to + apart) = round_to<T, N>(fb);
        }
        *reinterpret_cast<V*>(to) = x;
        from += src_step;
        to += dst_step;
      }
    }
  }
}

// What warp `group` of a rotation does; s_factors: abreast * factor_pitch pairs of the warp's own.
template <typename T, int N, bool kInterleaved>
__device__ __forceinline__ void rotate_tokens(const RotaryArgs& a, int64_t group, float2* s_factors) {
  if (group >= a.groups) return;
  const fdma_rotary_params& p = a.p;
  const RotaryUnits& ru = a.ru;
  const int lane = threadIdx.x & 31;
  // groups do not cross batch rows
  const int per_row = (p.seqlen + a.abreast - 1) / a.abreast;
  const int64_t b = a.groups <= 0x7FFFFFFF ? static_cast<uint32_t>(group) / static_cast<uint32_t>(per_row) : group / per_row;
  const int s = static_cast<int>(group - b * per_row) * a.abreast, n = min(a.abreast, p.seqlen - s);
  for (int i = lane; i < n * ru.half; i += 32) {
    const int t = a.abreast > 1 ? i / ru.half : 0, f = i - t * ru.half;
    int64_t pos = s + t;
    if (p.positions) {
      const int64_t at = b * p.pos_batch_stride + pos * p.pos_row_stride;
      pos = p.position_bits == 64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
    }
    s_factors[t * factor_pitch<N>(ru.half) + factor_at<N>(f)] = rotary_factors(pos, p.turns[f], p.amplitude, p.inverse != 0);
  }
  __syncwarp();
  const T* q = static_cast<const T*>(p.q) + b * p.q_batch_stride + s * p.q_row_stride;
  T* qo = static_cast<T*>(p.q_out) + b * p.qo_batch_stride + s * p.qo_row_stride;
  const T* k = static_cast<const T*>(p.k) + b * p.k_batch_stride + s * p.k_row_stride;
  T* ko = static_cast<T*>(p.k_out) + b * p.ko_batch_stride + s * p.ko_row_stride;
  rotate_heads<T, N, kInterleaved, true>(q, qo, p.q_row_stride, p.qo_row_stride, p.q_head_stride, p.qo_head_stride, p.h, n, ru, s_factors);
  if (p.h_k) rotate_heads<T, N, kInterleaved, true>(k, ko, p.k_row_stride, p.ko_row_stride, p.k_head_stride, p.ko_head_stride, p.h_k, n, ru, s_factors);
  if (ru.units > ru.pair_units) {
    rotate_heads<T, N, kInterleaved, false>(q, qo, p.q_row_stride, p.qo_row_stride, p.q_head_stride, p.qo_head_stride, p.h, n, ru, s_factors);
    if (p.h_k) rotate_heads<T, N, kInterleaved, false>(k, ko, p.k_row_stride, p.ko_row_stride, p.k_head_stride, p.ko_head_stride, p.h_k, n, ru, s_factors);
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
  a.ru = rotary_units(p.d, p.rotary_dim, n);
  a.abreast = std::max(1, std::min(p.seqlen, 32 / (p.h * std::max(1, a.ru.pair_units))));
  a.groups = static_cast<int64_t>(p.b) * ((p.seqlen + a.abreast - 1) / a.abreast);
  return a;
}
template <int N>
__host__ __device__ __forceinline__ int rotary_warp_pairs(const RotaryArgs& a) { return a.abreast * factor_pitch<N>(a.ru.half); }
template <int N>
inline size_t rotary_smem(const RotaryArgs& a) { return static_cast<size_t>(kRotaryWarps) * rotary_warp_pairs<N>(a) * sizeof(float2); }

}  // namespace fdma
