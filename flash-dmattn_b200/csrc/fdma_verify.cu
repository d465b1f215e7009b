// Verification of drafted tokens: how many drafts of each request the target's probabilities accept, and the token that comes next.
//
//   p = softmax(logits / T),  draft x behind a row is accepted if u q(x) < p(x); q: the drafter's probabilities (without them: 1 for x)
//   after the first rejection the next token is drawn from max(p - q, 0), after none from p, by its running sum: the first token whose
//   sum is above u times the total. T = 0: a draft is accepted if it is the row's largest logit, which is the next token otherwise.
//
// What it has to move is the logits, once: HBM-bound, 2 or 4 bytes a number. One launch: a cluster of CTAs has a request, each CTA a slice
// of the vocabulary. They stream the request's rows with a running maximum and sum, in 32 bits, join them through each other's shared
// memory and know how many drafts pass; then the row that the next token comes from is read again, from L2, with the drafter's.
// A random number beside a border decides between two tokens, so what is compared with it is summed up in 64 bits, with exponentials
// that are exact to 2^-46: the row of the next token always, a draft's own row where 32 bits leave the verdict open. Sums have one order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "fdma_internal.h"
#include "fdma_ptx.cuh"

namespace fdma {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kRows = 16;       // rows that are streamed before their verdicts
constexpr int kMaxCluster = 16;
constexpr int kSegments = 64;   // parts of a CTA's slice whose 64-bit sums are kept
constexpr int kAhead = 4;       // vectors in flight per thread
constexpr float kLog2e = 1.4426950408889634f;
// 32 bits leave a verdict open where both sides are nearer than this (their errors: 2^-22 of the exponentials, sums of 2^17 and more of them)
constexpr float kNear = 3e-5f;

struct VerifyArgs {
  fdma_verify_params p;
  int cluster;
};

// One row's part: the largest number, its index (of several the first), the sum of exponentials relative to it
struct Part {
  float top, sum;
  int at;
};

// 2^y for y <= 0, to 2^-46 of itself: the series of e^x for |x| <= ln(2) / 2 up to its 11th power; the 12th term is below 2^-47.
__device__ __forceinline__ double exp2_64(double y) {
  if (!(y > -1000.0)) return 0.0;
  const double shifted = y + 6755399441055744.0;  // 1.5 * 2^52: the nearest whole number in the low bits
  const double x = (y - (shifted - 6755399441055744.0)) * 0.693147180559945309417;
  double s = 1.0 / 39916800.0;
  s = fma(s, x, 1.0 / 3628800.0);
  s = fma(s, x, 1.0 / 362880.0);
  s = fma(s, x, 1.0 / 40320.0);
  s = fma(s, x, 1.0 / 5040.0);
  s = fma(s, x, 1.0 / 720.0);
  s = fma(s, x, 1.0 / 120.0);
  s = fma(s, x, 1.0 / 24.0);
  s = fma(s, x, 1.0 / 6.0);
  s = fma(s, x, 0.5);
  s = fma(s, x, 1.0);
  s = fma(s, x, 1.0);
  return __hiloint2double(__double2hiint(s) + (__double2loint(shifted) << 20), __double2loint(s));
}

// NaN counts as -inf, +inf as the largest finite number
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -CUDART_INF_F), 3.402823466e38f); }
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// The N numbers from element `at` on, which may be negative or end beyond n: those that are not there are `none`.
template <typename T, int N>
__device__ __forceinline__ void load(const T* row, int64_t at, int n, float none, float (&x)[N]) {
  using Vec = std::conditional_t<N * sizeof(T) % 16 == 0, uint4, uint2>;
  static_assert(N * sizeof(T) % sizeof(Vec) == 0, "whole vectors");
  if (at >= 0 && at + N <= n && reinterpret_cast<uintptr_t>(row + at) % sizeof(Vec) == 0) {
    constexpr int kPer = sizeof(Vec) / sizeof(T);
#pragma unroll
    for (int v = 0; v < N / kPer; ++v) {
      const Vec raw = __ldg(reinterpret_cast<const Vec*>(row + at) + v);
      T t[kPer];
      memcpy(t, &raw, sizeof(Vec));
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[v * kPer + i] = to_float(t[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = at + i >= 0 && at + i < n ? to_float(row[at + i]) : none;
  }
}

__device__ __forceinline__ Part join(const Part& a, const Part& b, float c) {
  Part r;
  r.top = fmaxf(a.top, b.top);
  r.at = b.top > a.top || (b.top == a.top && b.at < a.at) ? b.at : a.at;
  r.sum = (a.top == -CUDART_INF_F ? 0.f : a.sum * exp2f((a.top - r.top) * c)) + (b.top == -CUDART_INF_F ? 0.f : b.sum * exp2f((b.top - r.top) * c));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t shared_of(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ double ld_cluster_64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}

// A CTA's share of a row in vectors of N numbers, aligned to 16 bytes in memory: vectors [first, end), vector v begins at element v * N - skip.
template <typename T>
struct Slice {
  static constexpr int N = 16 / sizeof(T);
  const T* row;
  int skip, first, end;
  __device__ Slice(const T* row_, int vocab, int rank, int cluster) : row(row_) {
    skip = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int all = (skip + vocab + N - 1) / N, each = (all + cluster - 1) / cluster;
    first = min(all, rank * each);
    end = min(all, first + each);
  }
  __device__ int64_t element(int v) const { return static_cast<int64_t>(v) * N - skip; }
};

template <typename T, typename Q>
__global__ void __launch_bounds__(kThreads) verify_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int N = Slice<T>::N;
  __shared__ __align__(16) float4 s_part[kRows][kWarps];   // of each warp: largest, sum, index
  __shared__ float s_top[kRows];
  __shared__ int s_at[kRows], s_verdict[kRows];            // 0: rejected, 1: accepted, 2: open
  __shared__ double s_seg[2][kSegments];                   // sums of the probabilities, of what is left of them
  __shared__ __align__(16) double s_total[2];
  const fdma_verify_params& p = a.p;
  const int C = a.cluster, rank = static_cast<int>(blockIdx.x) % C, r = static_cast<int>(blockIdx.x) / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = p.vocab;
  const int first = max(0, min(p.cu_seqlens[r], p.tokens)), n = max(0, min(p.cu_seqlens[r + 1], p.tokens) - first);
  const int length = p.lengths[r];
  const bool lead = rank == 0 && tid == 0;
  if (n == 0 || (p.granted && !p.granted[r])) {  // (the whole cluster agrees)
    if (lead) {
      p.accepted[r] = 0;
      p.next_tokens[r] = -1;
      p.lengths_out[r] = length;
    }
    return;
  }
  const float temperature = p.temperatures ? p.temperatures[r] : p.temperature;
  const bool greedy = !(temperature > 0.f);
  const float c = greedy ? 0.f : fminf(fmaxf(kLog2e / temperature, 1e-30f), 1e30f);  // (not 0: of -inf that would be NaN)
  const double c64 = greedy ? 0.0 : 1.4426950408889634074 / static_cast<double>(temperature);
  auto logits = [&](int row) { return static_cast<const T*>(p.logits) + (first + row) * p.logits_row_stride; };
  auto probs = [&](int row) { return static_cast<const Q*>(p.draft_probs) + (first + row) * p.probs_row_stride; };
  auto draft = [&](int row) -> int64_t {  // the token behind a row, -1 where it is none of the vocabulary
    const int64_t x = p.id_bits == 64 ? static_cast<const int64_t*>(p.token_ids)[first + row + 1] : static_cast<const int32_t*>(p.token_ids)[first + row + 1];
    return x >= 0 && x < V ? x : -1;
  };
  auto e64 = [&](float x, float top) { return x == -CUDART_INF_F ? 0.0 : exp2_64((static_cast<double>(x) - static_cast<double>(top)) * c64); };

  // Sums of the row's exponentials in 64 bits, segment by segment; with `left` of what the drafter's row leaves of the probabilities,
  // given their sum z. Returns the total of the cluster's CTAs in their order.
  auto sum_up = [&](int row, float top, bool left, double z) {
    const Slice<T> s(logits(row), V, rank, C);
    const int each = (s.end - s.first + kSegments - 1) / kSegments;  // vectors of a segment
    const int64_t gone = left && !p.draft_probs ? draft(row) : -1;
    for (int g = warp * (kSegments / kWarps); g < (warp + 1) * (kSegments / kWarps); ++g) {
      const int from = min(s.end, s.first + g * each), to = min(s.end, from + each);
      double sum = 0.0;
      for (int v = from + lane; v < to; v += 32) {
        float x[N], q[N];
        load<T, N>(s.row, s.element(v), V, -CUDART_INF_F, x);
        if (left && p.draft_probs) load<Q, N>(probs(row), s.element(v), V, 0.f, q);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          double e = e64(clean(x[i]), top);
          if (left) {
            if (p.draft_probs) e = fmax(e - static_cast<double>(fmaxf(q[i], 0.f)) * z, 0.0);
            else if (s.element(v) + i == gone) e = 0.0;
          }
          sum += e;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s_seg[left][g] = sum;
    }
    __syncthreads();
    if (tid == 0) {
      double sum = 0.0;
      for (int g = 0; g < kSegments; ++g) sum += s_seg[left][g];
      s_total[left] = sum;
    }
    cluster_sync();
    double total = 0.0;
    for (int x = 0; x < C; ++x) total += ld_cluster_64(shared_of(&s_total[left], x));
    return total;
  };

  int accepted = 0, row = -1;  // row: that the next token comes from
  float top = 0.f;
  int best = -1;
  double z = -1.0;
  for (int base = 0; row < 0; base += kRows) {
    const int rows = min(kRows, n - base);
    // ---- maxima and sums of the rows ----
    for (int j = 0; j < rows; ++j) {
      const Slice<T> s(logits(base + j), V, rank, C);
      Part mine{-CUDART_INF_F, 0.f, 0x7FFFFFFF};
      for (int v0 = s.first + tid; v0 < s.end; v0 += kAhead * kThreads) {
        float x[kAhead][N];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int v = v0 + k * kThreads;
          load<T, N>(s.row, v < s.end ? s.element(v) : -N, V, -CUDART_INF_F, x[k]);
        }
        float high = -CUDART_INF_F;
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            x[k][i] = clean(x[k][i]);
            high = fmaxf(high, x[k][i]);
          }
        if (high > mine.top) {
          mine.sum = mine.top == -CUDART_INF_F ? 0.f : mine.sum * exp2f((mine.top - high) * c);
          mine.top = high;
          if (greedy) {
#pragma unroll
            for (int k = kAhead - 1; k >= 0; --k)
#pragma unroll
              for (int i = N - 1; i >= 0; --i)
                if (x[k][i] == high) mine.at = static_cast<int>(s.element(v0 + k * kThreads) + i);
          }
        }
        if (!greedy && mine.top > -CUDART_INF_F) {
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) mine.sum += exp2f((x[k][i] - mine.top) * c);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const Part other{__shfl_xor_sync(0xffffffffu, mine.top, o), __shfl_xor_sync(0xffffffffu, mine.sum, o), __shfl_xor_sync(0xffffffffu, mine.at, o)};
        mine = join(mine, other, c);
      }
      if (lane == 0) s_part[j][warp] = make_float4(mine.top, mine.sum, __int_as_float(mine.at), 0.f);
    }
    __syncthreads();
    cluster_sync();
    // ---- verdicts, by every CTA for itself: a warp per row ----
    for (int j = warp; j < rows; j += kWarps) {
      Part all{-CUDART_INF_F, 0.f, 0x7FFFFFFF};
      for (int x = lane; x < C * kWarps; x += 32) {
        const float4 f = ld_cluster(shared_of(&s_part[j][x % kWarps], x / kWarps));
        all = join(all, Part{f.x, f.y, __float_as_int(f.z)}, c);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const Part other{__shfl_xor_sync(0xffffffffu, all.top, o), __shfl_xor_sync(0xffffffffu, all.sum, o), __shfl_xor_sync(0xffffffffu, all.at, o)};
        // the same in every lane and CTA: of two lanes the lower one's part first
        all = (lane & o) ? join(other, all, c) : join(all, other, c);
      }
      if (lane == 0) {
        int verdict = 0;
        if (base + j < n - 1) {
          const int64_t x = draft(base + j);
          if (greedy) {
            verdict = x == all.at;
          } else if (x >= 0 && all.top > -CUDART_INF_F) {
            const float u = p.uniforms[first + base + j], q = p.draft_probs ? fmaxf(to_float(probs(base + j)[x]), 0.f) : 1.f;
            const float have = exp2f((clean(to_float(logits(base + j)[x])) - all.top) * c), need = u * q * all.sum;
            verdict = fabsf(have - need) <= kNear * fmaxf(have, need) ? 2 : need < have;
          }
        }
        s_top[j] = all.top;
        s_at[j] = all.at;
        s_verdict[j] = verdict;
      }
    }
    __syncthreads();
    for (int j = 0; j < rows && row < 0; ++j) {
      int verdict = s_verdict[j];
      if (verdict == 2) {
        const int64_t x = draft(base + j);
        z = sum_up(base + j, s_top[j], false, 0.0);
        const double u = p.uniforms[first + base + j], q = p.draft_probs ? static_cast<double>(fmaxf(to_float(probs(base + j)[x]), 0.f)) : 1.0;
        verdict = u * q * z < e64(clean(to_float(logits(base + j)[x])), s_top[j]);
        if (verdict) {
          z = -1.0;
          cluster_sync();  // the sums are read no more
        }
      }
      if (verdict) {
        ++accepted;
      } else {
        row = base + j;
        top = s_top[j];
        best = s_at[j] < V ? s_at[j] : -1;
      }
    }
    if (row < 0) cluster_sync();  // the parts are read no more
  }
  if (lead) {
    p.accepted[r] = accepted;
    p.lengths_out[r] = length - (n - 1 - accepted);
  }
  if (greedy || top == -CUDART_INF_F) {
    if (lead) p.next_tokens[r] = greedy && top > -CUDART_INF_F ? best : -1;
  } else {
    // ---- the next token ----
    if (z < 0.0) z = sum_up(row, top, false, 0.0);
    bool left = accepted < n - 1;
    double total = z;
    if (left) {
      total = sum_up(row, top, true, z);
      if (!(total > 0.0)) {  // the drafter is as sure of everything
        left = false;
        total = z;
      }
    }
    // the CTA, segment and vector where the running sum passes the target; where rounding leaves none, the last that add to it
    double target = static_cast<double>(p.uniforms[first + n - 1]) * total;
    int owner = -1;
    double before = 0.0, rest = 0.0;
    for (int x = 0; x < C; ++x) {
      const double t = ld_cluster_64(shared_of(&s_total[left], x));
      if (t > 0.0) {
        owner = x;
        rest = target - before;
      }
      before += t;
      if (t > 0.0 && before > target) break;
    }
    if (rank == owner && warp == 0) {
      int seg = -1;
      target = rest;
      before = 0.0;
      for (int g = 0; g < kSegments; ++g) {
        const double t = s_seg[left][g];
        if (t > 0.0) {
          seg = g;
          rest = target - before;
        }
        before += t;
        if (t > 0.0 && before > target) break;
      }
      const Slice<T> s(logits(row), V, rank, C);
      const int each = (s.end - s.first + kSegments - 1) / kSegments, from = min(s.end, s.first + seg * each), to = min(s.end, from + each);
      const int64_t gone = left && !p.draft_probs ? draft(row) : -1;
      target = rest;
      before = 0.0;
      int token = -1;
      bool found = false;
      for (int v0 = from; v0 < to && !found; v0 += 32) {
        const int v = v0 + lane;
        float x[N], q[N];
        double e[N], sum = 0.0;
        load<T, N>(s.row, v < to ? s.element(v) : -N, V, -CUDART_INF_F, x);
        if (left && p.draft_probs) load<Q, N>(probs(row), v < to ? s.element(v) : -N, V, 0.f, q);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          e[i] = e64(clean(x[i]), top);
          if (left) {
            if (p.draft_probs) e[i] = fmax(e[i] - static_cast<double>(fmaxf(q[i], 0.f)) * z, 0.0);
            else if (s.element(v) + i == gone) e[i] = 0.0;
          }
          sum += e[i];
        }
        double upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        double run = before + (upto - sum);
        int mine = -1;  // of this lane: the first token above the target, or the last that adds to the sum
        bool passed = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          run += e[i];
          if (!passed && e[i] > 0.0) {
            mine = static_cast<int>(s.element(v) + i);
            passed = run > target;
          }
        }
        const uint32_t pass = __ballot_sync(0xffffffffu, passed), some = __ballot_sync(0xffffffffu, mine >= 0);
        if (pass) {
          token = __shfl_sync(0xffffffffu, mine, __ffs(pass) - 1);
          found = true;
        } else if (some) {
          token = __shfl_sync(0xffffffffu, mine, 31 - __clz(some));
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
      if (lane == 0) p.next_tokens[r] = token;
    }
  }
  cluster_sync();  // nobody leaves while its shared memory may still be read
}

template <typename T, typename Q>
int launch(const VerifyArgs& a, cudaStream_t stream) {
  auto kern = verify_kernel<T, Q>;
  if (a.cluster > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.p.requests) * a.cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, a));
}
template <typename T>
int launch_t(const VerifyArgs& a, cudaStream_t stream) {
  switch (a.p.probs_dtype) {
    case FDMA_BF16: return launch<T, __nv_bfloat16>(a, stream);
    case FDMA_FP16: return launch<T, __half>(a, stream);
    default: return launch<T, float>(a, stream);
  }
}
bool known(int dtype) { return dtype == FDMA_BF16 || dtype == FDMA_FP16 || dtype == FDMA_FP32; }

// CTAs that share a request: slices of no less than 1024 numbers, and no more CTAs than four for each SM where there are many requests.
int pick_cluster(const fdma_verify_params& p) {
  int c = 1;
  while (c < kMaxCluster && p.vocab / (2 * c) >= 1024) c *= 2;
  while (c > 1 && static_cast<int64_t>(p.requests) * (c / 2) >= 4 * sm_count()) c /= 2;
  return c;
}

}  // namespace
}  // namespace fdma

using namespace fdma;

extern "C" int fdma_verify_drafts(const fdma_verify_params* pp, void* stream) {
  if (!pp) return FDMA_ERR_BAD_ARG;
  const fdma_verify_params& p = *pp;
  if (p.requests < 0 || p.tokens < 0 || p.vocab <= 0) return FDMA_ERR_BAD_ARG;
  if (!known(p.dtype) || (p.draft_probs && !known(p.probs_dtype)) || (p.id_bits != 32 && p.id_bits != 64) || p.requests > (1 << 26)) return FDMA_ERR_UNSUPPORTED;
  if (p.requests == 0) return FDMA_OK;
  if (!p.cu_seqlens || !p.lengths || !p.accepted || !p.next_tokens || !p.lengths_out) return FDMA_ERR_BAD_ARG;
  if (p.tokens > 0 && (!p.logits || !p.token_ids || !p.uniforms)) return FDMA_ERR_BAD_ARG;
  VerifyArgs a;
  a.p = p;
  if (!p.draft_probs) a.p.probs_dtype = FDMA_FP32;
  a.cluster = pick_cluster(p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p.dtype) {
    case FDMA_BF16: return launch_t<__nv_bfloat16>(a, s);
    case FDMA_FP16: return launch_t<__half>(a, s);
    default: return launch_t<float>(a, s);
  }
}
