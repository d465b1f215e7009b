// Verification of drafted tokens: how many drafts of each request the target's probabilities accept, and the token that comes next.
//
//   p = softmax(logits / T),  draft x behind a row is accepted if u q(x) < p(x); q: the drafter's probabilities (without them: 1 for x)
//   after the first rejection the next token is drawn from max(p - q, 0), after none from p, by its running sum: the first token whose
//   sum is above u times the total. T = 0: a draft is accepted if it is the row's largest logit, which is the next token otherwise.
//
// What it has to move is the logits, once: HBM-bound, 2 or 4 bytes a number. rows_kernel streams all rows, a part of one in each CTA, and
// leaves its maximum and the sum of its exponentials, in 32 bits. In verify_kernel a cluster of CTAs has a request: they know from those
// how many drafts pass, and read the row that the next token comes from again, from L2, with the drafter's, each a slice of the vocabulary.
// 64 requests of 9 rows, 131072 numbers, bf16, with fp32 probabilities: 82 us, rows_kernel 35 of them (4.3 TB/s), verify_kernel 49, bound by
// its instructions, the 64-bit ones among them; 200 of up to 6 rows, 50257 numbers, fp32: 63-68; one of 4 rows, 32000 numbers: 14, two launches and
// a chain of exchanges in a cluster. (In one launch, a cluster streaming its request's rows, few clusters ran at once: 64 requests of 9 rows, 131072 numbers each: 280 us.)
// A random number beside a border decides between two tokens, so what is compared with it is summed up in 64 bits, with exponentials
// that are exact to 2^-44: the row of the next token always, a draft's own row where 32 bits leave the verdict open. Sums have one order.
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
constexpr int kRows = 16;       // of which verdicts are made at once
constexpr int kMaxCluster = 16;
constexpr int kAhead = 4;       // 16-byte vectors per thread that rows_kernel has in flight while it works on as many
constexpr int kKept = 16;       // vectors of a thread of verify_kernel whose sums are kept
constexpr float kLog2e = 1.4426950408889634f;
// 32 bits leave a verdict open where both sides are nearer than this: exponentials are off by 2^-22 of themselves and by their argument's
// rounding, 2^-24 of up to 256, a thread's sums by less.
constexpr float kNear = 4e-5f;
constexpr float kPlain = 256.f;  // largest |top * log2(e) / T| for which an exponential's argument is one multiplication and addition

// The rows' vectors in units of kThreads, row after row: `units` for each row, `share` in a row for each CTA of rows_kernel. Its warps leave
// one part each for every row that the CTA has units of, at places that follow from the units' numbers.
struct VerifyArgs {
  fdma_verify_params p;
  int cluster, units, share, slots;  // slots: most CTAs that have units of a row
  float4* parts;  // [tokens][slots][kWarps]: largest number, sum of exponentials relative to it, index of the largest
  __device__ __forceinline__ int64_t first_unit(int row) const { return static_cast<int64_t>(row) * units; }
};

// One row's part: the largest number, its index (of several the first), the sum of exponentials relative to it
struct Part {
  float top, sum;
  int at;
};

// e^x for |x| <= ln(2) / 2: its series up to the 11th power; the next term is below 2^-47.
__device__ __forceinline__ double exp_series(double x) {
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
  return fma(s, x, 1.0);
}
constexpr double kLn2 = 0.693147180559945309417;
constexpr int kPow = 64;
// 2^y for |y| < 2^25, to 2^-44 of itself where that is at least 2^-1000: the nearest 64th below the point from the table pow[i] = 2^(i / 64),
// the rest, at most 1 / 128, from the series, whose 5th term is below 2^-44. Beyond, some number.
__device__ __forceinline__ double exp2_64(double y, const double* pow) {
  const double shifted = y + 105553116266496.0;  // 1.5 * 2^46: whole 64ths in the low bits
  const double x = y - (shifted - 105553116266496.0);
  const int n = __double2loint(shifted);
  double s = kLn2 * kLn2 * kLn2 * kLn2 / 24.0;
  s = fma(s, x, kLn2 * kLn2 * kLn2 / 6.0);
  s = fma(s, x, kLn2 * kLn2 / 2.0);
  s = fma(s, x, kLn2);
  s = fma(s, x, 1.0) * pow[n & (kPow - 1)];
  return __hiloint2double(__double2hiint(s) + ((n & ~(kPow - 1)) << 14), __double2loint(s));
}

// NaN counts as -inf, +inf as the largest finite number
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -CUDART_INF_F), 3.402823466e38f); }
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// N numbers, aligned to as many bytes or to 16.
template <typename T, int N>
__device__ __forceinline__ void load_whole(const T* p, float (&x)[N]) {
  using Vec = std::conditional_t<N * sizeof(T) % 16 == 0, uint4, uint2>;
  static_assert(N * sizeof(T) % sizeof(Vec) == 0, "whole vectors");
  constexpr int kPer = sizeof(Vec) / sizeof(T);
#pragma unroll
  for (int v = 0; v < N / kPer; ++v) {
    const Vec raw = __ldg(reinterpret_cast<const Vec*>(p) + v);
    T t[kPer];
    memcpy(t, &raw, sizeof(Vec));
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[v * kPer + i] = to_float(t[i]);
  }
}
// The N numbers from element `at` on, which may be negative or end beyond n: those that are not there are `none`.
template <typename T, int N>
__device__ __forceinline__ void load(const T* row, int64_t at, int n, float none, float (&x)[N]) {
  constexpr size_t kAlign = N * sizeof(T) < 16 ? N * sizeof(T) : 16;
  if (at >= 0 && at + N <= n && reinterpret_cast<uintptr_t>(row + at) % kAlign == 0) {
    load_whole<T, N>(row + at, x);
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

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// into the same place of another CTA's shared memory
__device__ __forceinline__ void st_cluster_64(double* p, uint32_t rank, double v) {
  asm volatile("{\n\t.reg .b32 to;\n\tmapa.shared::cluster.u32 to, %0, %1;\n\tst.shared::cluster.f64 [to], %2;\n\t}" ::"r"(smem_u32(p)), "r"(rank), "d"(v)
               : "memory");
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

__device__ __forceinline__ float scale_of(float temperature) {  // log2(e) / T; not 0: of -inf that would be NaN
  return temperature > 0.f ? fminf(fmaxf(kLog2e / temperature, 1e-30f), 1e30f) : 0.f;
}

// Read once, in one place: a plain load was made twice, to save registers, and came from L1 the second time.
__device__ __forceinline__ uint4 stream_v4(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// 16 bytes of numbers
template <typename T>
struct Raw {
  static constexpr int N = 16 / sizeof(T);
  uint4 v;
  __device__ __forceinline__ float operator[](int i) const {
    const uint32_t w = sizeof(T) == 4 ? (&v.x)[i] : (&v.x)[i >> 1];
    if constexpr (std::is_same_v<T, float>) return __uint_as_float(w);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
    else return __half2float(__ushort_as_half(static_cast<uint16_t>(i & 1 ? w >> 16 : w & 0xFFFFu)));
  }
  __device__ __forceinline__ float largest() const {  // NaN are passed over
    if constexpr (std::is_same_v<T, float>) {
      return fmaxf(fmaxf((*this)[0], (*this)[1]), fmaxf((*this)[2], (*this)[3]));
    } else {
      using Two = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
      Two t[4];
      memcpy(t, &v, 16);
      const Two m = __hmax2(__hmax2(t[0], t[1]), __hmax2(t[2], t[3]));
      return fmaxf(to_float(m.x), to_float(m.y));
    }
  }
  // vector `at` of a row, -inf where there is nothing
  __device__ __forceinline__ void load(const T* row, int64_t at, int n) {
    if (at >= 0 && at + N <= n && (reinterpret_cast<uintptr_t>(row + at) & 15) == 0) {
      v = __ldg(reinterpret_cast<const uint4*>(row + at));
    } else {
      T t[N];
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = at + i >= 0 && at + i < n ? row[at + i] : T(-CUDART_INF_F);
      memcpy(&v, t, 16);
    }
  }
};

// Every CTA has an equal share of all rows' units: for each row of them the largest number and, relative to that, the sum of the exponentials.
// What it does for a number beside the load are seven instructions, one of them an exponential: 3/4 of the time that memory takes. 4.3 TB/s; at the 64
// registers that leave four CTAs on an SM the 16-bit instances spill 112 and 136 bytes (bf16, fp16) of the two sets of vectors.
// kAhead vectors, of the next row too, are on their way while as many are worked on. (Two sets of registers in turn: when one was copied to the
// other the compiler put the loads behind the work, to save registers, and load and work took turns.)
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) rows_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int N = Slice<T>::N;
  const fdma_verify_params& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t u0 = static_cast<int64_t>(blockIdx.x) * a.share, u1 = min(a.first_unit(p.tokens), u0 + a.share);
  int row = static_cast<int>(u0 / a.units), unit = static_cast<int>(u0 - a.first_unit(row));  // of the next vectors to be asked for
  int left = static_cast<int>(u1 - u0);  // units from there on
  const uint4* at;   // this thread's first vector there
  int full0, full1;  // vectors of the row that are whole
  auto begin_row = [&]() {
    const Slice<T> s(static_cast<const T*>(p.logits) + row * p.logits_row_stride, p.vocab, 0, 1);
    at = reinterpret_cast<const uint4*>(s.row - s.skip) + unit * kThreads + tid;
    full0 = s.skip > 0;
    full1 = (s.skip + p.vocab) / N;
  };
  struct Batch {
    Raw<T> x[kAhead];
    int row, unit, units;  // units = 0: no more
  };
  auto take = [&](Batch& t) {
    t.row = row;
    t.unit = unit;
    t.units = min(kAhead, min(left, a.units - unit));
    if (t.units <= 0) return;
    const int v0 = unit * kThreads;
    if (t.units == kAhead && v0 >= full0 && v0 + kAhead * kThreads <= full1) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) t.x[k].v = stream_v4(at + k * kThreads);
    } else {
      const Slice<T> s(static_cast<const T*>(p.logits) + row * p.logits_row_stride, p.vocab, 0, 1);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int v = v0 + k * kThreads + tid;
        t.x[k].load(s.row, k < t.units && v < s.end ? s.element(v) : -N, p.vocab);
      }
    }
    at += kAhead * kThreads;
    unit += t.units;
    left -= t.units;
    if (unit >= a.units && left > 0) {
      unit = 0;
      ++row;
      begin_row();
    }
  };
  auto factor = [&](int of) {
    if (!p.temperatures) return scale_of(p.temperature);
    int lo = 0, len = p.requests;  // the request that has the row: the first one that ends behind it, 32 of them at a time
    while (len > 1) {
      const int step = (len + 31) / 32, end = min(lo + (lane + 1) * step, lo + len);
      const int n = __popc(__ballot_sync(0xffffffffu, lane * step < len && p.cu_seqlens[end] <= of));
      const int to = min(lo + n * step, lo + len - 1);
      len = min(step, lo + len - to);
      lo = to;
    }
    return scale_of(p.temperatures[lo]);
  };
  Part mine{-CUDART_INF_F, 0.f, 0x7FFFFFFF};
  float c = 0.f;
  auto work = [&](const Batch& t) {
    float high = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) high = fmaxf(high, t.x[k].largest());
    high = clean(high);
    if (high > mine.top) {
      mine.sum = mine.top == -CUDART_INF_F ? 0.f : mine.sum * exp2f((mine.top - high) * c);
      mine.top = high;
      mine.at = t.unit;
    }
    if (c > 0.f && mine.top > -CUDART_INF_F) {
      const float b = -mine.top * c;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      const float2 c2 = make_float2(c, c), b2 = make_float2(b, b);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const float2 y = __ffma2_rn(make_float2(t.x[k][i], t.x[k][i + 1]), c2, b2);
          sum[(i >> 1) & 1] = __fadd2_rn(sum[(i >> 1) & 1], make_float2(fast_exp2(y.x), fast_exp2(y.y)));
        }
      float both = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      if (!(fabsf(b) <= kPlain) || !(both < CUDART_INF_F)) {  // large numbers, or NaN or infinities among them
        both = 0.f;
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
#pragma unroll
          for (int i = 0; i < N; ++i) both += exp2f((clean(t.x[k][i]) - mine.top) * c);
      }
      mine.sum += both;
    }
  };
  auto end_row = [&](int of) {  // what the warp has found in the row
    if (c == 0.f) {  // where: the lanes whose largest number is the warp's look it up, in the vectors that began at unit mine.at
      float top = mine.top;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      int found = 0x7FFFFFFF;
      if (top > -CUDART_INF_F && mine.top == top) {
        const Slice<T> s(static_cast<const T*>(p.logits) + of * p.logits_row_stride, p.vocab, 0, 1);
        for (int k = kAhead - 1; k >= 0; --k) {
          const int v = (mine.at + k) * kThreads + tid;
          Raw<T> x;
          x.load(s.row, v < s.end ? s.element(v) : -N, p.vocab);
#pragma unroll
          for (int i = N - 1; i >= 0; --i)
            if (clean(x[i]) == top) found = static_cast<int>(s.element(v)) + i;
        }
      }
      mine.at = found;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Part other{__shfl_xor_sync(0xffffffffu, mine.top, o), __shfl_xor_sync(0xffffffffu, mine.sum, o), __shfl_xor_sync(0xffffffffu, mine.at, o)};
      mine = join(mine, other, c);
    }
    const int slot = static_cast<int>(blockIdx.x - a.first_unit(of) / a.share);
    if (lane == 0) a.parts[(static_cast<int64_t>(of) * a.slots + slot) * kWarps + warp] = make_float4(mine.top, mine.sum, __int_as_float(mine.at), 0.f);
    mine = Part{-CUDART_INF_F, 0.f, 0x7FFFFFFF};
  };
  Batch one, two;
  begin_row();
  take(one);
  take(two);
  c = factor(one.row);
  while (true) {
    auto turn = [&](Batch& now, const Batch& then) {
      work(now);
      if (then.units <= 0 || then.row != now.row) {
        end_row(now.row);
        if (then.units <= 0) return false;
        c = factor(then.row);
      }
      take(now);
      return true;
    };
    if (!turn(one, two) || !turn(two, one)) break;
  }
}

// Inclusive sum over the lanes, in one order.
__device__ __forceinline__ double scan_64(double x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}
// Of numbers x >= 0 with the inclusive sums upto: the first lane whose sum is above the target, or where rounding leaves none the last that
// adds to the sum; -1: none does. before: the sum in front of it.
__device__ __forceinline__ int pick_64(double x, double upto, double target, double& before) {
  const uint32_t pass = __ballot_sync(0xffffffffu, x > 0.0 && upto > target), some = __ballot_sync(0xffffffffu, x > 0.0);
  const int at = pass ? __ffs(pass) - 1 : 31 - __clz(some);
  before = __shfl_sync(0xffffffffu, upto - x, at & 31);
  return at;
}

template <typename T, typename Q>
__global__ void __launch_bounds__(kThreads, 4) verify_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int N = Slice<T>::N;
  extern __shared__ double s_kept[];  // [kKept][kThreads]: sums of the threads' vectors
  __shared__ float s_top[kRows], s_logit[kRows], s_q[kRows], s_u[kRows];
  __shared__ int s_at[kRows], s_verdict[kRows];  // 0: rejected, 1: accepted, 2: open
  __shared__ int64_t s_draft[kRows];
  __shared__ double s_pow[kPow], s_warp[kWarps], s_all[2][kMaxCluster];  // sums of the warps; of the CTAs, for sums that follow one another in turn
  const fdma_verify_params& p = a.p;
  const int C = a.cluster, rank = static_cast<int>(blockIdx.x) % C, r = static_cast<int>(blockIdx.x) / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = p.vocab;
  cluster_arrive();  // (that a CTA has begun: its shared memory may be written to)
  const int first = max(0, min(p.cu_seqlens[r], p.tokens)), n = max(0, min(p.cu_seqlens[r + 1], p.tokens) - first);
  const int length = p.lengths[r];
  const float temperature = p.temperatures ? p.temperatures[r] : p.temperature;
  const bool lead = rank == 0 && tid == 0;
  if (n == 0 || (p.granted && !p.granted[r])) {  // (the whole cluster agrees)
    // A call may be made of such requests alone. It does not end before rows_kernel, whose parts lie in scratch that the caller has back then.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (lead) {
      p.accepted[r] = 0;
      p.next_tokens[r] = -1;
      p.lengths_out[r] = length;
    }
    cluster_wait();
    return;
  }
  if (tid < kPow) s_pow[tid] = exp_series(tid * (kLn2 / kPow) - (tid > kPow / 2 ? kLn2 : 0.0)) * (tid > kPow / 2 ? 2.0 : 1.0);
  const bool greedy = !(temperature > 0.f);
  const float c = scale_of(temperature);
  auto logits = [&](int row) { return static_cast<const T*>(p.logits) + (first + row) * p.logits_row_stride; };
  auto probs = [&](int row) { return static_cast<const Q*>(p.draft_probs) + (first + row) * p.probs_row_stride; };
  // Exponentials of a row: of its largest number about 1 (the rounding of `shift` is one factor for all), of what is below 2^-1000 of that, of
  // -inf and of NaN 0; +inf counts as the largest number. Without a branch: the numbers of a thread are worked on side by side. (scale: for
  // temperatures so low that shift would lose the point, 2^30 leaves nothing but the largest number, too.)
  struct Exp {
    float top;
    double scale, shift;
  };
  auto exp_of = [&](float top) {
    const double scale = greedy ? 0.0 : fmin(1.4426950408889634074 / static_cast<double>(temperature), 1073741824.0 / fmax(fabs(static_cast<double>(top)), 1e-30));
    return Exp{top, scale, -static_cast<double>(top) * scale};
  };
  auto e64 = [&](float x, const Exp& f) {
    const double y = fma(static_cast<double>(fminf(x, f.top)), f.scale, f.shift);
    const bool some = x >= -3.402823466e38f && static_cast<uint32_t>(__double2hiint(y)) < 0xC08F4000u;  // y > -1000
    const double e = exp2_64(y, s_pow);
    return some ? e : 0.0;
  };

  // A CTA's slice of a row is cut into a part for each warp, `each` x 32 vectors.
  auto part = [&](const Slice<T>& s) { return (s.end - s.first + kThreads - 1) / kThreads; };
  // What a draw weighs the N numbers x of a vector by, the first one number `at` of the row: exponentials; with `left` what the draft `gone` or
  // the drafter's q leave of the probabilities, given the exponentials' sum z.
  auto weights = [&](const Raw<T>& x, const float (&q)[N], int64_t at, const Exp& f, bool left, int64_t gone, double z, double (&e)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = e64(x[i], f);
    if (left && p.draft_probs) {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = fmax(fma(-static_cast<double>(fmaxf(q[i], 0.f)), z, e[i]), 0.0);
    } else if (left) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at + i == gone) e[i] = 0.0;
    }
  };
  int sums = 0;  // made so far
  // The weights' sum over the cluster, added up in one order; s_all[(sums - 1) & 1], s_warp and s_kept hold its parts.
  auto sum_up = [&](int row, float top, bool left, int64_t gone, double z) {
    const Slice<T> s(logits(row), V, rank, C);
    const int each = part(s);
    const bool with_probs = left && p.draft_probs;
    const Exp f = exp_of(top);
    double sum = 0.0;
    Raw<T> next;
    float next_q[N];
    const int v0 = s.first + warp * each * 32 + lane;  // this lane's first vector
    const uint4* next_x = reinterpret_cast<const uint4*>(s.row - s.skip) + v0;
    const Q* next_p = with_probs ? probs(row) + s.element(v0) : nullptr;
    const int full0 = s.skip > 0, full1 = min(s.end, (s.skip + V) / N);  // vectors that are whole
    const bool q_vectors = with_probs && (reinterpret_cast<uintptr_t>(next_p) % (N * sizeof(Q) < 16 ? N * sizeof(Q) : 16)) == 0;
    auto fetch = [&](int k) {
      const int v = v0 + k * 32;
      if (k < each && v >= full0 && v < full1) {
        next.v = __ldg(next_x);
        if (q_vectors) load_whole<Q, N>(next_p, next_q);
        else if (with_probs) load<Q, N>(probs(row), s.element(v), V, 0.f, next_q);
      } else {
        const int64_t at = k < each && v < s.end ? s.element(v) : -N;
        next.load(s.row, at, V);
        if (with_probs) load<Q, N>(probs(row), at, V, 0.f, next_q);
      }
      next_x += 32;
      if (with_probs) next_p += 32 * N;
    };
    fetch(0);
#pragma unroll 1
    for (int k = 0; k < each; ++k) {
      const Raw<T> x = next;
      const int64_t at = v0 + k * 32 < s.end ? s.element(v0 + k * 32) : -N;
      float q[N];
#pragma unroll
      for (int i = 0; i < N; ++i) q[i] = next_q[i];
      fetch(k + 1);
      double e[N], mine = 0.0;
      weights(x, q, at, f, left, gone, z, e);
#pragma unroll
      for (int i = 0; i < N; ++i) mine += e[i];
      if (k < kKept) s_kept[k * kThreads + tid] = mine;
      sum += mine;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();  // (s_warp is read no more)
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    double* const all = s_all[sums & 1];
    if (sums == 0) cluster_wait();  // every CTA has begun
    if (warp == 0) {
      double total = 0.0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) total += s_warp[w];
      if (lane < C) st_cluster_64(all + rank, lane, total);
    }
    ++sums;
    cluster_arrive();
    cluster_wait();
    return __shfl_sync(0xffffffffu, scan_64(lane < C ? all[lane] : 0.0, lane), 31);
  };

  int accepted = 0, row = -1;  // row: that the next token comes from
  float top = 0.f;
  int best = -1;
  double z = -1.0;
  for (int base = 0; row < 0; base += kRows) {
    const int rows = min(kRows, n - base);
    if (tid < rows) {  // what the verdicts need of the drafts
      const int j = tid;
      int64_t token = -1;
      if (base + j < n - 1) {
        const int at = first + base + j;
        token = p.id_bits == 64 ? static_cast<const int64_t*>(p.token_ids)[at + 1] : static_cast<const int32_t*>(p.token_ids)[at + 1];
        if (token < 0 || token >= V) token = -1;
        s_u[j] = p.uniforms[at];
        if (token >= 0) {
          s_logit[j] = clean(to_float(logits(base + j)[token]));
          s_q[j] = p.draft_probs ? fmaxf(to_float(probs(base + j)[token]), 0.f) : 1.f;
        }
      }
      s_draft[j] = token;
    }
    if (base == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    // ---- verdicts, by every CTA for itself: half a warp per row ----
    for (int j = tid >> 4; j < kRows; j += kThreads / 16) {
      const int half = lane & 15;
      Part all{-CUDART_INF_F, 0.f, 0x7FFFFFFF};
      if (j < rows) {
        const int64_t unit = a.first_unit(first + base + j);
        const int parts = static_cast<int>((unit + a.units - 1) / a.share - unit / a.share + 1) * kWarps;
        const float4* const src = a.parts + static_cast<int64_t>(first + base + j) * a.slots * kWarps;
        for (int i0 = half; i0 < parts; i0 += 64) {
          float4 f[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) f[k] = i0 + 16 * k < parts ? __ldcg(src + i0 + 16 * k) : make_float4(-CUDART_INF_F, 0.f, __int_as_float(0x7FFFFFFF), 0.f);
#pragma unroll
          for (int k = 0; k < 4; ++k) all = join(all, Part{f[k].x, f[k].y, __float_as_int(f[k].z)}, c);
        }
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        const Part other{__shfl_xor_sync(0xffffffffu, all.top, o), __shfl_xor_sync(0xffffffffu, all.sum, o), __shfl_xor_sync(0xffffffffu, all.at, o)};
        // the same in every lane and CTA: of two lanes the lower one's part first
        all = (lane & o) ? join(other, all, c) : join(all, other, c);
      }
      if (half == 0 && j < rows) {
        int verdict = 0;
        const int64_t token = s_draft[j];
        if (base + j < n - 1) {
          if (greedy) {
            verdict = token == all.at;
          } else if (token >= 0 && all.top > -CUDART_INF_F) {
            const float have = exp2f((s_logit[j] - all.top) * c), need = s_u[j] * s_q[j] * all.sum;
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
        z = sum_up(base + j, s_top[j], false, -1, 0.0);
        verdict = static_cast<double>(s_u[j]) * static_cast<double>(s_q[j]) * z < e64(s_logit[j], exp_of(s_top[j]));
        if (verdict) z = -1.0;
      }
      if (verdict) {
        ++accepted;
      } else {
        row = base + j;
        top = s_top[j];
        best = s_at[j] < V ? s_at[j] : -1;
      }
    }
    if (row < 0) __syncthreads();  // (the verdicts are read no more)
  }
  if (lead) {
    p.accepted[r] = accepted;
    p.lengths_out[r] = length - (n - 1 - accepted);
  }
  if (greedy || top == -CUDART_INF_F) {
    if (lead) p.next_tokens[r] = greedy && top > -CUDART_INF_F ? best : -1;
    if (sums == 0) cluster_wait();
    return;
  }
  // ---- the next token ----
  bool left = accepted < n - 1;
  if (left && p.draft_probs) {  // the drafter's numbers are on their way to L2 while the exponentials are summed up
    const Slice<T> s(logits(row), V, rank, C);
    const int64_t end = min(static_cast<int64_t>(V), s.element(s.end));
    for (int64_t i = max(int64_t{0}, s.element(s.first)) + tid * (128 / sizeof(Q)); i < end; i += kThreads * (128 / sizeof(Q)))
      asm volatile("prefetch.global.L2 [%0];" ::"l"(probs(row) + i));
  }
  if (z < 0.0) z = sum_up(row, top, false, -1, 0.0);
  const int64_t gone = left && !p.draft_probs ? s_draft[row % kRows] : -1;
  double total = z;
  if (left) {
    // Without the drafter's probabilities the sum loses the draft's own number, and so does the part it is in; where that leaves
    // too few bits it is made again.
    const double lost = gone >= 0 ? e64(s_logit[row % kRows], exp_of(top)) : 0.0;
    if (!p.draft_probs && z - lost > z * 0x1p-8) {
      total = z - lost;
      if (gone >= 0) {
        const Slice<T> s(logits(row), V, 0, C);
        const int v = static_cast<int>((gone + s.skip) / N), of_cta = max(s.end, 1), each_cta = of_cta;
        const int cta = v / each_cta, in_cta = v - cta * each_cta;
        const Slice<T> mine(logits(row), V, cta, C);
        const int each = part(mine), w = in_cta / (each * 32), k = in_cta % (each * 32) / 32, l = in_cta % 32;
        __syncthreads();  // (the sums are read no more)
        if (tid == 0) s_all[(sums - 1) & 1][cta] -= lost;
        if (cta == rank && tid == 0) {
          s_warp[w] -= lost;
          if (k < kKept) s_kept[k * kThreads + w * 32 + l] -= lost;
        }
        __syncthreads();
      }
    } else {
      total = sum_up(row, top, true, gone, z);
    }
    if (!(total > 0.0)) {  // the drafter is as sure of everything
      left = false;
      total = sum_up(row, top, false, -1, 0.0);
    }
  }
  // the CTA, warp and token where the running sum passes the target
  double target = static_cast<double>(p.uniforms[first + n - 1]) * total, before;
  const double of_cta = lane < C ? s_all[(sums - 1) & 1][lane] : 0.0;
  if (pick_64(of_cta, scan_64(of_cta, lane), target, before) != rank) return;
  target -= before;
  const double of_warp = lane < kWarps ? s_warp[lane] : 0.0;
  if (pick_64(of_warp, scan_64(of_warp, lane), target, before) != warp) return;
  target -= before;
  const Slice<T> s(logits(row), V, rank, C);
  const int each = part(s);
  int from = 0, to = each;  // vectors of each lane that it can be among
  if (each <= kKept) {
    double of_vector = 0.0;  // lane k: of the lanes' k-th vectors
    if (lane < each)
      for (int i = 0; i < 32; ++i) of_vector += s_kept[lane * kThreads + warp * 32 + ((i + lane) & 31)];
    from = max(0, pick_64(of_vector, scan_64(of_vector, lane), target, before));
    to = from + 1;
    target -= before;
  }
  const Exp f = exp_of(top);
  int token = -1;
  bool found = false;
  for (int k = from; k < to && !found; ++k) {
    const int v = s.first + (warp * each + k) * 32 + lane;
    const int64_t at = v < s.end ? s.element(v) : -N;
    Raw<T> x;
    float q[N];
    x.load(s.row, at, V);
    if (left && p.draft_probs) load<Q, N>(probs(row), at, V, 0.f, q);
    double e[N], sum = 0.0;
    weights(x, q, at, f, left, gone, z, e);
#pragma unroll
    for (int i = 0; i < N; ++i) sum += e[i];
    const double upto = scan_64(sum, lane);
    double run = upto - sum;
    int mine = -1;  // of this lane: the first token above the target, or the last that adds to the sum
    bool passed = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      run += e[i];
      if (!passed && e[i] > 0.0) {
        mine = static_cast<int>(at) + i;
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
    target -= __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) p.next_tokens[r] = token;
}

template <typename T, typename Q>
int launch(const VerifyArgs& a, cudaStream_t stream) {
  if (a.p.tokens > 0) {
    const int64_t total = static_cast<int64_t>(a.p.tokens) * a.units;
    rows_kernel<T><<<static_cast<unsigned>((total + a.share - 1) / a.share), kThreads, 0, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  auto kern = verify_kernel<T, Q>;
  constexpr int kSmem = kKept * kThreads * sizeof(double);
  static std::atomic<uint64_t> prepared{0}, wide{0};
  int st = allow_smem_once(reinterpret_cast<const void*>(kern), kSmem, prepared);
  if (!st && a.cluster > 8) st = allow_wide_clusters_once(reinterpret_cast<const void*>(kern), wide);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.p.requests) * a.cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // its CTAs look up the drafts while the last rows are streamed
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.p.tokens > 0 ? 2 : 1;  // (without rows what runs before it is somebody else's)
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

// CTAs that share a request: slices of no less than 1024 numbers, and no more CTAs than one and a half times those that run at once, four on an
// SM. 64 requests of 9 rows, 131072 numbers: 8 CTAs 82 us, 4 91, 16 96; 200 of 4, 50257 numbers in fp32: 4 CTAs 90, 2 110.
int pick_cluster(const fdma_verify_params& p) {
  int c = 1;
  while (c < kMaxCluster && p.vocab / (2 * c) >= 1024) c *= 2;
  while (c > 1 && static_cast<int64_t>(p.requests) * c > 6 * sm_count()) c /= 2;
  return c;
}
// Shares of the rows' units for as many CTAs as run at once, four on an SM.
void pick_shares(VerifyArgs& a) {
  const fdma_verify_params& p = a.p;
  const int bytes = p.dtype == FDMA_FP32 ? 4 : 2, n = 16 / bytes;
  // a row that does not begin on 16 bytes has a vector more
  const bool aligned = (reinterpret_cast<uintptr_t>(p.logits) | static_cast<uint64_t>(p.logits_row_stride) * bytes) % 16 == 0;
  a.units = static_cast<int>((static_cast<int64_t>(p.vocab) + (aligned ? 0 : n - 1) + static_cast<int64_t>(n) * kThreads - 1) / (static_cast<int64_t>(n) * kThreads));
  const int64_t total = std::max<int64_t>(static_cast<int64_t>(p.tokens) * a.units, 1), ctas = 4 * sm_count();
  a.share = static_cast<int>((total + ctas - 1) / ctas);
  if (a.share > kAhead) a.share = (a.share + kAhead - 1) / kAhead * kAhead;
  a.slots = (a.units - 1) / a.share + 2;
}
int check_verify(const fdma_verify_params* pp) {
  if (!pp) return FDMA_ERR_BAD_ARG;
  const fdma_verify_params& p = *pp;
  if (p.requests < 0 || p.tokens < 0 || p.vocab <= 0) return FDMA_ERR_BAD_ARG;
  if (!known(p.dtype) || (p.draft_probs && !known(p.probs_dtype)) || (p.id_bits != 32 && p.id_bits != 64)) return FDMA_ERR_UNSUPPORTED;
  if (p.requests > (1 << 26) || p.vocab > 0x7FFFFFFF - 64) return FDMA_ERR_UNSUPPORTED;
  return 0;
}

}  // namespace
}  // namespace fdma

using namespace fdma;

extern "C" size_t fdma_verify_drafts_workspace_bytes(const fdma_verify_params* p) {
  if (check_verify(p)) return 0;
  VerifyArgs a;
  a.p = *p;
  pick_shares(a);
  return static_cast<size_t>(p->tokens) * a.slots * kWarps * sizeof(float4);
}

extern "C" int fdma_verify_drafts(const fdma_verify_params* pp, void* stream) {
  const int st = check_verify(pp);
  if (st) return st;
  const fdma_verify_params& p = *pp;
  if (p.requests == 0) return FDMA_OK;
  if (!p.cu_seqlens || !p.lengths || !p.accepted || !p.next_tokens || !p.lengths_out) return FDMA_ERR_BAD_ARG;
  if (p.tokens > 0 && (!p.logits || !p.token_ids || !p.uniforms)) return FDMA_ERR_BAD_ARG;
  if (p.tokens > 0 && (!p.workspace || p.workspace_bytes < fdma_verify_drafts_workspace_bytes(pp) || (reinterpret_cast<uintptr_t>(p.workspace) & 15)))
    return FDMA_ERR_WORKSPACE;
  VerifyArgs a;
  a.p = p;
  if (!p.draft_probs) a.p.probs_dtype = FDMA_FP32;
  a.cluster = pick_cluster(p);
  pick_shares(a);
  a.parts = static_cast<float4*>(p.workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p.dtype) {
    case FDMA_BF16: return launch_t<__nv_bfloat16>(a, s);
    case FDMA_FP16: return launch_t<__half>(a, s);
    default: return launch_t<float>(a, s);
  }
}
