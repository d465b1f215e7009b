// Rotary positions on queries and keys, forward and backward (the same rotation by the negative angle).
//
//   y1 = a (x1 cos - x2 sin),  y2 = a (x2 cos + x1 sin),  angle = position * frequency
//
// Memory-bound: every element is read once and written once, three operations each. A warp takes a token: one evaluation of sine
// and cosine per frequency, whatever the number of heads, then the heads in 16-byte vectors (rotate_tokens in fdma_rotary.cuh).
#include "fdma_rotary.cuh"

namespace fdma {
namespace {

template <typename T, int N, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryWarps * 32, 4) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) float2 s_factors[];
  const int warp = threadIdx.x >> 5;
  rotate_tokens<T, N, kInterleaved>(a, static_cast<int64_t>(blockIdx.x) * kRotaryWarps + warp, s_factors + warp * rotary_warp_pairs<N>(a));
}

constexpr int kMaxRotaryDim = 4096;  // a CTA's factors are held in 160 KB, 192 KB in fp32

template <typename T, int N, bool kInterleaved>
int launch(const fdma_rotary_params& p, cudaStream_t stream) {
  const RotaryArgs a = rotary_args(p, N);
  const int64_t ctas = (a.groups + kRotaryWarps - 1) / kRotaryWarps;
  if (ctas > 0x7FFFFFFF) return FDMA_ERR_UNSUPPORTED;
  const size_t smem = rotary_smem<N>(a);
  if (smem > 48 * 1024) {
    static std::atomic<uint64_t> prepared{0};
    const int most = kRotaryWarps * factor_pitch<N>(kMaxRotaryDim / 2) * static_cast<int>(sizeof(float2));
    const int st = allow_smem_once(reinterpret_cast<const void*>(rotary_kernel<T, N, kInterleaved>), most, prepared);
    if (st) return st;
  }
  rotary_kernel<T, N, kInterleaved><<<static_cast<unsigned>(ctas), kRotaryWarps * 32, smem, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int launch_t(const fdma_rotary_params& p, cudaStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  if (rotary_units_fit(p.d, p.rotary_dim, N) && rotary_aligned16(p, sizeof(T)))
    return p.interleaved ? launch<T, N, true>(p, stream) : launch<T, N, false>(p, stream);
  return p.interleaved ? launch<T, 1, true>(p, stream) : launch<T, 1, false>(p, stream);
}

}  // namespace
}  // namespace fdma

using namespace fdma;

extern "C" int fdma_rotary(const fdma_rotary_params* pp, void* stream_) {
  if (!pp) return FDMA_ERR_BAD_ARG;
  const fdma_rotary_params& p = *pp;
  if (!p.q || !p.q_out || !p.turns || p.b < 0 || p.seqlen < 0 || p.h <= 0 || p.h_k < 0 || p.d <= 0) return FDMA_ERR_BAD_ARG;
  if (p.h_k && (!p.k || !p.k_out)) return FDMA_ERR_BAD_ARG;
  if (p.rotary_dim <= 0 || p.rotary_dim % 2 || p.rotary_dim > p.d) return FDMA_ERR_BAD_ARG;
  if (p.positions && p.position_bits != 32 && p.position_bits != 64) return FDMA_ERR_BAD_ARG;
  if (p.rotary_dim > kMaxRotaryDim) return FDMA_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(p.h + p.h_k) * p.d > (1 << 24)) return FDMA_ERR_UNSUPPORTED;
  if (p.b == 0 || p.seqlen == 0) return FDMA_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  switch (p.dtype) {
    case FDMA_BF16: return launch_t<__nv_bfloat16>(p, stream);
    case FDMA_FP16: return launch_t<__half>(p, stream);
    case FDMA_FP32: return launch_t<float>(p, stream);
    default: return FDMA_ERR_UNSUPPORTED;
  }
}
