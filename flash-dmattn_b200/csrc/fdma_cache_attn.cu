// Attention over the paged 8-bit cache.
//
//   x_j = scale * q . k_j + bias_j over the visible keys j,  out = sum_j e^(x_j - max) v_j / sum_j e^(x_j - max),
//   k_j = k_scale[block, head] * e4m3, v_j likewise
//
// Few queries over many keys: HBM-bound, 2 d bytes per key and kv head. What follows from that:
//  * The queries of a request that share a kv head -- new tokens x query heads -- are the eight columns of mma.m16n8k16 (of two, when
//    there are more), so a key is read once for all of them, and the rows are full: 16 keys of K Q^T, 16 elements of V^T P^T.
//    (With the queries as the 16 rows half of each product, of its accumulators and of their moves was for nothing: 461 instructions
//    for 16 keys, 349 so.) The products are in fp16 with 32-bit sums: e4m3 numbers are fp16 numbers (one conversion instruction for
//    two), bf16 queries become fp16 after a power of two per row (exact up to 2^-29 of the row's largest), and scales, being powers
//    of two or common to a product, go into the scores and the softmax's exponents.
//  * A unit of work is a (request, kv head, tile of 8 or 16 rows), made of chunks of 64 keys. The chunks of all units form one row;
//    every CTA takes an equal part of it, however long the requests are, and starts and ends in the middle of a unit where it
//    must. Such partial results go through scratch and a second kernel; units that one CTA finishes are written directly.
//  * Where units are few and short, latency is what counts: a unit is shared by the CTAs of a cluster (kCluster), which join their sums
//    through each other's shared memory. No second kernel, and no sums over the requests before the first load. 1 request of 4096
//    tokens, 32 heads over 8, d = 128: 7.7 us in a graph, 12.2 with equal shares and the second kernel; 50 of 1000, 8 over 2: 9.5, 13.7.
//  * A warp of the CTA copies chunks to shared memory by TMA, three ahead; four warps take 16 keys of each. The 128-byte swizzle
//    and the order in which keys are assigned to the columns of the products (`key_row`) make all reads free of bank conflicts:
//    K fragments are 16-byte reads of a key's row, V fragments 4-byte reads of four keys whose bytes are then paired.
//  * With a list of kept keys the warps gather their 16 rows themselves with cp.async into the same layout.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>

#include "fdma_internal.h"
#include "fdma_ptx.cuh"

namespace fdma {

namespace {

constexpr int kChunk = 64;
constexpr int kWarps = 4;  // that compute; each has 16 keys of a chunk
constexpr int kSlice = kChunk / kWarps;
constexpr int kHeld = 128;  // requests whose work a CTA holds in shared memory
constexpr int kMinShare = 2;  // chunks per CTA
constexpr int kMostCluster = 16, kMostClusterChunks = 20;  // CTAs that share a unit (kCluster), and chunks of one of them
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPScale = 16384.f;  // probabilities in fp16: normal numbers down to 2^-28

struct AttnArgs {
  fdma_cache_attention_params p;
  int shift, group, row_shift;  // log2 of the block size, and of the rows of a tile
  uint32_t group_inverse, h_k_inverse;  // floor(2^32 / x), at most 2^32 - 1
  int list_chunks;         // kept keys: chunks per unit; 0: from cu_chunks
  int32_t* pre;            // sums of the requests' chunks x tiles, requests + 1: for more than kHeld requests made before, for fewer
                           // by the first CTA, for the second kernel
  int ctas;                // along the row of chunks
  float scale_log2;
  bool q_vec;              // queries in 16-byte vectors
  const int32_t* prompts;  // not null: rows of no request are written already, and if it points to 0, those of requests with
                           // kPromptTokens or more as well (one word: look-ups that read three more took 10 us of 340)
  int cluster, tiles;      // CTAs that share a unit, and tiles of a request, where there are few units (kCluster)
  bool merge_requests;     // CTAs of the second kernel: kPromptTokens - 1 for each request, not one for every token
  float* partial;          // [cta][2][rows][D + 4]: sums over the values, then maximum, sum and the maximum's exponent
  int* status;
};

// Where the work lies: unit (request, kv head, tile) has the chunks [start, start + n) of the row.
struct Unit {
  int r, hk, tile, n;
  int64_t start;
};
// Queries and keys of a request, made safe against plans that do not fit the call.
struct Request {
  int token0, n, length, rows, chunks;  // rows = -1: done already
};

// lowest key row of a slice's eight keys for column n of the products: pairs of lanes that read K together, and lanes that read
// V together, then fall into different banks
__device__ __forceinline__ int key_row(int n) { return n & 1 ? (((n >> 1) ^ 2) << 1) | 1 : n; }

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Sets the NaN among four e4m3 numbers to 0; whether there was one.
__device__ __forceinline__ uint32_t drop_nan(uint32_t& x) {
  const uint32_t nan = ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  x &= ~((nan >> 7) * 0xFFu);
  return nan != 0;
}
// An 8 x 8 matrix of 16-bit numbers, a row per four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
template <int kOffset>
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(v) : "r"(addr), "n"(kOffset) : "memory");
  return v;
}
__device__ __forceinline__ void cp_async16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <bool kBf16>
__device__ __forceinline__ float raw_to_f(uint16_t u) {
  if (kBf16) return __uint_as_float(static_cast<uint32_t>(u) << 16);
  return __half2float(__ushort_as_half(u));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (kBf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) { return pack2<false>(lo, hi); }
// In units of log2. The lowest finite number of a type stays finite, so that a row of nothing else is an average and not empty.
__device__ __forceinline__ float bias_log2(float b) {
  const float x = b * kLog2e;
  return fabsf(x) > 3.0e38f && fabsf(b) != CUDART_INF_F ? copysignf(3.0e38f, b) : x;
}
// Scales below 2^-100 stand for zeros: the keys count in the softmax's sum (which a smaller scale could carry out of range: it is
// held in units of the probabilities times the V scales), and their values do not count.
__device__ __forceinline__ float value_scale(float x) { return x < 0x1p-100f ? 0x1p-101f : x; }
__device__ __forceinline__ float p_scale(float exponent) { return exponent < -100.f ? 0.f : kPScale; }
__device__ __forceinline__ float exponent_of(float x) { return static_cast<float>(static_cast<int>(__float_as_uint(x) >> 23) - 127); }
// A running maximum over scores times V scales, 2^(m + z): the score m and the scale's exponent z are kept apart, because a bias can make
// m so large that the sum would lose z, and the values of blocks with other scales would then count by the wrong factor. Differences
// are small where they matter: of equal scores exactly 0.
struct Peak {
  float m, z;
};
// No key seen yet: below any score of one that is (see bias_log2), and finite, so that differences are numbers.
constexpr float kNone = -3.2e38f;
// log2 of a's ratio to b
__device__ __forceinline__ float above(const Peak& a, const Peak& b) { return (a.m - b.m) + (a.z - b.z); }
__device__ __forceinline__ Peak higher(const Peak& a, const Peak& b) { return above(b, a) > 0.f ? b : a; }
// what sums up to `from` are multiplied by in sums up to `to`, which is no lower
__device__ __forceinline__ float rescale(const Peak& from, const Peak& to) { return exp2f(above(from, to)); }
__device__ __forceinline__ Peak shuffled(const Peak& x, int mask) {
  return Peak{__shfl_xor_sync(0xffffffffu, x.m, mask), __shfl_xor_sync(0xffffffffu, x.z, mask)};
}
// Of eight lanes.
__device__ __forceinline__ float largest8(float x) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
// (lanes that compared in different orders may hold different ones of two equal peaks)
__device__ __forceinline__ Peak of_lane(const Peak& x, int lane) {
  return Peak{__shfl_sync(0xffffffffu, x.m, lane), __shfl_sync(0xffffffffu, x.z, lane)};
}

__device__ __forceinline__ Request load_request(const AttnArgs& a, int r) {
  const fdma_cache& c = a.p.c;
  Request q;
  const int first = c.cu_seqlens[r], end = c.cu_seqlens[r + 1], chunk0 = c.cu_chunks[r], chunk1 = c.cu_chunks[r + 1];
  q.length = c.lengths[r];
  q.token0 = max(0, first);
  q.n = max(0, min(end, c.tokens) - q.token0);
  q.chunks = max(0, chunk1 - chunk0);
  q.rows = q.chunks ? min(q.n, a.p.max_seqlen_q) * a.group : 0;  // no chunks: refused
  if (a.prompts && q.n >= kPromptTokens && *a.prompts == 0) q.rows = -1;
  if (a.list_chunks) q.chunks = a.list_chunks;
  return q;
}

// x / y and the remainder, given floor(2^32 / y): the product is at most one too small.
__device__ __forceinline__ uint2 divide(uint32_t x, uint32_t y, uint32_t inverse) {
  uint32_t quot = __umulhi(x, inverse), rem = x - quot * y;
  if (rem >= y) {
    ++quot;
    rem -= y;
  }
  return make_uint2(quot, rem);
}
// Both positive. (A 64-bit division is a few hundred cycles.)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
}
__device__ __forceinline__ int tiles_of(const AttnArgs& a, int rows) { return rows > 0 ? (rows + (1 << a.row_shift) - 1) >> a.row_shift : 0; }
// (token, head) of a request's row
__device__ __forceinline__ uint2 token_head(const AttnArgs& a, int row) { return divide(row, a.group, a.group_inverse); }

// The units in the order of their chunks. Up to kHeld requests: their data and the sums of their chunks x tiles are held in shared
// memory. More: the sums are in global memory, and the data is read where it is needed.
struct Held {
  int pre[kHeld + 1], token0[kHeld], n[kHeld], length[kHeld], rows[kHeld], chunks[kHeld], warp[4];
};
struct Cursor {
  int r, hk, tile;
};
struct Units {
  const AttnArgs& a;
  const Held* held;  // null: too many requests
  __device__ const int32_t* pre() const { return held ? held->pre : a.pre; }
  __device__ int64_t total() const { return static_cast<int64_t>(pre()[a.p.c.requests]) * a.p.c.h_k; }
  __device__ Request request(int r) const {
    if (!held) return load_request(a, r);
    return Request{held->token0[r], held->n[r], held->length[r], held->rows[r], held->chunks[r]};
  }
  __device__ Unit of(const Cursor& x, const Request& q) const {
    Unit u;
    u.r = x.r; u.hk = x.hk; u.tile = x.tile;
    u.n = q.chunks;
    u.start = static_cast<int64_t>(pre()[x.r]) * a.p.c.h_k + (static_cast<int64_t>(x.hk) * tiles_of(a, q.rows) + x.tile) * q.chunks;
    return u;
  }
  // the unit of chunk w, w < total(), and its request; the same w in all lanes of a warp
  __device__ Cursor at(int64_t w, Request& q) const {
    const fdma_cache& c = a.p.c;
    const int64_t per_head = w >> 32 ? w / c.h_k : divide(static_cast<uint32_t>(w), c.h_k, a.h_k_inverse).x;
    int r = 0;  // requests that end at or before it
    if (held) {
#pragma unroll
      for (int i = 0; i < kHeld; i += 32) {
        const int at = i + (threadIdx.x & 31);
        r += __popc(__ballot_sync(0xffffffffu, at < c.requests && held->pre[at + 1] <= per_head));
      }
    } else {
      int hi = c.requests - 1;
      while (r < hi) {
        const int mid = (r + hi) >> 1;
        if (a.pre[mid + 1] > per_head) hi = mid;
        else r = mid + 1;
      }
    }
    r = min(r, c.requests - 1);
    q = request(r);
    const int tiles = max(tiles_of(a, q.rows), 1);
    const int i = static_cast<int>(quotient(max(w - static_cast<int64_t>(pre()[r]) * c.h_k, int64_t{0}), max(q.chunks, 1)));
    return tiles == 1 ? Cursor{r, i, 0} : Cursor{r, i / tiles, i % tiles};
  }
  // the unit behind, whose request is q then; past the last one x.r == requests
  __device__ void advance(Cursor& x, Request& q) const {
    if (++x.tile < tiles_of(a, q.rows)) return;
    x.tile = 0;
    if (++x.hk < a.p.c.h_k) return;
    x.hk = 0;
    while (++x.r < a.p.c.requests) {
      q = request(x.r);
      if (q.chunks > 0 && q.rows > 0) return;
    }
  }
};
// All threads of a CTA of at least 128.
__device__ __forceinline__ Units make_units(const AttnArgs& a, Held& h) {
  const int R = a.p.c.requests;
  if (R > kHeld) return Units{a, nullptr};
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int w = 0;
  if (tid < R) {
    const Request q = load_request(a, tid);
    h.token0[tid] = q.token0; h.n[tid] = q.n; h.length[tid] = q.length; h.rows[tid] = q.rows; h.chunks[tid] = q.chunks;
    w = q.chunks * tiles_of(a, q.rows);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  if (lane == 31 && warp < 4) h.warp[warp] = w;
  __syncthreads();
  if (tid < kHeld) {
    for (int i = 0; i < warp; ++i) w += h.warp[i];
    h.pre[tid + 1] = w;
    if (tid == 0) h.pre[0] = 0;
  }
  __syncthreads();
  return Units{a, &h};
}
// The same of a CTA that knows its unit.
struct OneUnit {
  const AttnArgs& a;
  Cursor x;
  Request q;
  __device__ Unit of(const Cursor&, const Request&) const { return Unit{x.r, x.hk, x.tile, q.chunks, 0}; }
  __device__ Cursor at(int64_t, Request& request) const {
    request = q;
    return x;
  }
  __device__ void advance(Cursor& at, Request&) const { at.r = a.p.c.requests; }
};
__device__ __forceinline__ OneUnit make_one_unit(const AttnArgs& a) {
  const int slot = static_cast<int>(blockIdx.x) / a.cluster, per_request = a.p.c.h_k * a.tiles;
  Cursor x;
  x.r = slot / per_request;
  x.hk = (slot - x.r * per_request) / a.tiles;
  x.tile = slot - (x.r * a.p.c.h_k + x.hk) * a.tiles;
  OneUnit u{a, x, load_request(a, x.r)};
  if (a.list_chunks && a.p.kept_count) {
    const int kept = a.p.kept_count[x.r * a.p.count_batch_stride + x.hk * a.p.count_head_stride];
    u.q.chunks = (max(0, min(kept, a.p.kept_capacity)) + kChunk - 1) / kChunk;
  }
  return u;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
// of another CTA of the cluster
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
__device__ __forceinline__ int64_t share_of(int64_t total, int ctas) { return max(static_cast<int64_t>(kMinShare), quotient(total + ctas - 1, ctas)); }

template <int D, int ROWS, bool kGather>
struct Layout {
  static constexpr int kHalves = D > 128 ? 2 : 1;                   // 128-byte tiles side by side
  static constexpr int kTileBytes = kChunk * 128 * kHalves;         // K or V of a chunk
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = D > 128 ? 2 : ROWS > 8 ? 4 : 3;
  static constexpr int kSteps = D / 16;                             // k steps of Q K^T
  static constexpr int kQBytes = ROWS / 8 * kSteps * 256;
  static constexpr int kBufFloats = ROWS * D;                       // one warp's sums
  static constexpr int kBufs = D > 128 ? 1 : 2;
  static constexpr int kRing = 0;
  static constexpr int kQ = kRing + kStages * kStageBytes;
  static constexpr int kBuf = kQ + kQBytes;
  static constexpr int kTotal = kBuf + kBufs * kBufFloats * 4 + 1024;
  static constexpr int kThreads = kWarps * 32 + (kGather ? 0 : 32);
  // Per SM. Three with 16 rows, at 128 registers, spill: 8 requests of up to 65536 tokens, 4 new ones each, 32 heads over 8, d = 128:
  // 105 us, two 93.
  static constexpr int kCtas = D > 128 || ROWS > 8 ? 2 : 3;
};

// kBias: with a bias, dense (without one the loop is shorter by its loads: 14.2 us instead of 14.7 for 16 requests of drafts). With a list
// of kept keys the bias is looked for when it runs.
template <int D, int ROWS, bool kGather, bool kBf16, bool kCluster, bool kBias>
__global__ void __launch_bounds__(Layout<D, ROWS, kGather>::kThreads, Layout<D, ROWS, kGather>::kCtas)
cache_attend_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using L = Layout<D, ROWS, kGather>;
  constexpr int kTiles = ROWS / 8;                     // of eight queries
  constexpr bool kQHeld = kTiles * L::kSteps <= 8;     // queries in registers
  extern __shared__ unsigned char s_raw[];
  __shared__ __align__(8) uint64_t s_full[L::kStages], s_empty[L::kStages];
  // of a slice: 1 if its block is there, K scale, exponent of the V scale, its reciprocal; of a kept key: bias (-inf: not there),
  // K scale, exponent of the V scale, position
  __shared__ float4 s_meta[L::kStages][kGather ? kChunk : kWarps];
  __shared__ Held s_held;
  // kCluster: maximum, sum and the maximum's exponent of this CTA's part; the sums over the values are in s_buf
  __shared__ __align__(16) float4 s_part[ROWS];
  __shared__ float s_row_scale[ROWS], s_l[kWarps][ROWS];
  __shared__ Peak s_m[kWarps][ROWS];
  __shared__ int s_abort;
  unsigned char* smem = align_smem_1024(s_raw);
  const fdma_cache_attention_params& p = a.p;
  const fdma_cache& c = p.c;
  const bool biased = kGather ? p.bias != nullptr : kBias;
  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    s_abort = 0;
    if (!kGather) {
      for (int i = 0; i < L::kStages; ++i) {
        mbar_init(&s_full[i], 2);  // the copies, and the scales
        mbar_init(&s_empty[i], kWarps);
      }
      fence_mbar_init();
    }
  }
  if (kGather && c.d < D)  // columns beyond the head dim stay zero in every stage
    for (int i = tid; i < L::kStages * L::kStageBytes / 16; i += L::kThreads) reinterpret_cast<uint4*>(smem + L::kRing)[i] = make_uint4(0, 0, 0, 0);
  const auto units = [&] {
    if constexpr (kCluster) return make_one_unit(a);
    else return make_units(a, s_held);
  }();
  if (kCluster && tid < ROWS) s_part[tid] = make_float4(kNone, 0.f, 0.f, 0.f);
  __syncthreads();
  int64_t w0, w1;
  if constexpr (kCluster) {
    const int n = units.q.rows > units.x.tile * ROWS ? units.q.chunks : 0, rank = static_cast<int>(cluster_rank()), shift = 31 - __clz(a.cluster);
    w0 = static_cast<int64_t>(n) * rank >> shift;
    w1 = static_cast<int64_t>(n) * (rank + 1) >> shift;
  } else {
    if (blockIdx.x == 0 && units.held)
      for (int i = tid; i <= c.requests; i += L::kThreads) a.pre[i] = s_held.pre[i];
    const int64_t total = units.total(), share = share_of(total, a.ctas);
    w0 = min(total, blockIdx.x * share);
    w1 = min(total, w0 + share);
    if (w0 >= w1) return;
  }
  const WaitCtl ctl{&s_abort, a.status};

  if (!kGather && warp == kWarps) {
    // ---- the copying warp: lanes look up the blocks and scales of eight chunks at a time, four 16-key slices each ----
    const int pages = max(1, kChunk >> a.shift), rows_per_copy = min(kChunk, 1 << a.shift);
    Request lane_q;
    Cursor at = units.at(w0, lane_q);  // of this lane's chunk, from here on
    auto look_up = [&](int64_t w, int& block, int& row, int& hk, float& ks, float& vs, bool& used) {
      block = -1;
      row = hk = 0;
      ks = vs = 0.f;
      used = false;
      if (w < w1) {
        Unit u = units.of(at, lane_q);
        while (w >= u.start + u.n) {
          units.advance(at, lane_q);
          if (at.r >= c.requests) return;
          u = units.of(at, lane_q);
        }
        hk = u.hk;
        used = lane_q.rows > u.tile * ROWS;
        const int pos = static_cast<int>(w - u.start) * kChunk + (lane & 3) * kSlice;
        if (used && pos < min(lane_q.length, p.max_seqlen_k) && (pos >> a.shift) < c.width) {
          block = c.table[static_cast<int64_t>(u.r) * c.width + (pos >> a.shift)];
          row = pos & ((1 << a.shift) - 1);
          if (block < 0 || block >= c.num_blocks) block = -1;
        }
        if (block >= 0) {
          ks = __ldg(c.k_scale + static_cast<int64_t>(block) * c.h_k + hk);
          vs = __ldg(c.v_scale + static_cast<int64_t>(block) * c.h_k + hk);
        }
      }
    };
    int block, row, hk, n_block, n_row, n_hk;
    float ks, vs, n_ks, n_vs;
    bool used, n_used;
    look_up(w0 + (lane >> 2), n_block, n_row, n_hk, n_ks, n_vs, n_used);
    int st = 0;
    uint32_t phase = 0;
    int issued = 0;
    for (int64_t w = w0; w < w1; w += 8) {
      block = n_block; row = n_row; hk = n_hk; ks = n_ks; vs = n_vs; used = n_used;
      for (int i = 0; i < 8 && w + i < w1; ++i) {
        // the next eight are looked up, three dependent loads, when the ring has been filled from these
        if (i == L::kStages - 1) look_up(w + 8 + (lane >> 2), n_block, n_row, n_hk, n_ks, n_vs, n_used);
        if (!__shfl_sync(0xffffffffu, used, i * 4)) continue;  // no rows of this unit in this row tile
        mbar_wait(&s_empty[st], phase ^ 1, ctl, 701);
        const int hk_i = __shfl_sync(0xffffffffu, hk, i * 4);
        unsigned char* dst = smem + L::kRing + st * L::kStageBytes;
        uint32_t bytes = 0;
        int blocks[4], rows[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int first = g * (4 / pages);  // the page's first slice
          blocks[g] = g < pages ? __shfl_sync(0xffffffffu, block, (i * 4 + first) & 31) : -1;
          rows[g] = __shfl_sync(0xffffffffu, row, (i * 4 + first) & 31);
          if (blocks[g] >= 0) bytes += 2u * rows_per_copy * 128 * L::kHalves;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(&s_full[st], bytes);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (blocks[g] < 0) continue;
            const int at_block = blocks[g] * c.h_k + hk_i;
#pragma unroll
            for (int x = 0; x < L::kHalves; ++x) {
              unsigned char* to = dst + x * kChunk * 128 + g * rows_per_copy * 128;
              tma_load_4d(to, &map_k, &s_full[st], x * 128, rows[g], at_block, 0);
              tma_load_4d(to + L::kTileBytes, &map_v, &s_full[st], x * 128, rows[g], at_block, 0);
            }
          }
        }
        if ((lane >> 2) == i) {
          const float v = value_scale(vs);
          s_meta[st][lane & 3] = make_float4(block >= 0 ? 1.f : 0.f, ks, exponent_of(v), block >= 0 ? __frcp_rn(v) : 0.f);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_full[st]);
        ++issued;
        if (++st == L::kStages) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    // after a wait that gave up: the copies in flight land before the CTA ends
    if (s_abort) {
      for (int i = 0; i < min(issued, L::kStages); ++i) {
        if (st == 0) phase ^= 1;
        st = st == 0 ? L::kStages - 1 : st - 1;
        mbar_wait_limit(&s_full[st], phase, WaitCtl{&s_abort, a.status}, 703, 1000000ull);
      }
    }
    if (kCluster) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  // ---- the computing warps ----
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + L::kRing + warp * kSlice * 128;
  // K: row key_row(g), 16-byte piece t (^ 4 for the second four); V: rows key_row(2 t), key_row(2 t + 1), word g of 32 columns
  const uint32_t k_at = key_row(g) * 128 + ((t ^ (key_row(g) & 7)) << 4);
  const int r0 = key_row(2 * t), r1 = key_row(2 * t + 1);
  const uint32_t v_at0 = L::kTileBytes + r0 * 128 + (((g >> 2) ^ (r0 & 7)) << 4) + (g & 3) * 4;
  const uint32_t v_at1 = L::kTileBytes + r1 * 128 + (((g >> 2) ^ (r1 & 7)) << 4) + (g & 3) * 4;
  const uint32_t q_at = smem_u32(smem) + L::kQ + lane * 8;
  float* const s_buf = reinterpret_cast<float*>(smem + L::kBuf);
  int st = 0;
  uint32_t phase = 0;
  int64_t w = w0;
  Request q;
  for (Cursor at = units.at(w0, q); w < w1 && at.r < c.requests; units.advance(at, q)) {
    const Unit u = units.of(at, q);
    const int64_t unit_end = max(u.start + u.n, w + 1);
    const int first = static_cast<int>(w - u.start), last = static_cast<int>(min(unit_end, w1) - u.start);
    const int row0 = u.tile * ROWS;
    w = min(unit_end, w1);
    const int nrows = min(ROWS, q.rows - row0);
    if (nrows <= 0) continue;
    const int length = min(q.length, p.max_seqlen_k);
    // oldest key that not every row sees
    const int sure = p.is_causal ? min(length, q.length - q.n + static_cast<int>(token_head(a, row0).x) + 1) : length;

    // queries: eight threads a row, to fp16 in the order of the fragments
    consumers_sync();
    for (int rr = tid >> 3; rr < ROWS; rr += 16) {
      constexpr int E = D / 8;  // elements per thread, in 16-byte vectors vec * 8 + part
      const int part = tid & 7, row = row0 + rr;
      uint32_t x[E / 2];
      float most = 0.f;
      const bool there = rr < nrows;
      const uint16_t* src = static_cast<const uint16_t*>(p.query);
      const uint2 th = token_head(a, row);
      if (there) src += static_cast<int64_t>(q.token0 + th.x) * p.query_row_stride + (u.hk * a.group + th.y) * p.query_head_stride;
#pragma unroll
      for (int e = 0; e < E / 8; ++e) {
        const int at = (e * 8 + part) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (there && at < c.d) {
          if (a.q_vec) {
            v = *reinterpret_cast<const uint4*>(src + at);
          } else {
            uint32_t y[4];
            for (int j = 0; j < 4; ++j) y[j] = src[at + 2 * j] | static_cast<uint32_t>(src[at + 2 * j + 1]) << 16;
            v = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
        x[4 * e] = v.x; x[4 * e + 1] = v.y; x[4 * e + 2] = v.z; x[4 * e + 3] = v.w;
      }
      float scale = 1.f;
      if (kBf16) {
#pragma unroll
        for (int e = 0; e < E / 2; ++e)
#pragma unroll
          for (int hw = 0; hw < 2; ++hw) {
            const float f = fabsf(raw_to_f<true>(static_cast<uint16_t>(x[e] >> (16 * hw))));
            if (f < CUDART_INF_F) most = fmaxf(most, f);
          }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        // the largest becomes 2^13 ... 2^14
        const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100), 127) - 13;
        scale = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        if (part == 0) s_row_scale[rr] = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      } else if (part == 0) {
        s_row_scale[rr] = a.scale_log2;
      }
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        uint32_t y = x[e];
        if (kBf16) y = pack_f16(raw_to_f<true>(static_cast<uint16_t>(y)) * scale, raw_to_f<true>(static_cast<uint16_t>(y >> 16)) * scale);
        const int dd = ((e >> 2) * 8 + part) * 8 + (e & 3) * 2;  // element of the row
        const int step = (dd >> 6) * 4 + ((dd >> 2) & 3), to_lane = (rr & 7) * 4 + ((dd >> 4) & 3);
        reinterpret_cast<uint32_t*>(smem + L::kQ)[(((rr >> 3) * L::kSteps + step) * 32 + to_lane) * 2 + ((dd >> 1) & 1)] = y;
      }
    }
    consumers_sync();
    constexpr int kHeldSteps = kQHeld ? kTiles * L::kSteps : 1;
    uint2 q_held[kHeldSteps];
    if (kQHeld) {
#pragma unroll
      for (int x = 0; x < kHeldSteps; ++x) q_held[x] = lds64(q_at + x * 256);
    }

    // of queries 8 tile + 2 t, + 1: sums over the values (elements 32 j + 4 g + 2 half + {0: [0, 1], 1: [2, 3]}), maximum, this lane's
    // share of the softmax's sum, factor of the scores, newest position seen
    float o[kTiles][D / 32][2][4], l[kTiles][2], row_scale[kTiles][2];
    Peak top[kTiles][2];
    int newest[kTiles][2];
    const uint16_t* bias_row[kTiles][2];
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[nt][e] = Peak{kNone, 0.f};
        l[nt][e] = 0.f;
        const int rr = min(8 * nt + 2 * t + e, nrows - 1), row = row0 + rr;
        row_scale[nt][e] = s_row_scale[rr];
        const uint2 th = token_head(a, row);
        newest[nt][e] = p.is_causal ? min(length - 1, q.length - q.n + static_cast<int>(th.x)) : length - 1;
        const int head = u.hk * a.group + th.y;
        bias_row[nt][e] = biased ? static_cast<const uint16_t*>(p.bias) + u.r * p.bias_batch_stride +
                                       (p.h_bias == p.h ? head : p.h_bias == c.h_k ? u.hk : 0) * p.bias_head_stride
                                 : nullptr;
      }
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[nt][j][i >> 2][i & 3] = 0.f;
    }

    // Kept keys: at chunk i the rows of chunk i + kAhead are asked for, the block numbers of the one behind it and the positions
    // of the next, so that nothing here waits for a load of its own. Lanes 0 - 15 stand for the slice's keys.
    constexpr int kAhead = L::kStages - 1;
    const int32_t* list = nullptr;
    int slots = 0, pos2 = -1, pos3 = -1, block2 = -1;
    float g_scale_k = 0.f, g_scale_v = 1.f;  // as loaded: a conversion beside a load would wait for it
    uint16_t g_bias = 0;
    int g_pos = -1;
    const bool head_bias = biased && p.h_bias == p.h && a.group > 1;
    auto load_pos = [&](int chunk) {
      const int slot = chunk * kChunk + warp * kSlice + (lane & 15);
      return chunk < last && slot < slots ? __ldg(list + slot) : -1;
    };
    auto load_block = [&](int& pos) {
      if (pos < 0 || pos >= length || (pos >> a.shift) >= c.width) pos = -1;
      return pos < 0 ? -1 : __ldg(c.table + static_cast<int64_t>(u.r) * c.width + (pos >> a.shift));
    };
    if (kGather) {
      list = p.kept_pos + u.r * p.kept_batch_stride + u.hk * p.kept_head_stride;
      slots = p.kept_count ? min(p.kept_count[u.r * p.count_batch_stride + u.hk * p.count_head_stride], p.kept_capacity) : p.kept_capacity;
      pos2 = load_pos(first);
      pos3 = load_pos(first + 1);
      block2 = load_block(pos2);
    }
    auto gather = [&](int i) {       // st: the stage of chunk i
      if (i + kAhead - 1 >= first) {  // what the iteration before has loaded about chunk i + kAhead - 1
        const int at = (st + kAhead - 1) % L::kStages;
        if (lane < kSlice)
          s_meta[at][warp * kSlice + lane] = make_float4(g_pos < 0 ? -CUDART_INF_F : bias_log2(raw_to_f<kBf16>(g_bias)), g_scale_k,
                                                         exponent_of(value_scale(g_scale_v)), __int_as_float(g_pos));
      }
      if (block2 < 0 || block2 >= c.num_blocks) pos2 = block2 = -1;
      g_pos = pos2;
      if (pos2 >= 0) {
        const int64_t at = static_cast<int64_t>(block2) * c.h_k + u.hk;
        g_scale_k = __ldg(c.k_scale + at);
        g_scale_v = __ldg(c.v_scale + at);
        g_bias = biased && !head_bias && pos2 < p.bias_keys ? __ldg(bias_row[0][0] + pos2) : static_cast<uint16_t>(0);
      }
      if (i + kAhead < last) {
        constexpr int kLanes = D / 16;  // 16-byte pieces of a row
        const int piece = lane % kLanes;
        const uint32_t dst = ring + (st == 0 ? L::kStages - 1 : st - 1) * L::kStageBytes + (piece >> 3) * kChunk * 128;
#pragma unroll
        for (int r = lane / kLanes; r < kSlice; r += 32 / kLanes) {
          const int pos = __shfl_sync(0xffffffffu, pos2, r), block = __shfl_sync(0xffffffffu, block2, r);
          const uint32_t to = dst + r * 128 + (((piece & 7) ^ (r & 7)) << 4);
          if (piece * 16 < c.d) {
            if (pos >= 0) {
              const int64_t row = ((static_cast<int64_t>(block) * c.h_k + u.hk) << a.shift) + (pos & ((1 << a.shift) - 1));
              cp_async16(to, static_cast<const uint8_t*>(c.k) + row * c.d + piece * 16);
              cp_async16(to + L::kTileBytes, static_cast<const uint8_t*>(c.v) + row * c.d + piece * 16);
            } else {
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(to), "r"(0) : "memory");
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(to + L::kTileBytes), "r"(0) : "memory");
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      pos2 = pos3;
      block2 = load_block(pos2);
      pos3 = load_pos(i + kAhead + 2);
    };
    if (kGather) {
      st = L::kStages - kAhead;
      for (int i = first - kAhead; i < first; ++i) {
        gather(i);
        if (++st == L::kStages) st = 0;
      }
    }

    for (int chunk = first; chunk < last; ++chunk) {
      const int pos0 = chunk * kChunk + warp * kSlice;
      if (kGather) gather(chunk);
      const int key = key_row(g);  // this lane's scores: keys pos0 + key, + 8
      uint16_t raw_bias[kTiles][2][2];
      constexpr bool with_bias = kBias;
      const bool head_bias_dense = with_bias && head_bias;
      if (with_bias) {
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int pos = pos0 + (k >> 1) * 8 + key;
            if ((k & 1) == 0 || head_bias_dense) raw_bias[nt][k >> 1][k & 1] = pos < min(length, p.bias_keys) ? __ldg(bias_row[nt][k & 1] + pos) : static_cast<uint16_t>(0);
            else raw_bias[nt][k >> 1][1] = raw_bias[nt][k >> 1][0];
          }
      }
      float4 meta;
      float4 key_meta[2];
      if (kGather) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 2; ++k) key_meta[k] = s_meta[st][warp * kSlice + k * 8 + key];
      } else {
        mbar_wait(&s_full[st], phase, ctl, 702);
        meta = s_meta[st][warp];
      }
      const uint32_t tile = ring + st * L::kStageBytes;
      // scores: s[tile][2 * (second eight keys) + (second query)]
      float s[kTiles][4];
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int jj = 0; jj < D / 64; ++jj) {
        const uint32_t at = tile + (jj >> 1) * kChunk * 128 + (k_at ^ ((jj & 1) << 6));
        const uint4 ka = lds128(at), kb = lds128(at + 1024);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t a0 = e4m3x2_to_f16x2(wa[x]), a1 = e4m3x2_to_f16x2(wb[x]), a2 = e4m3x2_hi_to_f16x2(wa[x]), a3 = e4m3x2_hi_to_f16x2(wb[x]);
#pragma unroll
          for (int nt = 0; nt < kTiles; ++nt) {
            const int step = nt * L::kSteps + jj * 4 + x;
            const uint2 f = kQHeld ? q_held[kQHeld ? step : 0] : lds64(q_at + step * 256);
            mma_f16(s[nt], a0, a1, a2, a3, f.x, f.y);
          }
        }
      }
      // all 16 keys are there and seen by every row
      const bool clean = !kGather && pos0 + kSlice <= sure && meta.x != 0.f;
      float x[kTiles][4];
      auto z_of = [&](int k) { return kGather ? key_meta[k >> 1].z : meta.z; };  // exponent of the V scale of score k
      // log2 of its ratio to the maximum
      auto ratio = [&](int nt, int k) {
        const float diff = x[nt][k] - top[nt][k & 1].m;
        return diff + (z_of(k) - top[nt][k & 1].z);
      };
      float d[kTiles][4];
      bool grows = false;
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float& v = x[nt][k];
          if (kGather) {
            const float4& km = key_meta[k >> 1];
            const int pos = __float_as_int(km.w);
            float add = km.x;
            if (head_bias && pos >= 0 && pos < p.bias_keys) add = bias_log2(raw_to_f<kBf16>(__ldg(bias_row[nt][k & 1] + pos)));
            v = fmaf(s[nt][k], row_scale[nt][k & 1] * km.y, add);
            if (add == -CUDART_INF_F || pos > newest[nt][k & 1]) v = -CUDART_INF_F;  // even where the key is NaN
          } else {
            v = s[nt][k] * (row_scale[nt][k & 1] * meta.y);
            if (with_bias) {
              const float add = bias_log2(raw_to_f<kBf16>(raw_bias[nt][k >> 1][k & 1]));
              v = add == -CUDART_INF_F ? add : v + add;
            }
            if (!clean && (pos0 + (k >> 1) * 8 + key > newest[nt][k & 1] || meta.x == 0.f)) v = -CUDART_INF_F;
          }
          d[nt][k] = ratio(nt, k);
          grows |= d[nt][k] > 0.f;
        }
      }
      uint32_t poisoned = 0;  // scores, a bit each, whose value is NaN
      if (!clean || with_bias) {
        float least = x[0][0];
#pragma unroll
        for (int i = 1; i < 4 * kTiles; ++i) least = fminf(least, x[i >> 2][i & 3]);
        // Values that some query does not see must not reach it, which 0 times NaN would: NaN become 0 where they are, and who sees
        // them gets NaN otherwise. What lies behind the last key may be anything.
        if (__any_sync(0xffffffffu, least == -CUDART_INF_F)) {
          uint32_t found = 0;  // a bit for each of this lane's 16-byte pieces
#pragma unroll
          for (int i = 0; i < 4 * L::kHalves; ++i) {
            const int r = (i & 3) * 4 + (lane >> 3);
            const uint32_t at = tile + L::kTileBytes + (i >> 2) * kChunk * 128 + r * 128 + (lane & 7) * 16;
            uint4 v = lds128(at);
            if (drop_nan(v.x) | drop_nan(v.y) | drop_nan(v.z) | drop_nan(v.w)) {
              asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
              found |= 1u << i;
            }
          }
          __syncwarp();
          if (__any_sync(0xffffffffu, found)) {
            fence_proxy_async_smem();  // before the next copy into this stage
            const int there = kGather ? kSlice : meta.x != 0.f ? min(max(length - pos0, 0), kSlice) : 0;
            uint32_t nan_rows = 0;
            for (int i = 0; i < 4 * L::kHalves; ++i) {
              const bool used = D >= 128 || ((lane & 7) ^ (((i & 3) * 4 + (lane >> 3)) & 7)) < D / 16;  // a row of 128 bytes may be half empty
              const uint32_t lanes = __ballot_sync(0xffffffffu, used && found >> i & 1);
#pragma unroll
              for (int k = 0; k < 4; ++k) nan_rows |= static_cast<uint32_t>((lanes >> (8 * k) & 0xFF) != 0) << ((i & 3) * 4 + k);
            }
            nan_rows &= (1u << there) - 1;
#pragma unroll
            for (int i = 0; i < 4 * kTiles; ++i)
              if (x[i >> 2][i & 3] != -CUDART_INF_F && nan_rows >> ((i >> 1 & 1) * 8 + key) & 1) poisoned |= 1u << i;
          }
        }
      }
      if (__any_sync(0xffffffffu, grows)) {  // a query's maxima are compared over its keys only when one of them grows
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt) {
          float corr[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            Peak now;
            if (kGather) {
              now = higher(Peak{x[nt][e], z_of(e)}, Peak{x[nt][2 + e], z_of(2 + e)});
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) now = higher(now, shuffled(now, off));
              now = of_lane(now, t);
            } else {  // of one block: the scores alone
              now = Peak{fmaxf(x[nt][e], x[nt][2 + e]), z_of(e)};
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) now.m = fmaxf(now.m, __shfl_xor_sync(0xffffffffu, now.m, off));
            }
            now = higher(top[nt][e], now);
            corr[e] = rescale(top[nt][e], now);
            top[nt][e] = now;
            l[nt][e] *= corr[e];
          }
#pragma unroll
          for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[nt][j][i >> 2][i & 3] *= corr[i & 1];
#pragma unroll
          for (int k = 0; k < 4; ++k) d[nt][k] = ratio(nt, k);
        }
      }
      uint32_t pb[kTiles][2];  // P^T: queries' probabilities, keys 0-7 | 8-15
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) {
        float e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = exp2f(d[nt][k]);
        if (kGather) {
#pragma unroll
          for (int k = 0; k < 4; ++k) l[nt][k & 1] = fmaf(e[k], exp2f(-key_meta[k >> 1].z), l[nt][k & 1]);
        } else {
          l[nt][0] = fmaf(e[0] + e[2], meta.w, l[nt][0]);
          l[nt][1] = fmaf(e[1] + e[3], meta.w, l[nt][1]);
        }
        if (poisoned) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (poisoned >> (nt * 4 + k) & 1) l[nt][k & 1] = CUDART_NAN_F;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float f = p_scale(kGather ? key_meta[k].z : meta.z);
          pb[nt][k] = transpose8(pack_f16(e[2 * k] * f, e[2 * k + 1] * f));
        }
      }
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint32_t half = tile + (j >> 2) * kChunk * 128;
        const uint32_t at0 = half + (v_at0 ^ ((j & 3) << 5)), at1 = half + (v_at1 ^ ((j & 3) << 5));
        const uint32_t y0 = lds32<0>(at0), y1 = lds32<0>(at1), y2 = lds32<1024>(at0), y3 = lds32<1024>(at1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // bytes 0, 1 | 2, 3 of the words: rows g | g + 8 of the product
          const uint32_t first = __byte_perm(y0, y1, h ? 0x7362 : 0x5140), second = __byte_perm(y2, y3, h ? 0x7362 : 0x5140);
          const uint32_t a0 = e4m3x2_to_f16x2(first), a1 = e4m3x2_hi_to_f16x2(first), a2 = e4m3x2_to_f16x2(second), a3 = e4m3x2_hi_to_f16x2(second);
#pragma unroll
          for (int nt = 0; nt < kTiles; ++nt) mma_f16(o[nt][j][h], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
        }
      }
      __syncwarp();  // every lane has read the stage before it is overwritten
      if (!kGather && lane == 0) mbar_arrive(&s_empty[st]);
      if (++st == L::kStages) {
        st = 0;
        phase ^= 1;
      }
    }

    // ---- the four warps' sums: to a common maximum, then added up through shared memory ----
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
        if (g == 0) {
          s_m[warp][8 * nt + 2 * t + e] = top[nt][e];
          s_l[warp][8 * nt + 2 * t + e] = l[nt][e];
        }
      }
    consumers_sync();
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = 8 * nt + 2 * t + e;
        Peak all = s_m[0][rr];
        float cl = 0.f;
#pragma unroll
        for (int x = 1; x < kWarps; ++x) all = higher(all, s_m[x][rr]);
#pragma unroll
        for (int x = 0; x < kWarps; ++x) cl = fmaf(s_l[x][rr], rescale(s_m[x][rr], all), cl);
        f[e] = rescale(top[nt][e], all) * (1.f / kPScale);
        top[nt][e] = all;
        l[nt][e] = cl;
      }
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[nt][j][i >> 2][i & 3] *= f[i & 1];
    }
    auto put = [&](float* buf) {
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const float(&y)[4] = o[nt][i >> 1][i & 1];
          *reinterpret_cast<float4*>(buf + (nt * (D / 16) + i) * 128 + lane * 4) = make_float4(y[0], y[1], y[2], y[3]);
        }
    };
    auto add = [&](const float* buf) {
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          float(&y)[4] = o[nt][i >> 1][i & 1];
          const float4 x = *reinterpret_cast<const float4*>(buf + (nt * (D / 16) + i) * 128 + lane * 4);
          y[0] += x.x; y[1] += x.y; y[2] += x.z; y[3] += x.w;
        }
    };
    if constexpr (L::kBufs == 2) {
      if (warp >= 2) put(s_buf + (warp - 2) * L::kBufFloats);
      consumers_sync();
      if (warp < 2) add(s_buf + warp * L::kBufFloats);
      consumers_sync();
      if (warp == 1) put(s_buf);
      consumers_sync();
      if (warp == 0) add(s_buf);
    } else {
      for (int x = kWarps - 1; x > 0; --x) {
        if (warp == x) put(s_buf);
        consumers_sync();
        if (warp == 0) add(s_buf);
        consumers_sync();
      }
    }
    if (warp != 0) continue;
    if (kCluster) __syncwarp();  // (the sums are read no more)
    const bool complete = !kCluster && first == 0 && last == u.n;
    float* part = kCluster ? s_buf : a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (first > 0 ? 0 : 1)) * ROWS * (D + 4);
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = 8 * nt + 2 * t + e, row = row0 + rr;
        if (rr >= nrows) continue;
        if (complete) {
          const float inv = l[nt][e] == 0.f ? 0.f : 1.f / l[nt][e];
          const uint2 th = token_head(a, row);
          uint16_t* dst = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(q.token0 + th.x) * p.out_row_stride + (u.hk * a.group + th.y) * p.out_head_stride;
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const int dd = 32 * j + 4 * g;
            const float(&y)[2][4] = o[nt][j];
            if (dd < c.d)
              *reinterpret_cast<uint2*>(dst + dd) = make_uint2(pack2<kBf16>(y[0][e] * inv, y[0][2 + e] * inv), pack2<kBf16>(y[1][e] * inv, y[1][2 + e] * inv));
          }
        } else {
          float* dst = part + rr * (kCluster ? D : D + 4);
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const float(&y)[2][4] = o[nt][j];
            *reinterpret_cast<float4*>(dst + 32 * j + 4 * g) = make_float4(y[0][e], y[0][2 + e], y[1][e], y[1][2 + e]);
          }
          if (g == 0) *(kCluster ? s_part + rr : reinterpret_cast<float4*>(dst + D)) = make_float4(top[nt][e].m, l[nt][e], top[nt][e].z, 0.f);
        }
      }
  }

  if constexpr (kCluster) {
    // ---- the CTAs' sums: each joins its share of the numbers, eight threads for four of them ----
    cluster_sync();
    const Request& q = units.q;
    const int rank = static_cast<int>(cluster_rank()), row0 = units.x.tile * ROWS, nrows = min(ROWS, q.rows - row0), of = tid & 7;
    for (int base = rank * 16; base < nrows * (D / 4); base += a.cluster * 16) {
      const int v = base + (tid >> 3), rr = min(v / (D / 4), nrows - 1), col = v % (D / 4) * 4;
      float4 ml[2], y[2];
      float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        ml[k] = make_float4(kNone, 0.f, 0.f, 0.f);
        if (of + 8 * k < a.cluster) {
          ml[k] = ld_cluster(shared_of(s_part + rr, of + 8 * k));
          y[k] = ld_cluster(shared_of(s_buf + rr * D + col, of + 8 * k));
        }
      }
      // maxima relative to about the largest, and the largest of those
      const float about = largest8(fmaxf(ml[0].x + ml[0].z, ml[1].x + ml[1].z));
      const float rel[2] = {(ml[0].x - about) + ml[0].z, (ml[1].x - about) + ml[1].z}, most = largest8(fmaxf(rel[0], rel[1]));
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (ml[k].x != kNone || ml[k].y != 0.f) {  // (otherwise its sums are zeros, or were not written; NaN is not 0)
          const float f = exp2f(rel[k] - most);
          sum = fmaf(ml[k].y, f, sum);
          acc[0] = fmaf(y[k].x, f, acc[0]); acc[1] = fmaf(y[k].y, f, acc[1]);
          acc[2] = fmaf(y[k].z, f, acc[2]); acc[3] = fmaf(y[k].w, f, acc[3]);
        }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
      }
      if (of == 0 && v < nrows * (D / 4) && col < c.d) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const uint2 th = token_head(a, row0 + rr);
        uint16_t* dst = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(q.token0 + th.x) * p.out_row_stride + (units.x.hk * a.group + th.y) * p.out_head_stride;
        *reinterpret_cast<uint2*>(dst + col) = make_uint2(pack2<kBf16>(acc[0] * inv, acc[1] * inv), pack2<kBf16>(acc[2] * inv, acc[3] * inv));
      }
    }
    // rows that nobody computes: of this request, and behind the last one
    if (units.x.tile == 0) {
      auto clear = [&](int token0, int64_t from, int64_t to) {
        for (int64_t i = from * (c.d / 8) + rank * 128 + tid; i < to * (c.d / 8); i += a.cluster * 128) {
          const int row = static_cast<int>(i / (c.d / 8));
          const uint2 th = token_head(a, row);
          uint16_t* dst = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(token0 + th.x) * p.out_row_stride + (units.x.hk * a.group + th.y) * p.out_head_stride;
          *reinterpret_cast<uint4*>(dst + (i - static_cast<int64_t>(row) * (c.d / 8)) * 8) = make_uint4(0, 0, 0, 0);
        }
      };
      if (q.rows < q.n * a.group) clear(q.token0, q.rows, static_cast<int64_t>(q.n) * a.group);
      if (units.x.r == c.requests - 1) {
        const int end = max(0, min(c.cu_seqlens[c.requests], c.tokens));
        if (end < c.tokens) clear(end, 0, static_cast<int64_t>(c.tokens - end) * a.group);
      }
    }
    cluster_sync();  // nobody leaves while its shared memory may still be read
  }
}

// AttnArgs::pre for many requests, by one CTA.
__global__ void __launch_bounds__(1024) cache_sums_kernel(const __grid_constant__ AttnArgs a, int32_t* pre) {
  __shared__ int s_warp[32];
  const int R = a.p.c.requests, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int carry = 0;
  for (int base = 0; base < R; base += 1024) {
    int x = 0;
    if (base + tid < R) {
      const Request q = load_request(a, base + tid);
      x = q.chunks * tiles_of(a, q.rows);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    x += carry;
    for (int i = 0; i < 32; ++i) {
      if (i < warp) x += s_warp[i];
      carry += s_warp[i];
    }
    if (base + tid < R) pre[base + tid + 1] = x;
    __syncthreads();
  }
  if (tid == 0) pre[0] = 0;
}

// Joins the sums of units that several CTAs share, and writes the zeros of rows that nobody computes: a CTA per (token, head),
// whose warps take a quarter of the sums each.
template <int D, bool kBf16>
__global__ void __launch_bounds__(128, D > 128 ? 4 : 8) cache_merge_kernel(const __grid_constant__ AttnArgs a) {
  const fdma_cache_attention_params& p = a.p;
  const fdma_cache& c = p.c;
  __shared__ int s_request;
  __shared__ Peak s_top[4];
  __shared__ float s_sum[4], s_acc[4][D];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = static_cast<int>(blockIdx.x / p.h), head = static_cast<int>(blockIdx.x - static_cast<unsigned>(slot) * p.h);
  int r, token = slot, end = slot + 1;
  if (a.merge_requests) {  // tokens i, i + 31 ... of request r
    r = slot / (kPromptTokens - 1);
    token = max(0, c.cu_seqlens[r]) + slot - r * (kPromptTokens - 1);
    end = min(c.cu_seqlens[r + 1], c.tokens);
  } else if (token < c.requests && c.cu_seqlens[token] == token && c.cu_seqlens[token + 1] == token + 1) {
    r = token;  // one token each
  } else {
    if (tid == 0) s_request = -1;
    __syncthreads();
    for (int x = tid; x < c.requests; x += 128)
      if (c.cu_seqlens[x] <= token && token < c.cu_seqlens[x + 1]) s_request = x;
    __syncthreads();
    r = s_request;
  }
  const Units units{a, nullptr};
  const int64_t step = (static_cast<int64_t>(D) + 4) << a.row_shift;
  Request q{};
  if (r >= 0) q = units.request(r);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (q.rows < 0) return;  // done already
  const int64_t share = share_of(units.total(), a.ctas);
  for (; token < end; token += kPromptTokens - 1) {
    int c0 = 0, c1 = -1;
    const float* base = nullptr;
    const uint2 kv = token_head(a, head);  // kv head, and the head among those that share it
    const int row = (token - q.token0) * a.group + kv.y, tile = row >> a.row_shift;
    if (r >= 0 && row >= 0 && row < q.rows) {
      const Unit u = units.of(Cursor{r, static_cast<int>(kv.x), tile}, q);
      c0 = static_cast<int>(quotient(u.start, share));
      c1 = static_cast<int>(quotient(u.start + u.n - 1, share));
      base = a.partial + static_cast<int64_t>(row - (tile << a.row_shift)) * (D + 4);
      if (c0 == c1) continue;  // written by that CTA
    }
    // each warp takes every fourth sum, four at a time, and scales to its own maximum
    constexpr int E = D / 32, kAhead = 4;  // elements per lane
    float acc[E], sum = 0.f;
    Peak top{kNone, 0.f};
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
    for (int x0 = c0 + warp; x0 <= c1; x0 += 4 * kAhead) {
      float4 ml[kAhead];
      float2 y[kAhead][E / 2];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int x = x0 + 4 * k;
        ml[k] = make_float4(kNone, 0.f, 0.f, 0.f);
        if (x <= c1) {
          const float* src = base + (2 * static_cast<int64_t>(x) + (x == c0)) * step;
          ml[k] = *reinterpret_cast<const float4*>(src + D);
#pragma unroll
          for (int i = 0; i < E / 2; ++i) y[k][i] = *reinterpret_cast<const float2*>(src + lane * E + 2 * i);
        }
      }
      Peak now = top;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) now = higher(now, Peak{ml[k].x, ml[k].z});
      const float f0 = rescale(top, now);
      top = now;
      sum *= f0;
#pragma unroll
      for (int i = 0; i < E; ++i) acc[i] *= f0;
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (x0 + 4 * k <= c1) {
          const float f = rescale(Peak{ml[k].x, ml[k].z}, now);
          sum = fmaf(ml[k].y, f, sum);
#pragma unroll
          for (int i = 0; i < E / 2; ++i) {
            acc[2 * i] = fmaf(y[k][i].x, f, acc[2 * i]);
            acc[2 * i + 1] = fmaf(y[k][i].y, f, acc[2 * i + 1]);
          }
        }
    }
    if (lane == 0) {
      s_top[warp] = top;
      s_sum[warp] = sum;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) s_acc[warp][lane * E + i] = acc[i];
    __syncthreads();
    top = higher(higher(s_top[0], s_top[1]), higher(s_top[2], s_top[3]));
    float f[4];
    sum = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      f[x] = rescale(s_top[x], top);
      sum = fmaf(s_sum[x], f[x], sum);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* dst = static_cast<uint16_t*>(p.out) + token * p.out_row_stride + head * p.out_head_stride;
    for (int i = 2 * tid; i < c.d; i += 256) {
      float y[2] = {0.f, 0.f};
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int k = 0; k < 2; ++k) y[k] = fmaf(s_acc[x][i + k], f[x], y[k]);
      *reinterpret_cast<uint32_t*>(dst + i) = pack2<kBf16>(y[0] * inv, y[1] * inv);
    }
    __syncthreads();  // (the next token uses the same shared memory)
  }
}

int tile_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

struct Plan {
  int D, rows, ctas, list_chunks;
  bool sums;  // by a kernel of their own: many requests, and not one tile of cu_chunks' chunks for each
  int64_t most_chunks;
  bool prompts;
  int cluster, tiles, units;
  size_t sums_off, prompt_off, bytes;
};
Plan plan_of(const fdma_cache_attention_params& p) {
  Plan pl;
  pl.prompts = cache_prompt_taken(p);
  const int64_t most = static_cast<int64_t>(std::max(std::min(p.max_seqlen_q, p.c.tokens), 1)) * (p.h / p.c.h_k);
  pl.D = tile_dim(p.c.d);
  // (at head dim 256, two tiles of 8 rows that read the same keys one after the other are faster than one of 16, whose accumulators
  // do not fit: 8 requests of 16384 tokens, 4 new ones each, 32 heads over 8: 59 us against 70)
  pl.rows = most <= 8 || pl.D == 256 ? 8 : 16;
  pl.ctas = (pl.D == 256 || pl.rows > 8 ? 2 : 3) * sm_count();
  pl.list_chunks = p.kept_pos ? (p.kept_capacity + kChunk - 1) / kChunk : 0;
  pl.sums = p.c.requests > kHeld && (pl.list_chunks || most > pl.rows);
  const int64_t tiles = static_cast<int64_t>(p.c.tokens) * (p.h / p.c.h_k) / pl.rows + p.c.requests;
  pl.most_chunks = tiles * (pl.list_chunks ? pl.list_chunks : (static_cast<int64_t>(p.c.width) * p.c.block_size + kChunk - 1) / kChunk);
  pl.tiles = static_cast<int>((most + pl.rows - 1) / pl.rows);
  const int64_t units = static_cast<int64_t>(p.c.requests) * p.c.h_k * pl.tiles;
  const int64_t chunks = pl.list_chunks ? pl.list_chunks : (std::min<int64_t>(p.max_seqlen_k, static_cast<int64_t>(p.c.width) * p.c.block_size) + kChunk - 1) / kChunk;
  pl.units = static_cast<int>(std::min<int64_t>(units, 1 << 20));
  pl.cluster = 0;
  // Few and short enough units get a cluster each: as many CTAs as run at once (clusters leave places of a GPU's parts empty, 16 a
  // quarter of them and 8 an eighth), but fewer than two for a chunk. From 24 chunks a CTA on equal shares are as fast (1 request of
  // 24000 tokens, 32 heads over 8, d = 128: 20.5 us, 20.3); up to 16 they take longer (4096 tokens: 7.7, 12.2; 16384: 15.5, 16.9).
  if (!pl.prompts && units > 0)
    for (int n = kMostCluster; n > 1 && !pl.cluster; n /= 2)
      if (units * n <= pl.ctas - pl.ctas * n / 64 && (n < 2 * chunks || n == 2) && chunks <= static_cast<int64_t>(kMostClusterChunks) * n) pl.cluster = n;
  pl.sums_off = align256(static_cast<size_t>(pl.ctas) * 2 * pl.rows * (pl.D + 4) * sizeof(float));
  pl.prompt_off = pl.sums_off + align256((static_cast<size_t>(p.c.requests) + 1) * sizeof(int32_t));
  pl.bytes = pl.cluster ? 0 : pl.prompt_off + (pl.prompts ? cache_prompt_workspace_bytes(p) : 0);
  return pl;
}

int allow_wide_clusters_once(const void* kernel, std::atomic<uint64_t>& prepared) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (prepared.load(std::memory_order_acquire) & bit)) return 0;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 64) prepared.fetch_or(bit, std::memory_order_release);
  return 0;
}

template <int D, int ROWS, bool kGather, bool kBf16, bool kCluster, bool kBias>
int launch(AttnArgs a, const Plan& pl, cudaStream_t stream) {
  using L = Layout<D, ROWS, kGather>;
  const fdma_cache& c = a.p.c;
  CUtensorMap map_k{}, map_v{};
  if (!kGather) {
    const uint64_t d = c.d, bs = c.block_size, heads = static_cast<uint64_t>(c.num_blocks) * c.h_k;
    const uint64_t dims[4] = {d, bs, heads, 1}, strides[3] = {d, bs * d, heads * bs * d};
    const uint32_t box[4] = {128, std::min<uint32_t>(bs, kChunk), 1, 1};
    int st = encode_tmap_4d(&map_k, c.k, 1, dims, strides, box);
    if (!st) st = encode_tmap_4d(&map_v, c.v, 1, dims, strides, box);
    if (st) return st;
  }
  auto kern = cache_attend_kernel<D, ROWS, kGather, kBf16, kCluster, kBias>;
  static std::atomic<uint64_t> prepared{0}, wide{0};
  const int st_smem = allow_smem_once(reinterpret_cast<const void*>(kern), L::kTotal, prepared);
  if (st_smem) return st_smem;
  if constexpr (kCluster) {
    a.cluster = pl.cluster;
    a.tiles = pl.tiles;
    const int st = pl.cluster > 8 ? allow_wide_clusters_once(reinterpret_cast<const void*>(kern), wide) : 0;
    if (st) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(pl.units) * pl.cluster);
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kTotal;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = pl.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, a, map_k, map_v));
  }
  kern<<<pl.ctas, L::kThreads, L::kTotal, stream>>>(a, map_k, map_v);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  // the second kernel's CTAs start while the first one's finish, and wait for them only where they need their sums
  cudaLaunchConfig_t cfg = {};
  const int64_t few = static_cast<int64_t>(c.requests) * (kPromptTokens - 1);
  a.merge_requests = a.prompts && few < c.tokens;
  cfg.gridDim = dim3(static_cast<unsigned>(a.merge_requests ? few : c.tokens) * a.p.h);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, cache_merge_kernel<D, kBf16>, a));
}
template <int D, int ROWS, bool kCluster, bool kBf16>
int launch_c(const AttnArgs& a, const Plan& pl, cudaStream_t stream) {
  if (a.list_chunks) return launch<D, ROWS, true, kBf16, kCluster, false>(a, pl, stream);
  return a.p.bias ? launch<D, ROWS, false, kBf16, kCluster, true>(a, pl, stream) : launch<D, ROWS, false, kBf16, kCluster, false>(a, pl, stream);
}
template <int D, int ROWS>
int launch_t(const AttnArgs& a, const Plan& pl, cudaStream_t stream) {
  if (a.p.dtype == FDMA_BF16) return pl.cluster ? launch_c<D, ROWS, true, true>(a, pl, stream) : launch_c<D, ROWS, false, true>(a, pl, stream);
  return pl.cluster ? launch_c<D, ROWS, true, false>(a, pl, stream) : launch_c<D, ROWS, false, false>(a, pl, stream);
}

int check_attention(const fdma_cache_attention_params* pp) {
  if (!pp) return FDMA_ERR_BAD_ARG;
  const fdma_cache_attention_params& p = *pp;
  const int st = check_cache(p.c);
  if (st) return st;
  if (p.h <= 0 || p.h % p.c.h_k || p.max_seqlen_q < 0 || p.max_seqlen_k < 0) return FDMA_ERR_BAD_ARG;
  if (p.bias && ((p.h_bias != 1 && p.h_bias != p.c.h_k && p.h_bias != p.h) || p.bias_keys <= 0)) return FDMA_ERR_BAD_ARG;
  if (p.kept_pos && p.kept_capacity <= 0) return FDMA_ERR_BAD_ARG;
  if (p.dtype != FDMA_BF16 && p.dtype != FDMA_FP16) return FDMA_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(p.c.num_blocks) * p.c.h_k > 0x7FFFFFFF || static_cast<int64_t>(p.c.tokens) * p.h > 0x7FFFFFFF) return FDMA_ERR_UNSUPPORTED;
  return 0;
}

}  // namespace
}  // namespace fdma

using namespace fdma;

extern "C" size_t fdma_cache_attention_workspace_bytes(const fdma_cache_attention_params* p) {
  if (check_attention(p) || p->c.tokens == 0) return 0;
  return plan_of(*p).bytes;
}

extern "C" int fdma_cache_attention(const fdma_cache_attention_params* pp, void* stream_) {
  const int st = check_attention(pp);
  if (st) return st;
  const fdma_cache_attention_params& p = *pp;
  if (p.c.tokens == 0) return FDMA_OK;
  if (!p.query || !p.out) return FDMA_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(p.out) | static_cast<uint64_t>(p.out_row_stride | p.out_head_stride) * 2) % 16) return FDMA_ERR_UNSUPPORTED;
  const Plan pl = plan_of(p);
  if (pl.most_chunks > 0x7FFFFFFF) return FDMA_ERR_TOO_LARGE;
  if (pl.bytes && (!p.workspace || p.workspace_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(p.workspace) & 255))) return FDMA_ERR_WORKSPACE;
  AttnArgs a = {};
  a.p = p;
  a.shift = p.c.block_size == 16 ? 4 : p.c.block_size == 32 ? 5 : p.c.block_size == 64 ? 6 : 7;
  a.group = p.h / p.c.h_k;
  a.row_shift = pl.rows == 8 ? 3 : 4;
  auto inverse = [](int x) { return static_cast<uint32_t>(std::min<uint64_t>((uint64_t{1} << 32) / x, 0xFFFFFFFFu)); };
  a.group_inverse = inverse(a.group);
  a.h_k_inverse = inverse(p.c.h_k);
  a.p.max_seqlen_q = std::max(a.p.max_seqlen_q, 1);
  a.list_chunks = pl.list_chunks;
  a.ctas = pl.ctas;
  a.scale_log2 = p.softmax_scale * kLog2e;
  a.q_vec = (reinterpret_cast<uintptr_t>(p.query) | static_cast<uint64_t>(p.query_row_stride | p.query_head_stride) * 2) % 16 == 0;
  a.status = kernel_status_ptr();
  if (!a.status) return FDMA_ERR_DRIVER;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!pl.cluster) {
    char* const ws = static_cast<char*>(p.workspace);
    a.partial = static_cast<float*>(p.workspace);
    if (pl.prompts) {
      const int status = cache_prompt(p, a.shift, ws + pl.prompt_off, stream);
      if (status) return status;
      a.prompts = reinterpret_cast<const int32_t*>(ws + pl.prompt_off + cache_prompt_again(p));
    }
    a.pre = reinterpret_cast<int32_t*>(ws + pl.sums_off);
    if (pl.sums) {
      cache_sums_kernel<<<1, 1024, 0, stream>>>(a, a.pre);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return static_cast<int>(e);
    } else if (p.c.requests > kHeld) {  // a tile for each request: their chunks
      a.pre = const_cast<int32_t*>(p.c.cu_chunks);
    }
  }
  if (pl.D == 256) return launch_t<256, 8>(a, pl, stream);
  if (pl.D == 128) return pl.rows == 8 ? launch_t<128, 8>(a, pl, stream) : launch_t<128, 16>(a, pl, stream);
  return pl.rows == 8 ? launch_t<64, 8>(a, pl, stream) : launch_t<64, 16>(a, pl, stream);
}
