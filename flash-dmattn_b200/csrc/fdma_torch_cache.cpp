// Native host path of the rotary positions, the block tables and the 8-bit cache: argument checks, allocations, the autograd
// node and the launches of flash_sparse_attn/rotary.py and cache.py, on top of the C ABI (include/fdma.h). Wrong arguments raise
// RuntimeError here. Tensors that stand for something else (tracing, subclasses, functorch) get None: the Python layer then goes
// through its custom operators, which come back here with plain tensors.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/fdma.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::variable_list;

namespace {

struct Api {
  decltype(&fdma_rotary) rotary;
  decltype(&fdma_tables_extend) tables_extend;
  decltype(&fdma_tables_truncate) tables_truncate;
  decltype(&fdma_cache_append) cache_append;
  decltype(&fdma_cache_attention) cache_attention;
  decltype(&fdma_cache_attention_workspace_bytes) cache_attention_workspace_bytes;
  decltype(&fdma_strerror) strerror;
  decltype(&fdma_poll_kernel_status) poll_kernel_status;
  decltype(&fdma_last_kernel_status) last_kernel_status;
} api;

void need(bool ok, const char* what) {
  if (!ok) throw std::runtime_error(what);
}
void check(int status, const char* what) {
  if (status != 0)
    throw std::runtime_error(std::string(what) + " failed: " + api.strerror(status) + " (status " + std::to_string(status) + ")");
}
cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
// A kernel whose bounded wait gave up surfaces at the next operator call (one host load, no GPU work).
void raise_if_timed_out(cudaStream_t stream) {
  if (api.poll_kernel_status(nullptr) == 0) return;
  int32_t detail = 0;
  api.last_kernel_status(stream, &detail);
  throw std::runtime_error("an earlier attention kernel on this device gave up a bounded wait (code " + std::to_string(detail) +
                           "): " + api.strerror(FDMA_ERR_TIMEOUT) + "; results of calls since then are not valid");
}
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
Tensor inner_contiguous(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return FDMA_BF16;
    case at::kHalf: return FDMA_FP16;
    case at::kFloat: return FDMA_FP32;
    default: return -1;
  }
}
// 0 along dimensions of one element, whose stride says nothing
int64_t stride_of(const Tensor& t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

Tensor given(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// ---- rotary positions -----------------------------------------------------------------------------------------------
struct Rotation {
  Tensor turns;
  bool interleaved = false, inverse = false;
  double amplitude = 1.0;
};

void check_rotation(const Tensor& turns, const Tensor& x, int64_t d) {
  need(turns.scalar_type() == at::kLong && turns.dim() == 1 && turns.is_contiguous(), "the frequencies must be a contiguous int64 tensor (see rotary_frequencies)");
  need(turns.device() == x.device(), "the frequencies must be on the same device as the tensors they turn");
  need(turns.size(0) > 0 && 2 * turns.size(0) <= d, "the frequencies turn more than the head dimension");
}

// q (B, S, H, d) or (T, H, d), k the same with heads of its own or undefined; positions ({B|1}, S), (S,) or undefined.
variable_list rotate(const Tensor& q0, const Tensor& k0, const Tensor& positions, const Rotation& r) {
  at::AutoDispatchBelowADInplaceOrView guard;
  const c10::cuda::CUDAGuard device(q0.device());
  const cudaStream_t stream = stream_of(q0);
  fdma_rotary_params p = {};
  const bool batched = q0.dim() == 4;
  const int64_t row = batched ? 1 : 0, head = row + 1;
  p.b = static_cast<int32_t>(batched ? q0.size(0) : 1);
  p.seqlen = static_cast<int32_t>(q0.size(row));
  p.d = static_cast<int32_t>(q0.size(-1));
  p.dtype = dtype_code(q0);
  p.turns = r.turns.data_ptr<int64_t>();
  p.rotary_dim = static_cast<int32_t>(2 * r.turns.size(0));
  p.interleaved = r.interleaved;
  p.inverse = r.inverse;
  p.amplitude = static_cast<float>(r.amplitude);
  if (positions.defined()) {
    p.positions = positions.data_ptr();
    p.position_bits = positions.scalar_type() == at::kLong ? 64 : 32;
    p.pos_row_stride = stride_of(positions, positions.dim() - 1);
    p.pos_batch_stride = positions.dim() == 2 ? stride_of(positions, 0) : 0;
  }
  const Tensor q = inner_contiguous(q0), k = k0.defined() ? inner_contiguous(k0) : k0;
  variable_list out;
  auto fill = [&](const Tensor& x, const void*& src, void*& dst, int32_t& heads, int64_t& sb, int64_t& sr, int64_t& sh, int64_t& ob, int64_t& orow,
                  int64_t& oh) {
    Tensor y = empty(x.sizes(), x.scalar_type(), x);
    src = x.data_ptr();
    dst = y.data_ptr();
    heads = static_cast<int32_t>(x.size(head));
    sb = batched ? stride_of(x, 0) : 0; sr = stride_of(x, row); sh = stride_of(x, head);
    ob = batched ? stride_of(y, 0) : 0; orow = stride_of(y, row); oh = stride_of(y, head);
    out.push_back(std::move(y));
  };
  fill(q, p.q, p.q_out, p.h, p.q_batch_stride, p.q_row_stride, p.q_head_stride, p.qo_batch_stride, p.qo_row_stride, p.qo_head_stride);
  if (k.defined())
    fill(k, p.k, p.k_out, p.h_k, p.k_batch_stride, p.k_row_stride, p.k_head_stride, p.ko_batch_stride, p.ko_row_stride, p.ko_head_stride);
  if (q.numel() || (k.defined() && k.numel())) check(api.rotary(&p, stream), "fdma_rotary");
  return out;
}

variable_list rotate_differentiable(const Tensor& q, const Tensor& k, const Tensor& positions, const Rotation& r);

// The gradient of a rotation is the rotation by the negative angle, itself differentiable.
struct RotaryFunction : public torch::autograd::Function<RotaryFunction> {
  static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k, const OptTensor& positions,
                               const Tensor& turns, bool interleaved, bool inverse, double amplitude) {
    ctx->save_for_backward({given(positions), turns});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["amplitude"] = amplitude;
    return rotate(q, given(k), given(positions), Rotation{turns, interleaved, inverse, amplitude});
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Rotation r{saved[1], ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool(),
                     ctx->saved_data["amplitude"].toDouble()};
    variable_list res(7);
    const bool both = grads.size() == 2 && grads[0].defined() && grads[1].defined();
    if (both) {
      variable_list g = rotate_differentiable(grads[0], grads[1], saved[0], r);
      res[0] = g[0];
      res[1] = g[1];
    } else {
      for (size_t i = 0; i < grads.size(); ++i)
        if (grads[i].defined()) res[i] = rotate_differentiable(grads[i], Tensor(), saved[0], r)[0];
    }
    return res;
  }
};

variable_list rotate_differentiable(const Tensor& q, const Tensor& k, const Tensor& positions, const Rotation& r) {
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad())))
    return RotaryFunction::apply(q, optional(k), optional(positions), r.turns, r.interleaved, r.inverse, r.amplitude);
  return rotate(q, k, positions, r);
}

variable_list rotary(const Tensor& q, const Tensor& k, const Tensor& positions, const Rotation& r) {
  need(q.is_cuda(), "Input tensor must be on CUDA device");
  need(dtype_code(q) >= 0, "apply_rotary supports bf16, fp16 and fp32 tensors");
  need(q.dim() == 3 || q.dim() == 4, "query must be (batch, seqlen, nheads, headdim) or (tokens, nheads, headdim)");
  need(q.size(-2) > 0 && q.size(-1) > 0, "query must have heads");
  const int64_t lead = q.dim() - 2;
  if (k.defined()) {
    need(k.device() == q.device() && k.scalar_type() == q.scalar_type(), "query and key must have the same dtype and device");
    need(k.dim() == q.dim() && k.size(-1) == q.size(-1) && k.sizes().slice(0, lead) == q.sizes().slice(0, lead) && k.size(-2) > 0,
         "key must have query's batch, length and head dimension");
  }
  check_rotation(r.turns, q, q.size(-1));
  for (int64_t i = 0; i < q.dim(); ++i) need(q.size(i) <= 0x7FFFFFFF, "query is too large");
  if (positions.defined()) {
    need(positions.device() == q.device(), "positions must be on the same device as query");
    need(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, "positions must be int32 or int64");
    const int64_t S = q.size(lead - 1);
    const bool flat = positions.dim() == 1 && positions.size(0) == S;
    const bool rows = q.dim() == 4 && positions.dim() == 2 && (positions.size(0) == 1 || positions.size(0) == q.size(0)) && positions.size(1) == S;
    need(flat || rows, "positions must be (seqlen,) or ({1|batch}, seqlen)");
  }
  return rotate_differentiable(q, k, positions, r);
}

// ---- block tables ---------------------------------------------------------------------------------------------------
struct Tables {
  Tensor table, lengths, free_list, free_count, ticket;
  int64_t block_size;
};

void check_int(const Tensor& t, const Tensor& like, int64_t dims, const char* what) {
  need(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == dims && t.is_contiguous(), what);
}
void check_block_size(int64_t n) { need(n == 16 || n == 32 || n == 64 || n == 128, "block_size must be 16, 32, 64 or 128"); }

fdma_tables_params tables_params(const Tables& t, const Tensor& lengths) {
  need(t.table.is_cuda(), "Input tensor must be on CUDA device");
  check_int(t.table, t.table, 2, "the block table must be a contiguous int32 tensor (requests, blocks)");
  check_int(t.lengths, t.table, 1, "the tables' lengths must be a contiguous int32 tensor on the table's device");
  check_int(t.free_list, t.table, 1, "the free list must be a contiguous int32 tensor on the table's device");
  check_int(t.free_count, t.table, 1, "the free list's count must be a contiguous int32 tensor on the table's device");
  check_int(t.ticket, t.table, 1, "the ticket must be a contiguous int32 tensor on the table's device");
  check_int(lengths, t.table, 1, "lengths must be a contiguous int32 tensor on the table's device");
  check_block_size(t.block_size);
  const int64_t R = t.table.size(0);
  need(t.lengths.size(0) == R && lengths.size(0) == R, "there must be one length per request of the table");
  need(t.table.size(1) > 0 && t.free_list.size(0) > 0 && t.free_count.size(0) == 1 && t.ticket.size(0) == 1, "the tables are empty");
  need(R > 0 && R <= 8192, "tables hold 1 to 8192 requests");
  need(t.table.size(1) * t.block_size <= 0x7FFFFFFF && R * t.table.size(1) * t.block_size / 64 <= 0x7FFFFFFF && t.free_list.size(0) <= 0x7FFFFFFF,
       "the tables are too large");
  fdma_tables_params p = {};
  p.table = t.table.data_ptr<int32_t>();
  p.lengths = t.lengths.data_ptr<int32_t>();
  p.free_list = t.free_list.data_ptr<int32_t>();
  p.free_count = t.free_count.data_ptr<int32_t>();
  p.ticket = t.ticket.data_ptr<int32_t>();
  p.new_lengths = lengths.data_ptr<int32_t>();
  p.requests = static_cast<int32_t>(R);
  p.width = static_cast<int32_t>(t.table.size(1));
  p.num_blocks = static_cast<int32_t>(t.free_list.size(0));
  p.block_size = static_cast<int32_t>(t.block_size);
  return p;
}
void bump(std::initializer_list<Tensor> written) {
  for (const Tensor& t : written)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// `n` elements of a buffer from a byte offset on, as a tensor of its own that shares the storage
Tensor part_of(const Tensor& buf, int64_t bytes, int64_t n, at::ScalarType type) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), c10::scalarTypeToTypeMeta(type));
  c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  impl->set_sizes_contiguous({n});
  impl->set_storage_offset(bytes / static_cast<int64_t>(c10::elementSize(type)));
  return t;
}

std::vector<Tensor> extend(const Tables& t, const Tensor& new_lengths, int64_t tokens) {
  fdma_tables_params p = tables_params(t, new_lengths);
  need(tokens >= 0 && tokens <= (1 << 30), "the number of tokens must be between 0 and 2^30");
  at::AutoDispatchBelowADInplaceOrView guard;
  const c10::cuda::CUDAGuard device(t.table.device());
  const int64_t R = p.requests;
  p.tokens = static_cast<int32_t>(tokens);
  // the plan in one allocation
  const int64_t parts[] = {R + 1, tokens, tokens, R, R, R + 1, R + 1};
  const at::ScalarType types[] = {at::kInt, at::kInt, at::kLong, at::kInt, at::kBool, at::kInt, at::kInt};
  int64_t offsets[8] = {0};
  for (int i = 0; i < 7; ++i) offsets[i + 1] = offsets[i] + (parts[i] * static_cast<int64_t>(c10::elementSize(types[i])) + 127) / 128 * 128;
  const Tensor buf = empty({offsets[7]}, at::kByte, t.table);
  Tensor part[7];
  for (int i = 0; i < 7; ++i) part[i] = part_of(buf, offsets[i], parts[i], types[i]);
  p.cu_seqlens = part[0].data_ptr<int32_t>();
  p.positions = tokens ? part[1].data_ptr<int32_t>() : nullptr;
  p.slots = tokens ? part[2].data_ptr<int64_t>() : nullptr;
  p.lengths_after = part[3].data_ptr<int32_t>();
  p.granted = static_cast<uint8_t*>(part[4].data_ptr());
  p.cu_blocks = part[5].data_ptr<int32_t>();
  p.cu_chunks = part[6].data_ptr<int32_t>();
  check(api.tables_extend(&p, stream_of(t.table)), "fdma_tables_extend");
  bump({t.table, t.lengths, t.free_count});
  return std::vector<Tensor>(part, part + 7);
}

void truncate(const Tables& t, const Tensor& lengths) {
  const fdma_tables_params p = tables_params(t, lengths);
  const c10::cuda::CUDAGuard device(t.table.device());
  check(api.tables_truncate(&p, stream_of(t.table)), "fdma_tables_truncate");
  bump({t.table, t.lengths, t.free_count, t.free_list});
}

// ---- cache ----------------------------------------------------------------------------------------------------------
struct Cache {
  Tensor k, v, k_scale, v_scale, table, cu_seqlens, positions, lengths, cu_blocks, cu_chunks;
};

fdma_cache cache_params(const Cache& t, int64_t tokens) {
  need(t.k.is_cuda(), "Input tensor must be on CUDA device");
  for (const Tensor* x : {&t.k, &t.v})
    need(x->scalar_type() == at::kFloat8_e4m3fn && x->dim() == 4 && x->is_contiguous() && x->sizes() == t.k.sizes() && x->device() == t.k.device(),
         "the cache must be two contiguous float8_e4m3fn tensors (blocks, kv heads, block size, headdim)");
  for (const Tensor* x : {&t.k_scale, &t.v_scale})
    need(x->scalar_type() == at::kFloat && x->dim() == 2 && x->is_contiguous() && x->size(0) == t.k.size(0) && x->size(1) == t.k.size(1) &&
             x->device() == t.k.device(),
         "the cache's scales must be two contiguous float32 tensors (blocks, kv heads)");
  need(!(at::GradMode::is_enabled() && (t.k.requires_grad() || t.v.requires_grad() || t.k_scale.requires_grad() || t.v_scale.requires_grad())),
       "the 8-bit cache has no gradients: call it under torch.no_grad()");
  check_block_size(t.k.size(2));
  need(t.k.size(3) > 0 && t.k.size(3) % 16 == 0 && t.k.size(3) <= 256, "the cache supports head dimensions that are multiples of 16 up to 256");
  need(t.k.size(0) > 0 && t.k.size(1) > 0, "the cache is empty");
  need((reinterpret_cast<uintptr_t>(t.k.data_ptr()) | reinterpret_cast<uintptr_t>(t.v.data_ptr())) % 16 == 0, "the cache must be 16-byte aligned");
  check_int(t.table, t.k, 2, "the block table must be a contiguous int32 tensor (requests, blocks) on the cache's device");
  const int64_t R = t.table.size(0);
  check_int(t.cu_seqlens, t.k, 1, "the step's tensors must be contiguous int32 tensors on the cache's device");
  check_int(t.positions, t.k, 1, "the step's tensors must be contiguous int32 tensors on the cache's device");
  check_int(t.lengths, t.k, 1, "the step's tensors must be contiguous int32 tensors on the cache's device");
  check_int(t.cu_blocks, t.k, 1, "the step's tensors must be contiguous int32 tensors on the cache's device");
  check_int(t.cu_chunks, t.k, 1, "the step's tensors must be contiguous int32 tensors on the cache's device");
  need(R > 0 && t.table.size(1) > 0 && t.cu_seqlens.size(0) == R + 1 && t.cu_blocks.size(0) == R + 1 && t.cu_chunks.size(0) == R + 1 && t.lengths.size(0) == R,
       "the step and the tables are of different numbers of requests");
  need(t.positions.size(0) == tokens, "the step was made for another number of tokens");
  need(t.table.size(1) * t.k.size(2) <= 0x7FFFFFFF && t.k.size(0) <= 0x7FFFFFFF, "the tables are too large");
  fdma_cache c = {};
  c.k = t.k.data_ptr(); c.v = t.v.data_ptr();
  c.k_scale = t.k_scale.data_ptr<float>(); c.v_scale = t.v_scale.data_ptr<float>();
  c.table = t.table.data_ptr<int32_t>();
  c.cu_seqlens = t.cu_seqlens.data_ptr<int32_t>();
  c.lengths = t.lengths.data_ptr<int32_t>();
  c.cu_blocks = t.cu_blocks.data_ptr<int32_t>();
  c.cu_chunks = t.cu_chunks.data_ptr<int32_t>();
  c.positions = t.positions.data_ptr<int32_t>();
  c.requests = static_cast<int32_t>(R);
  c.width = static_cast<int32_t>(t.table.size(1));
  c.num_blocks = static_cast<int32_t>(t.k.size(0));
  c.h_k = static_cast<int32_t>(t.k.size(1));
  c.block_size = static_cast<int32_t>(t.k.size(2));
  c.d = static_cast<int32_t>(t.k.size(3));
  c.tokens = static_cast<int32_t>(tokens);
  return c;
}

void check_tokens(const Tensor& x, const Cache& t, const char* what) {
  need(x.device() == t.k.device() && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf) && x.dim() == 3 && x.size(2) == t.k.size(3) &&
           x.size(0) <= (1 << 30),
       what);
  need(!(at::GradMode::is_enabled() && x.requires_grad()), "the 8-bit cache has no gradients: call it under torch.no_grad()");
}

std::optional<Tensor> append(const Cache& t, const Tensor& key0, const Tensor& value0, const Tensor& query0, const Rotation& r) {
  check_tokens(key0, t, "key must be a bf16 or fp16 tensor (tokens, kv heads, headdim) on the cache's device");
  check_tokens(value0, t, "value must be a bf16 or fp16 tensor (tokens, kv heads, headdim) on the cache's device");
  need(key0.scalar_type() == value0.scalar_type() && key0.sizes() == value0.sizes(), "key and value must have the same dtype and shape");
  need(key0.size(1) == t.k.size(1), "key and the cache must have the same heads");
  fdma_cache_append_params p = {};
  p.c = cache_params(t, key0.size(0));
  if (query0.defined()) {
    check_tokens(query0, t, "query must be a bf16 or fp16 tensor (tokens, heads, headdim) on the cache's device");
    need(query0.scalar_type() == key0.scalar_type() && query0.size(0) == key0.size(0) && query0.size(1) > 0, "query must have key's dtype and tokens");
    need(r.turns.defined(), "query is turned by the frequencies: without them it is used as it is");
  }
  if (r.turns.defined()) {
    check_rotation(r.turns, key0, key0.size(2));
    p.turns = r.turns.data_ptr<int64_t>();
    p.rotary_dim = static_cast<int32_t>(2 * r.turns.size(0));
    p.interleaved = r.interleaved;
    p.amplitude = static_cast<float>(r.amplitude);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  const c10::cuda::CUDAGuard device(t.k.device());
  const Tensor key = inner_contiguous(key0), value = inner_contiguous(value0);
  Tensor query, out;
  p.key = key.data_ptr(); p.value = value.data_ptr();
  p.key_row_stride = stride_of(key, 0); p.key_head_stride = stride_of(key, 1);
  p.value_row_stride = stride_of(value, 0); p.value_head_stride = stride_of(value, 1);
  p.dtype = dtype_code(key);
  if (query0.defined()) {
    query = inner_contiguous(query0);
    out = empty(query.sizes(), query.scalar_type(), query);
    p.query = query.data_ptr(); p.query_out = out.data_ptr();
    p.h = static_cast<int32_t>(query.size(1));
    p.query_row_stride = stride_of(query, 0); p.query_head_stride = stride_of(query, 1);
    p.out_row_stride = stride_of(out, 0); p.out_head_stride = stride_of(out, 1);
  }
  check(api.cache_append(&p, stream_of(t.k)), "fdma_cache_append");
  bump({t.k, t.v, t.k_scale, t.v_scale});
  if (!out.defined()) return std::nullopt;
  return out;
}

Tensor attend(const Cache& t, const Tensor& query0, const Tensor& key_pos, const Tensor& count, const Tensor& bias0, std::optional<double> scale,
              bool causal, int64_t max_q, int64_t max_k) {
  check_tokens(query0, t, "query must be a bf16 or fp16 tensor (tokens, heads, headdim) on the cache's device");
  const int64_t T = query0.size(0), H = query0.size(1), d = query0.size(2), Hk = t.k.size(1), R = t.table.size(0);
  need(H > 0 && H % Hk == 0, "Number of heads in key/value must divide number of heads in query");
  need(max_q >= 0 && max_k >= 0, "max_seqlen_q and max_seqlen_k must not be negative");
  fdma_cache_attention_params p = {};
  p.c = cache_params(t, T);
  at::AutoDispatchBelowADInplaceOrView guard;
  const c10::cuda::CUDAGuard device(t.k.device());
  const cudaStream_t stream = stream_of(t.k);
  raise_if_timed_out(stream);
  const Tensor query = inner_contiguous(query0);
  Tensor bias, out = empty({T, H, d}, query.scalar_type(), query);
  p.query = query.data_ptr(); p.out = out.data_ptr();
  p.query_row_stride = stride_of(query, 0); p.query_head_stride = stride_of(query, 1);
  p.out_row_stride = stride_of(out, 0); p.out_head_stride = stride_of(out, 1);
  p.h = static_cast<int32_t>(H);
  p.dtype = dtype_code(query);
  p.is_causal = causal;
  p.softmax_scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(d)));
  p.max_seqlen_q = static_cast<int32_t>(std::min<int64_t>(max_q, T));
  p.max_seqlen_k = static_cast<int32_t>(std::min<int64_t>(max_k, static_cast<int64_t>(p.c.width) * p.c.block_size));
  if (bias0.defined()) {
    need(bias0.device() == query.device() && bias0.scalar_type() == query.scalar_type(), "bias must have the same dtype and device as query");
    need(bias0.dim() == 4 && (bias0.size(0) == 1 || bias0.size(0) == R) && (bias0.size(1) == 1 || bias0.size(1) == Hk || bias0.size(1) == H) &&
             bias0.size(2) == 1 && bias0.size(3) > 0 && bias0.size(3) <= 0x7FFFFFFF,
         "bias must be ({1|requests}, {1|num_heads_k|num_heads}, 1, keys)");
    need(!(at::GradMode::is_enabled() && bias0.requires_grad()), "the 8-bit cache has no gradients: call it under torch.no_grad()");
    bias = inner_contiguous(bias0);
    p.bias = bias.data_ptr();
    p.h_bias = static_cast<int32_t>(bias.size(1));
    p.bias_keys = static_cast<int32_t>(bias.size(3));
    p.bias_batch_stride = stride_of(bias, 0); p.bias_head_stride = stride_of(bias, 1);
  }
  if (key_pos.defined()) {
    check_int(key_pos, t.k, 3, "the kept keys must be a contiguous int32 tensor on the cache's device");
    check_int(count, t.k, 2, "the numbers of kept keys must be a contiguous int32 tensor on the cache's device");
    need((key_pos.size(0) == 1 || key_pos.size(0) == R) && (key_pos.size(1) == 1 || key_pos.size(1) == Hk) && key_pos.size(2) > 0 &&
             key_pos.size(2) <= 0x7FFFFFFF && count.size(0) == key_pos.size(0) && count.size(1) == key_pos.size(1),
         "the kept keys must be of ({1|requests}, {1|num_heads_k}) rows");
    p.kept_pos = key_pos.data_ptr<int32_t>();
    p.kept_count = count.data_ptr<int32_t>();
    p.kept_capacity = static_cast<int32_t>(key_pos.size(2));
    p.kept_batch_stride = stride_of(key_pos, 0); p.kept_head_stride = stride_of(key_pos, 1);
    p.count_batch_stride = stride_of(count, 0); p.count_head_stride = stride_of(count, 1);
  }
  const size_t bytes = api.cache_attention_workspace_bytes(&p);
  Tensor ws;
  if (bytes) {
    ws = empty({static_cast<int64_t>(bytes)}, at::kByte, query);
    p.workspace = ws.data_ptr();
    p.workspace_bytes = bytes;
  }
  check(api.cache_attention(&p, stream), "fdma_cache_attention");
  return out;
}

// ---- Python -----------------------------------------------------------------------------------------------------------
bool eager() { return !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::tracer::impl::is_dispatch_enabled(); }
bool ordinary(const Tensor& t) {
  constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                          c10::DispatchKey::Functionalize, c10::DispatchKey::Python, c10::DispatchKey::Conjugate,
                                          c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
  return !t.key_set().has_any(kWrapped) && !t._fw_grad(0).defined();
}
// The tensors of a Python tuple (None: undefined); false if one is not a plain tensor.
bool unpack(const py::tuple& in, std::vector<Tensor>& out) {
  if (!eager()) return false;
  for (const py::handle& o : in) {
    if (o.is_none()) {
      out.emplace_back();
      continue;
    }
    if (!THPVariable_CheckExact(o.ptr())) return false;
    out.push_back(THPVariable_Unpack(o.ptr()));
    if (!ordinary(out.back())) return false;
    need(out.back().layout() == at::kStrided, "tensors must be dense");
  }
  return true;
}
py::object wrap(const Tensor& t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }
py::tuple wrap(const std::vector<Tensor>& v) {
  py::tuple out(v.size());
  for (size_t i = 0; i < v.size(); ++i) out[i] = wrap(v[i]);
  return out;
}

// tensors: query, key or None, positions or None, turns
py::object py_rotary(const py::tuple& tensors, bool interleaved, double amplitude, bool inverse) {
  std::vector<Tensor> t;
  if (!unpack(tensors, t)) return py::none();
  variable_list res;
  {
    py::gil_scoped_release release;
    res = rotary(t.at(0), t.at(1), t.at(2), Rotation{t.at(3), interleaved, inverse, amplitude});
  }
  return wrap(res);
}

// tensors: table, lengths, free list, its count, ticket, new lengths
py::object py_extend(const py::tuple& tensors, int64_t block_size, int64_t tokens) {
  std::vector<Tensor> t, res;
  if (!unpack(tensors, t)) return py::none();
  {
    py::gil_scoped_release release;
    res = extend(Tables{t.at(0), t.at(1), t.at(2), t.at(3), t.at(4), block_size}, t.at(5), tokens);
  }
  return wrap(res);
}
bool py_truncate(const py::tuple& tensors, int64_t block_size) {
  std::vector<Tensor> t;
  if (!unpack(tensors, t)) return false;
  py::gil_scoped_release release;
  truncate(Tables{t.at(0), t.at(1), t.at(2), t.at(3), t.at(4), block_size}, t.at(5));
  return true;
}

Cache cache_of(const std::vector<Tensor>& t) { return Cache{t.at(0), t.at(1), t.at(2), t.at(3), t.at(4), t.at(5), t.at(6), t.at(7), t.at(8), t.at(9)}; }

// tensors: k, v, k_scale, v_scale, table, cu_seqlens, positions, lengths, cu_blocks, cu_chunks; key, value, query, turns.
// (done, the turned query or None)
py::object py_append(const py::tuple& tensors, bool interleaved, double amplitude) {
  std::vector<Tensor> t;
  if (!unpack(tensors, t)) return py::none();
  std::optional<Tensor> out;
  {
    py::gil_scoped_release release;
    out = append(cache_of(t), t.at(10), t.at(11), t.at(12), Rotation{t.at(13), interleaved, false, amplitude});
  }
  return py::make_tuple(out ? wrap(*out) : py::object(py::none()));
}

// tensors: the same ten; query, key_pos, count, bias
py::object py_attend(const py::tuple& tensors, const py::object& scale, bool causal, int64_t max_q, int64_t max_k) {
  std::vector<Tensor> t;
  if (!unpack(tensors, t)) return py::none();
  const std::optional<double> s = scale.is_none() ? std::nullopt : std::optional<double>(py::cast<double>(scale));
  Tensor out;
  {
    py::gil_scoped_release release;
    out = attend(cache_of(t), t.at(10), t.at(11), t.at(12), t.at(13), s, causal, max_q, max_k);
  }
  return wrap(out);
}

}  // namespace

void init_cache_ops(void* library) {
  auto get = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(dlsym(library, name));
    if (!fn) throw std::runtime_error(std::string("libfdma_sm100.so does not export ") + name);
  };
  get(api.rotary, "fdma_rotary");
  get(api.tables_extend, "fdma_tables_extend");
  get(api.tables_truncate, "fdma_tables_truncate");
  get(api.cache_append, "fdma_cache_append");
  get(api.cache_attention, "fdma_cache_attention");
  get(api.cache_attention_workspace_bytes, "fdma_cache_attention_workspace_bytes");
  get(api.strerror, "fdma_strerror");
  get(api.poll_kernel_status, "fdma_poll_kernel_status");
  get(api.last_kernel_status, "fdma_last_kernel_status");
}

void bind_cache_ops(py::module& m) {
  m.def("rotary", &py_rotary);
  m.def("tables_extend", &py_extend);
  m.def("tables_truncate", &py_truncate);
  m.def("cache_append", &py_append);
  m.def("cache_attention", &py_attend);
}
