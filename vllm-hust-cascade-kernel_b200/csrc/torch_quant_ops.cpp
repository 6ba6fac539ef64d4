// torch op registration of the 4-bit key-value cache (write, read, attention)
// and of the log probabilities of tokens. Same manner as torch_ops.cpp:
// arguments are checked here, outputs come from the caching allocator on the
// input's device, and the C ABI runs on the current stream.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <tuple>

#include "../../include/cascade_b200.h"

namespace cascade_torch {
namespace {

void check_rc(int rc) { TORCH_CHECK(rc == CASCADE_OK, cascade_last_error()); }

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return CASCADE_BF16;
    case at::kHalf: return CASCADE_FP16;
    case at::kFloat: return CASCADE_FP32;
    default: return -1;
  }
}

cascade_stream_t current_stream(const at::Tensor& t) {
  return reinterpret_cast<cascade_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

// `t` lives on `like`'s device, has type `type` and is contiguous.
void check_tensor(const char* op, const char* name, const at::Tensor& t, const at::Tensor& like, at::ScalarType type) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == like.get_device(), op, ": ", name, " must be on ", like.device());
  TORCH_CHECK(t.scalar_type() == type, op, ": ", name, " must be ", type);
  TORCH_CHECK(t.is_contiguous(), op, ": ", name, " must be contiguous");
}

// The two caches: equal shapes [blocks, block size, kv heads, 80].
void check_caches(const char* op, const at::Tensor& key_cache, const at::Tensor& value_cache, const at::Tensor& like) {
  check_tensor(op, "key_cache", key_cache, like, at::kByte);
  check_tensor(op, "value_cache", value_cache, like, at::kByte);
  TORCH_CHECK(key_cache.dim() == 4 && key_cache.size(3) == CASCADE_QUANT_ROW_BYTES, op,
              ": caches must be [blocks, block size, kv heads, 80]");
  TORCH_CHECK(value_cache.sizes() == key_cache.sizes(), op, ": caches must have equal shapes");
}

void cascade_quant_write(const at::Tensor& key, const at::Tensor& value, const at::Tensor& key_cache,
                         const at::Tensor& value_cache, const at::Tensor& slots) {
  const char* op = "cascade_quant_write";
  TORCH_CHECK(key.is_cuda(), op, ": key must be a CUDA tensor");
  TORCH_CHECK(key.scalar_type() == at::kBFloat16 || key.scalar_type() == at::kHalf, op,
              ": key and value must be bf16 or fp16");
  TORCH_CHECK(value.is_cuda() && value.get_device() == key.get_device() && value.scalar_type() == key.scalar_type(), op,
              ": value must be on key's device and have its type");
  check_caches(op, key_cache, value_cache, key);
  check_tensor(op, "slots", slots, key, at::kLong);
  TORCH_CHECK(key.dim() == 3 && key.size(1) == key_cache.size(2) && key.size(2) == 128, op,
              ": key must be [tokens, kv heads, 128]");
  TORCH_CHECK(value.sizes() == key.sizes(), op, ": value must have key's shape");
  TORCH_CHECK(key.stride(2) == 1 && value.stride(2) == 1, op, ": the last dimension of key and value must be contiguous");
  TORCH_CHECK(slots.dim() == 1 && slots.numel() == key.size(0), op, ": slots must have an entry per token");
  const c10::cuda::CUDAGuard guard(key.device());
  check_rc(::cascade_quant_write(key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0),
                                 value.stride(1), key_cache.data_ptr(), value_cache.data_ptr(),
                                 slots.data_ptr<int64_t>(), key.size(0), key.size(1), key.size(2), key_cache.size(0),
                                 key_cache.size(1), dtype_code(key.scalar_type()), current_stream(key)));
}

std::tuple<at::Tensor, at::Tensor> cascade_quant_read(const at::Tensor& key_cache, const at::Tensor& value_cache,
                                                      const at::Tensor& slots, at::ScalarType dtype) {
  const char* op = "cascade_quant_read";
  TORCH_CHECK(key_cache.is_cuda(), op, ": caches must be CUDA tensors");
  check_caches(op, key_cache, value_cache, key_cache);
  check_tensor(op, "slots", slots, key_cache, at::kLong);
  TORCH_CHECK(slots.dim() == 1, op, ": slots must be one-dimensional");
  const c10::cuda::CUDAGuard guard(key_cache.device());
  TORCH_CHECK(dtype_code(dtype) >= 0, op, ": key and value must be bf16, fp16 or fp32");
  auto key = at::empty({slots.numel(), key_cache.size(2), 128}, key_cache.options().dtype(dtype));
  auto value = at::empty_like(key);
  check_rc(::cascade_quant_read(key_cache.data_ptr(), value_cache.data_ptr(), slots.data_ptr<int64_t>(), key.data_ptr(),
                                value.data_ptr(), slots.numel(), key_cache.size(2), 128, key_cache.size(0),
                                key_cache.size(1), dtype_code(dtype), current_stream(key_cache)));
  return {key, value};
}

std::tuple<at::Tensor, at::Tensor> cascade_quant_decode(const at::Tensor& query, const at::Tensor& key_cache,
                                                        const at::Tensor& value_cache, const at::Tensor& block_table,
                                                        const at::Tensor& actual_q_seqlens,
                                                        const at::Tensor& actual_kv_seqlens, int64_t q_seqlen_value,
                                                        double scale, bool causal) {
  const char* op = "cascade_quant_decode";
  TORCH_CHECK(query.is_cuda(), op, ": query must be a CUDA tensor");
  TORCH_CHECK(query.scalar_type() == at::kBFloat16 || query.scalar_type() == at::kHalf, op,
              ": query must be bf16 or fp16");
  check_tensor(op, "query", query, query, query.scalar_type());
  check_caches(op, key_cache, value_cache, query);
  check_tensor(op, "block_table", block_table, query, at::kInt);
  check_tensor(op, "actual_q_seqlens", actual_q_seqlens, query, at::kLong);
  check_tensor(op, "actual_kv_seqlens", actual_kv_seqlens, query, at::kLong);
  TORCH_CHECK(query.dim() == 3 && query.size(2) == 128, op, ": query must be [tokens, heads, 128]");
  TORCH_CHECK(block_table.dim() == 2, op, ": block_table must be (B, cols)");
  const int64_t batch = actual_kv_seqlens.numel();
  TORCH_CHECK(actual_q_seqlens.numel() == batch, op, ": seqlen tensors must have batch entries");
  TORCH_CHECK(block_table.size(0) >= batch, op, ": block_table must have a row per request");
  cascade_quant_attn_t d{};
  d.query = query.data_ptr();
  d.key_cache = key_cache.data_ptr();
  d.value_cache = value_cache.data_ptr();
  d.block_table = block_table.data_ptr<int32_t>();
  d.actual_q_seqlens = actual_q_seqlens.data_ptr<int64_t>();
  d.actual_kv_seqlens = actual_kv_seqlens.data_ptr<int64_t>();
  d.num_tokens = query.size(0);
  d.num_heads = query.size(1);
  d.kv_heads = key_cache.size(2);
  d.head_dim = 128;
  d.num_blocks = key_cache.size(0);
  d.block_size = key_cache.size(1);
  d.batch = batch;
  d.block_cols = block_table.size(1);
  d.q_seqlen_value = q_seqlen_value;
  d.scale = static_cast<float>(scale);
  d.causal = causal;
  d.dtype = dtype_code(query.scalar_type());
  const c10::cuda::CUDAGuard guard(query.device());
  auto out = at::empty_like(query);
  auto lse = at::empty({d.num_tokens * d.num_heads}, query.options().dtype(at::kFloat));
  const size_t ws_bytes = cascade_quant_decode_workspace_size(&d);
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({static_cast<int64_t>(ws_bytes)}, query.options().dtype(at::kByte));
  check_rc(::cascade_quant_decode(&d, out.data_ptr(), lse.data_ptr<float>(), ws_bytes ? ws.data_ptr() : nullptr,
                                  ws_bytes, current_stream(query)));
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> cascade_token_logprobs(const at::Tensor& logits,
                                                                                              const at::Tensor& tokens,
                                                                                              int64_t top) {
  const char* op = "cascade_token_logprobs";
  TORCH_CHECK(logits.is_cuda(), op, ": logits must be a CUDA tensor");
  const int32_t type = dtype_code(logits.scalar_type());
  TORCH_CHECK(type >= 0, op, ": logits must be bf16, fp16 or fp32");
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1), op,
              ": logits must be [rows, vocabulary] with contiguous rows");
  check_tensor(op, "tokens", tokens, logits, at::kLong);
  const int64_t N = logits.size(0), V = logits.size(1);
  TORCH_CHECK(tokens.sizes() == at::IntArrayRef({N}), op, ": tokens must have an entry per row");
  TORCH_CHECK(top >= 0 && top <= 32 && top <= V, op, ": top must be at most 32 and at most the vocabulary");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto f32 = logits.options().dtype(at::kFloat);
  auto logprob = at::empty({N}, f32), entropy = at::empty({N}, f32), top_logprobs = at::empty({N, top}, f32);
  auto rank = at::empty({N}, tokens.options()), top_tokens = at::empty({N, top}, tokens.options());
  check_rc(::cascade_token_logprobs(logits.data_ptr(), logits.stride(0), tokens.data_ptr<int64_t>(), type, N, V, top,
                                    logprob.data_ptr<float>(), entropy.data_ptr<float>(), rank.data_ptr<int64_t>(),
                                    top ? top_logprobs.data_ptr<float>() : nullptr,
                                    top ? top_tokens.data_ptr<int64_t>() : nullptr, current_stream(logits)));
  return {logprob, entropy, rank, top_logprobs, top_tokens};
}

}  // namespace
}  // namespace cascade_torch

TORCH_LIBRARY_FRAGMENT(npu, m) {
  m.def(
      "cascade_quant_write(Tensor key, Tensor value, Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor slots) "
      "-> ()");
  m.def("cascade_quant_read(Tensor key_cache, Tensor value_cache, Tensor slots, ScalarType dtype) -> (Tensor, Tensor)");
  m.def(
      "cascade_quant_decode(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, "
      "Tensor actual_q_seqlens, Tensor actual_kv_seqlens, int q_seqlen_value, float scale, bool causal=True) "
      "-> (Tensor, Tensor)");
  m.def(
      "cascade_token_logprobs(Tensor logits, Tensor tokens, int top=0) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
  m.impl("cascade_quant_write", TORCH_FN(cascade_torch::cascade_quant_write));
  m.impl("cascade_quant_read", TORCH_FN(cascade_torch::cascade_quant_read));
  m.impl("cascade_quant_decode", TORCH_FN(cascade_torch::cascade_quant_decode));
  m.impl("cascade_token_logprobs", TORCH_FN(cascade_torch::cascade_token_logprobs));
}
