// torch op registration of the paged latent cache: latent attention (absorbed
// and expanded), pages, verification of drafted tokens. Same manner as
// torch_ops.cpp: arguments are checked here, outputs come from the caching
// allocator on the input's device, and the C ABI runs on the current stream.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <tuple>
#include <vector>

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

at::Tensor bytes(size_t n, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

std::tuple<at::Tensor, at::Tensor> cascade_latent_decode(const at::Tensor& query, const at::Tensor& cache,
                                                         const at::Tensor& block_table,
                                                         const at::Tensor& actual_q_seqlens,
                                                         const at::Tensor& actual_kv_seqlens, int64_t q_seqlen_value,
                                                         double scale, bool causal) {
  const char* op = "cascade_latent_decode";
  TORCH_CHECK(query.is_cuda(), op, ": query must be a CUDA tensor");
  TORCH_CHECK(query.scalar_type() == at::kBFloat16 || query.scalar_type() == at::kHalf, op,
              ": query/cache must be bf16 or fp16");
  check_tensor(op, "query", query, query, query.scalar_type());
  check_tensor(op, "cache", cache, query, query.scalar_type());
  check_tensor(op, "block_table", block_table, query, at::kInt);
  check_tensor(op, "actual_q_seqlens", actual_q_seqlens, query, at::kLong);
  check_tensor(op, "actual_kv_seqlens", actual_kv_seqlens, query, at::kLong);
  TORCH_CHECK(query.dim() == 3 && query.size(2) == 576, op, ": query must be [tokens, heads, 576]");
  TORCH_CHECK(cache.dim() == 3 && cache.size(2) == 576, op, ": cache must be [blocks, block size, 576]");
  TORCH_CHECK(block_table.dim() == 2, op, ": block_table must be (B, cols)");
  const int64_t batch = actual_kv_seqlens.numel();
  TORCH_CHECK(actual_q_seqlens.numel() == batch, op, ": seqlen tensors must have batch entries");
  TORCH_CHECK(block_table.size(0) >= batch, op, ": block_table must have a row per request");
  cascade_latent_attn_t d{};
  d.query = query.data_ptr();
  d.cache = cache.data_ptr();
  d.block_table = block_table.data_ptr<int32_t>();
  d.actual_q_seqlens = actual_q_seqlens.data_ptr<int64_t>();
  d.actual_kv_seqlens = actual_kv_seqlens.data_ptr<int64_t>();
  d.num_tokens = query.size(0);
  d.num_heads = query.size(1);
  d.latent_dim = 512;
  d.rope_dim = 64;
  d.num_blocks = cache.size(0);
  d.block_size = cache.size(1);
  d.batch = batch;
  d.block_cols = block_table.size(1);
  d.q_seqlen_value = q_seqlen_value;
  d.scale = static_cast<float>(scale);
  d.causal = causal;
  d.dtype = dtype_code(query.scalar_type());
  const c10::cuda::CUDAGuard guard(query.device());
  auto out = at::empty({d.num_tokens, d.num_heads, 512}, query.options());
  auto lse = at::empty({d.num_tokens * d.num_heads}, query.options().dtype(at::kFloat));
  const size_t ws_bytes = cascade_latent_decode_workspace_size(&d);
  at::Tensor ws;
  if (ws_bytes) ws = bytes(ws_bytes, query);
  check_rc(cascade_latent_decode(&d, out.data_ptr(), lse.data_ptr<float>(), ws_bytes ? ws.data_ptr() : nullptr,
                                 ws_bytes, current_stream(query)));
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> cascade_latent_prefill(const at::Tensor& query, const at::Tensor& key,
                                                          const at::Tensor& key_rope, const at::Tensor& value,
                                                          const at::Tensor& cu_q_seqlens,
                                                          const at::Tensor& cu_kv_seqlens, int64_t max_q_seqlen,
                                                          double scale, bool causal) {
  const char* op = "cascade_latent_prefill";
  TORCH_CHECK(query.is_cuda(), op, ": query must be a CUDA tensor");
  TORCH_CHECK(query.scalar_type() == at::kBFloat16 || query.scalar_type() == at::kHalf, op,
              ": inputs must be bf16 or fp16");
  check_tensor(op, "query", query, query, query.scalar_type());
  check_tensor(op, "cu_q_seqlens", cu_q_seqlens, query, at::kLong);
  check_tensor(op, "cu_kv_seqlens", cu_kv_seqlens, query, at::kLong);
  for (const at::Tensor& t : {key, key_rope, value}) {
    TORCH_CHECK(t.is_cuda() && t.get_device() == query.get_device(), op, ": all inputs must be on one device");
    TORCH_CHECK(t.scalar_type() == query.scalar_type(), op, ": all inputs must have query's type");
  }
  const int64_t H = query.dim() == 3 ? query.size(1) : 0, S = key.size(0);
  TORCH_CHECK(query.dim() == 3 && query.size(2) == 192, op, ": query must be [tokens, heads, 192]");
  TORCH_CHECK(key.dim() == 3 && key.size(1) == H && key.size(2) == 128, op, ": key must be [kv tokens, heads, 128]");
  TORCH_CHECK(value.dim() == 3 && value.size(0) == S && value.size(1) == H && value.size(2) == 128, op,
              ": value must be [kv tokens, heads, 128]");
  TORCH_CHECK(key_rope.dim() == 2 && key_rope.size(0) == S && key_rope.size(1) == 64, op,
              ": key_rope must be [kv tokens, 64]");
  TORCH_CHECK(key.stride(2) == 1 && value.stride(2) == 1 && key_rope.stride(1) == 1, op,
              ": the last dimension of key, key_rope and value must be contiguous");
  TORCH_CHECK(cu_q_seqlens.dim() == 1 && cu_q_seqlens.numel() >= 1 && cu_q_seqlens.numel() == cu_kv_seqlens.numel(),
              op, ": cumulative lengths must be two [batch + 1] tensors");
  cascade_latent_prefill_t d{};
  d.query = query.data_ptr();
  d.key = key.data_ptr();
  d.key_rope = key_rope.data_ptr();
  d.value = value.data_ptr();
  d.cu_q_seqlens = cu_q_seqlens.data_ptr<int64_t>();
  d.cu_kv_seqlens = cu_kv_seqlens.data_ptr<int64_t>();
  d.num_tokens = query.size(0);
  d.num_kv = S;
  d.num_heads = H;
  d.batch = cu_q_seqlens.numel() - 1;
  d.max_q_seqlen = max_q_seqlen;
  d.key_token_stride = key.stride(0);
  d.key_head_stride = key.stride(1);
  d.rope_token_stride = key_rope.stride(0);
  d.value_token_stride = value.stride(0);
  d.value_head_stride = value.stride(1);
  d.scale = static_cast<float>(scale);
  d.causal = causal;
  d.dtype = dtype_code(query.scalar_type());
  const c10::cuda::CUDAGuard guard(query.device());
  auto out = at::empty({d.num_tokens, H, 128}, query.options());
  auto lse = at::empty({d.num_tokens * H}, query.options().dtype(at::kFloat));
  check_rc(cascade_latent_prefill(&d, out.data_ptr(), lse.data_ptr<float>(), current_stream(query)));
  return {out, lse};
}

// The pools of a page op: equal shapes [num_blocks, block size, ...],
// contiguous, one device.
struct PoolArgs {
  std::vector<void*> ptrs;
  int64_t num_blocks, block_size, row_bytes;
};

PoolArgs pool_args(const char* op, at::TensorList pools) {
  TORCH_CHECK(!pools.empty(), op, ": needs at least one pool");
  const at::Tensor& first = pools[0];
  TORCH_CHECK(first.is_cuda(), op, ": pools must be CUDA tensors");
  TORCH_CHECK(first.dim() >= 3 && first.size(1) > 0, op, ": pools must be [blocks, block size, ...]");
  PoolArgs a;
  for (const at::Tensor& t : pools) {
    check_tensor(op, "every pool", t, first, first.scalar_type());
    TORCH_CHECK(t.sizes() == first.sizes(), op, ": pools must have equal shapes");
    a.ptrs.push_back(t.data_ptr());
  }
  a.num_blocks = first.size(0);
  a.block_size = first.size(1);
  a.row_bytes = first.numel() ? first.numel() / (a.num_blocks * a.block_size) * first.element_size() : 0;
  return a;
}

void check_state(const char* op, const at::Tensor& block_table, const at::Tensor& kv_seqlens,
                 const at::Tensor& page_refs, const at::Tensor& like) {
  TORCH_CHECK(like.is_cuda(), op, ": all inputs must be CUDA tensors");
  check_tensor(op, "block_table", block_table, like, at::kInt);
  check_tensor(op, "kv_seqlens", kv_seqlens, like, at::kLong);
  check_tensor(op, "page_refs", page_refs, like, at::kInt);
  TORCH_CHECK(block_table.dim() == 2 && kv_seqlens.dim() == 1 && kv_seqlens.numel() == block_table.size(0), op,
              ": block_table must be (rows, cols) and kv_seqlens have its rows");
  TORCH_CHECK(page_refs.dim() == 1, op, ": page_refs must be one-dimensional");
}

void cascade_page_copy(at::TensorList pools, const at::Tensor& src, const at::Tensor& dst) {
  const char* op = "cascade_page_copy";
  const PoolArgs a = pool_args(op, pools);
  check_tensor(op, "src", src, pools[0], at::kLong);
  check_tensor(op, "dst", dst, pools[0], at::kLong);
  TORCH_CHECK(src.dim() == 1 && dst.dim() == 1 && src.numel() == dst.numel(), op,
              ": src and dst must be one-dimensional and equally long");
  const c10::cuda::CUDAGuard guard(pools[0].device());
  check_rc(cascade_page_copy(a.ptrs.data(), static_cast<int64_t>(a.ptrs.size()), a.num_blocks,
                             a.row_bytes * a.block_size, src.data_ptr<int64_t>(), dst.data_ptr<int64_t>(), src.numel(),
                             current_stream(pools[0])));
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> cascade_page_fork(at::TensorList pools, const at::Tensor& block_table,
                                                                 const at::Tensor& kv_seqlens,
                                                                 const at::Tensor& page_refs,
                                                                 const at::Tensor& parents) {
  const char* op = "cascade_page_fork";
  const PoolArgs a = pool_args(op, pools);
  check_state(op, block_table, kv_seqlens, page_refs, pools[0]);
  check_tensor(op, "parents", parents, pools[0], at::kLong);
  TORCH_CHECK(parents.dim() == 1, op, ": parents must be one-dimensional");
  TORCH_CHECK(page_refs.numel() == a.num_blocks, op, ": page_refs must have an entry per page of the pools");
  const c10::cuda::CUDAGuard guard(pools[0].device());
  const int64_t n = parents.numel(), cols = block_table.size(1);
  auto table = at::empty({n, cols}, block_table.options());
  auto lens = at::empty({n}, kv_seqlens.options());
  auto refs = at::empty_like(page_refs);
  const size_t ws_bytes = cascade_page_fork_workspace_size(a.num_blocks, n);
  auto ws = bytes(ws_bytes, pools[0]);
  check_rc(cascade_page_fork(a.ptrs.data(), static_cast<int64_t>(a.ptrs.size()), a.num_blocks, a.block_size,
                             a.row_bytes, block_table.data_ptr<int32_t>(), block_table.size(0), cols,
                             kv_seqlens.data_ptr<int64_t>(), page_refs.data_ptr<int32_t>(),
                             parents.data_ptr<int64_t>(), n, table.data_ptr<int32_t>(), lens.data_ptr<int64_t>(),
                             refs.data_ptr<int32_t>(), ws.data_ptr(), ws_bytes, current_stream(pools[0])));
  return {table, lens, refs};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> cascade_page_free(const at::Tensor& block_table,
                                                                 const at::Tensor& kv_seqlens,
                                                                 const at::Tensor& page_refs,
                                                                 const at::Tensor& keep_seqlens, int64_t block_size) {
  const char* op = "cascade_page_free";
  check_state(op, block_table, kv_seqlens, page_refs, block_table);
  check_tensor(op, "keep_seqlens", keep_seqlens, block_table, at::kLong);
  TORCH_CHECK(keep_seqlens.sizes() == kv_seqlens.sizes(), op, ": keep_seqlens must have an entry per row");
  const c10::cuda::CUDAGuard guard(block_table.device());
  auto table = at::empty_like(block_table);
  auto lens = at::empty_like(kv_seqlens);
  auto refs = at::empty_like(page_refs);
  check_rc(cascade_page_free(block_table.data_ptr<int32_t>(), block_table.size(0), block_table.size(1),
                             kv_seqlens.data_ptr<int64_t>(), page_refs.data_ptr<int32_t>(), page_refs.numel(),
                             keep_seqlens.data_ptr<int64_t>(), block_size, table.data_ptr<int32_t>(),
                             lens.data_ptr<int64_t>(), refs.data_ptr<int32_t>(), current_stream(block_table)));
  return {table, lens, refs};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> cascade_page_compact(at::TensorList pools,
                                                                    const at::Tensor& block_table,
                                                                    const at::Tensor& kv_seqlens,
                                                                    const at::Tensor& page_refs) {
  const char* op = "cascade_page_compact";
  const PoolArgs a = pool_args(op, pools);
  check_state(op, block_table, kv_seqlens, page_refs, pools[0]);
  TORCH_CHECK(page_refs.numel() == a.num_blocks, op, ": page_refs must have an entry per page of the pools");
  const c10::cuda::CUDAGuard guard(pools[0].device());
  auto table = at::empty_like(block_table);
  auto refs = at::empty_like(page_refs);
  auto live = at::empty({1}, page_refs.options());
  const size_t ws_bytes = cascade_page_compact_workspace_size(a.num_blocks);
  auto ws = bytes(ws_bytes, pools[0]);
  check_rc(cascade_page_compact(a.ptrs.data(), static_cast<int64_t>(a.ptrs.size()), a.num_blocks, a.block_size,
                                a.row_bytes, block_table.data_ptr<int32_t>(), block_table.size(0),
                                block_table.size(1), kv_seqlens.data_ptr<int64_t>(), page_refs.data_ptr<int32_t>(),
                                table.data_ptr<int32_t>(), refs.data_ptr<int32_t>(), live.data_ptr<int32_t>(),
                                ws.data_ptr(), ws_bytes, current_stream(pools[0])));
  return {table, refs, live};
}

std::tuple<at::Tensor, at::Tensor> cascade_verify_drafts(const at::Tensor& draft_tokens, const at::Tensor& draft_lens,
                                                         const std::optional<at::Tensor>& draft_probs,
                                                         const at::Tensor& target_probs, const at::Tensor& uniform,
                                                         const at::Tensor& noise) {
  const char* op = "cascade_verify_drafts";
  TORCH_CHECK(target_probs.is_cuda(), op, ": target_probs must be a CUDA tensor");
  const auto type = target_probs.scalar_type();
  TORCH_CHECK(dtype_code(type) >= 0, op, ": probabilities must be bf16, fp16 or fp32");
  const at::Tensor& like = target_probs;
  check_tensor(op, "target_probs", target_probs, like, type);
  check_tensor(op, "draft_tokens", draft_tokens, like, at::kLong);
  check_tensor(op, "draft_lens", draft_lens, like, at::kLong);
  check_tensor(op, "uniform", uniform, like, at::kFloat);
  check_tensor(op, "noise", noise, like, at::kFloat);
  TORCH_CHECK(draft_tokens.dim() == 2, op, ": draft_tokens must be [batch, drafts]");
  const int64_t B = draft_tokens.size(0), K = draft_tokens.size(1);
  TORCH_CHECK(target_probs.dim() == 3 && target_probs.size(0) == B && target_probs.size(1) == K + 1, op,
              ": target_probs must be [batch, drafts + 1, vocabulary]");
  const int64_t V = target_probs.size(2);
  const bool has_draft = draft_probs.has_value() && draft_probs->defined();
  if (has_draft) {
    check_tensor(op, "draft_probs", *draft_probs, like, type);
    TORCH_CHECK(draft_probs->sizes() == at::IntArrayRef({B, K, V}), op,
                ": draft_probs must be [batch, drafts, vocabulary]");
  }
  TORCH_CHECK(draft_lens.sizes() == at::IntArrayRef({B}), op, ": draft_lens must be [batch]");
  TORCH_CHECK(uniform.sizes() == draft_tokens.sizes(), op, ": uniform must be [batch, drafts]");
  TORCH_CHECK(noise.sizes() == at::IntArrayRef({B, V}), op, ": noise must be [batch, vocabulary]");
  const c10::cuda::CUDAGuard guard(like.device());
  auto tokens = at::empty({B, K + 1}, draft_tokens.options());
  auto accepted = at::empty({B}, draft_lens.options());
  check_rc(cascade_verify_drafts(draft_tokens.data_ptr<int64_t>(), draft_lens.data_ptr<int64_t>(),
                                 has_draft ? draft_probs->data_ptr() : nullptr, target_probs.data_ptr(),
                                 uniform.data_ptr<float>(), noise.data_ptr<float>(), dtype_code(type), B, K, V,
                                 tokens.data_ptr<int64_t>(), accepted.data_ptr<int64_t>(), current_stream(like)));
  return {tokens, accepted};
}

}  // namespace
}  // namespace cascade_torch

TORCH_LIBRARY_FRAGMENT(npu, m) {
  m.def(
      "cascade_latent_decode(Tensor query, Tensor cache, Tensor block_table, Tensor actual_q_seqlens, "
      "Tensor actual_kv_seqlens, int q_seqlen_value, float scale, bool causal=True) -> (Tensor, Tensor)");
  m.def(
      "cascade_latent_prefill(Tensor query, Tensor key, Tensor key_rope, Tensor value, Tensor cu_q_seqlens, "
      "Tensor cu_kv_seqlens, int max_q_seqlen, float scale, bool causal=True) -> (Tensor, Tensor)");
  m.def("cascade_page_copy(Tensor(a!)[] pools, Tensor src, Tensor dst) -> ()");
  m.def(
      "cascade_page_fork(Tensor(a!)[] pools, Tensor block_table, Tensor kv_seqlens, Tensor page_refs, "
      "Tensor parents) -> (Tensor, Tensor, Tensor)");
  m.def(
      "cascade_page_free(Tensor block_table, Tensor kv_seqlens, Tensor page_refs, Tensor keep_seqlens, "
      "int block_size) -> (Tensor, Tensor, Tensor)");
  m.def(
      "cascade_page_compact(Tensor(a!)[] pools, Tensor block_table, Tensor kv_seqlens, Tensor page_refs) "
      "-> (Tensor, Tensor, Tensor)");
  m.def(
      "cascade_verify_drafts(Tensor draft_tokens, Tensor draft_lens, Tensor? draft_probs, Tensor target_probs, "
      "Tensor uniform, Tensor noise) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
  m.impl("cascade_latent_decode", TORCH_FN(cascade_torch::cascade_latent_decode));
  m.impl("cascade_latent_prefill", TORCH_FN(cascade_torch::cascade_latent_prefill));
  m.impl("cascade_page_copy", TORCH_FN(cascade_torch::cascade_page_copy));
  m.impl("cascade_page_fork", TORCH_FN(cascade_torch::cascade_page_fork));
  m.impl("cascade_page_free", TORCH_FN(cascade_torch::cascade_page_free));
  m.impl("cascade_page_compact", TORCH_FN(cascade_torch::cascade_page_compact));
  m.impl("cascade_verify_drafts", TORCH_FN(cascade_torch::cascade_verify_drafts));
}
