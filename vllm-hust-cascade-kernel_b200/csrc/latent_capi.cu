// C ABI entry points of the paged latent cache (include/cascade_b200.h):
// latent attention, pages, verification of drafted tokens. Argument checks and
// launches; nothing here reads device memory.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/cascade_b200.h"
#include "kernels.h"

namespace cascade {
namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}

int finish(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return CASCADE_OK;
  return fail(CASCADE_ERR_CUDA, "%s: CUDA error %d (%s)", op, static_cast<int>(e), cudaGetErrorString(e));
}

bool misaligned(const void* p, uintptr_t bytes = 16) { return reinterpret_cast<uintptr_t>(p) & (bytes - 1); }
bool half_type(int32_t t) { return t == CASCADE_BF16 || t == CASCADE_FP16; }
constexpr int64_t kI32 = INT32_MAX;

int check_workspace(const char* op, const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need))
    return fail(CASCADE_ERR_WORKSPACE, "%s: workspace too small (%zu bytes, need %zu)", op, have, need);
  if (need && misaligned(ws)) return fail(CASCADE_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", op);
  return CASCADE_OK;
}

int check_decode(const cascade_latent_attn_t* p, const char* op) {
  if (!p) return fail(CASCADE_ERR_INVALID, "%s: null argument", op);
  if (!half_type(p->dtype)) return fail(CASCADE_ERR_INVALID, "%s: query/cache must be bf16 or fp16", op);
  if (p->latent_dim != kLatentDim || p->rope_dim != kLatentRow - kLatentDim)
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: cache rows must hold 512 latent and 64 rotary values", op);
  const int64_t bs = p->block_size;
  if (bs < 16 || bs > 512 || (bs & (bs - 1)))
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: paged blockSize must be one of 16, 32, 64, 128, 256, 512", op);
  if (p->num_tokens < 0 || p->num_heads < 0 || p->batch < 0 || p->num_blocks < 0 || p->block_cols < 0)
    return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (p->q_seqlen_value < 0)
    return fail(CASCADE_ERR_INVALID, "%s: q_seqlen_value must be >= 0 (0 = per request)", op);
  if (p->batch > kI32 || p->q_seqlen_value > kI32)  // their product has to hold in 64 bits
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large for 32-bit row indices", op);
  if (p->q_seqlen_value > 0 && p->num_tokens != p->batch * p->q_seqlen_value)
    return fail(CASCADE_ERR_INVALID, "%s: with q_seqlen_value=%lld, query.size(0) must equal batch * q_seqlen_value",
                op, static_cast<long long>(p->q_seqlen_value));
  if (p->num_heads > kI32 || p->num_tokens > kI32 || p->num_tokens * p->num_heads > kI32 ||
      p->block_cols > kI32 || p->num_blocks > kI32 || p->num_blocks * bs > kI32 ||
      p->block_cols * bs > kI32 / 2)
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large for 32-bit row indices", op);
  if (!(p->scale > 0.f) || p->scale > 3e38f) return fail(CASCADE_ERR_INVALID, "%s: scale must be positive", op);
  if (p->flags & ~CASCADE_FLAG_DEBUG_STALL) return fail(CASCADE_ERR_INVALID, "%s: unknown flags", op);
  return CASCADE_OK;
}

LatentDecodeLaunch decode_launch(const cascade_latent_attn_t* p, void* out, float* lse) {
  LatentDecodeLaunch L = {};
  L.query = p->query;
  L.cache = p->cache;
  L.block_table = p->block_table;
  L.q_lens = p->q_seqlen_value > 0 ? nullptr : p->actual_q_seqlens;
  L.kv_lens = p->actual_kv_seqlens;
  L.out = out;
  L.lse = lse;
  L.num_tokens = p->num_tokens;
  L.num_heads = static_cast<int32_t>(p->num_heads);
  L.num_blocks = static_cast<int32_t>(p->num_blocks);
  L.block_size = static_cast<int32_t>(p->block_size);
  L.batch = static_cast<int32_t>(p->batch);
  L.block_cols = static_cast<int32_t>(p->block_cols);
  L.q_len = static_cast<int32_t>(p->q_seqlen_value);
  L.causal = p->causal != 0;
  L.scale = p->scale;
  L.debug_stall = (p->flags & CASCADE_FLAG_DEBUG_STALL) != 0;
  // The warps that load a unit's query wait while the unit before it is worked on: 1 to 2 us per 64 cached tokens
  // (measured), so 4 on top of the 100 ms of the other waits.
  L.wait_limit_us = L.debug_stall ? 1000 : static_cast<uint32_t>(100000 + p->block_cols * p->block_size / 16);
  return L;
}

// The pools and index arrays that fork, free and compact share.
int check_pages(const char* op, void* const* pools, int64_t num_pools, int64_t num_blocks, int64_t block_size,
                int64_t row_bytes, int64_t rows, int64_t cols) {
  if (num_pools < 0 || num_blocks < 0 || rows < 0 || cols < 0 || row_bytes < 0)
    return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (block_size < 1) return fail(CASCADE_ERR_INVALID, "%s: block size must be >= 1", op);
  if (num_blocks > kI32 - 1 || rows > kI32 || cols > kI32 || block_size > kI32)
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large for 32-bit page ids", op);
  if (num_pools && !pools) return fail(CASCADE_ERR_INVALID, "%s: null pool list", op);
  if (num_pools && row_bytes % 16) return fail(CASCADE_ERR_INVALID, "%s: pool rows must be multiples of 16 bytes", op);
  for (int64_t i = 0; i < num_pools; ++i)
    if (!pools[i] || misaligned(pools[i]))
      return fail(CASCADE_ERR_INVALID, "%s: pools must be non-null and 16-byte aligned", op);
  return CASCADE_OK;
}

}  // namespace
}  // namespace cascade

using namespace cascade;

extern "C" {

size_t cascade_latent_decode_workspace_size(const cascade_latent_attn_t* p) {
  if (check_decode(p, "cascade_latent_decode") != CASCADE_OK) return 0;
  if (p->num_tokens == 0 || p->num_heads == 0 || p->batch == 0) return 0;
  return latent_decode_workspace(decode_launch(p, nullptr, nullptr));
}

int cascade_latent_decode(const cascade_latent_attn_t* p, void* out, float* lse, void* workspace,
                          size_t workspace_bytes, cascade_stream_t stream) {
  const char* op = "cascade_latent_decode";
  int rc = check_decode(p, op);
  if (rc) return rc;
  if (p->num_tokens == 0 || p->num_heads == 0) return CASCADE_OK;
  if (p->batch == 0) return fail(CASCADE_ERR_INVALID, "%s: query tokens but no requests", op);
  if (!p->query || !p->actual_kv_seqlens || !out || !lse || (p->block_cols && !p->block_table) ||
      (p->num_blocks && !p->cache) || (p->q_seqlen_value == 0 && !p->actual_q_seqlens))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  if (misaligned(p->query) || misaligned(p->cache) || misaligned(out))
    return fail(CASCADE_ERR_INVALID, "%s: query/cache/out must be 16-byte aligned", op);
  const LatentDecodeLaunch L = decode_launch(p, out, lse);
  rc = check_workspace(op, workspace, workspace_bytes, latent_decode_workspace(L));
  if (rc) return rc;
  return finish(op, launch_latent_decode(L, p->dtype == CASCADE_FP16, workspace,
                                         reinterpret_cast<cudaStream_t>(stream)));
}

int cascade_latent_prefill(const cascade_latent_prefill_t* p, void* out, float* lse, cascade_stream_t stream) {
  const char* op = "cascade_latent_prefill";
  if (!p) return fail(CASCADE_ERR_INVALID, "%s: null argument", op);
  if (!half_type(p->dtype)) return fail(CASCADE_ERR_INVALID, "%s: inputs must be bf16 or fp16", op);
  if (p->num_tokens < 0 || p->num_kv < 0 || p->num_heads < 0 || p->batch < 0 || p->max_q_seqlen < 0)
    return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (p->num_heads > 65535 || p->batch > 65535 || p->num_tokens > kI32 || p->num_kv > kI32 ||
      p->num_tokens * p->num_heads > kI32 || p->max_q_seqlen > kI32 - 256)
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large", op);
  if (!(p->scale > 0.f) || p->scale > 3e38f) return fail(CASCADE_ERR_INVALID, "%s: scale must be positive", op);
  if (p->flags & ~CASCADE_FLAG_DEBUG_STALL) return fail(CASCADE_ERR_INVALID, "%s: unknown flags", op);
  if (p->num_tokens == 0 || p->num_heads == 0) return CASCADE_OK;
  if (p->batch == 0 || p->max_q_seqlen == 0)
    return fail(CASCADE_ERR_INVALID, "%s: query tokens but no sequences (batch or max_q_seqlen is 0)", op);
  if (!p->query || !p->cu_q_seqlens || !p->cu_kv_seqlens || !out || !lse ||
      (p->num_kv && (!p->key || !p->key_rope || !p->value)))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  if (misaligned(p->query) || misaligned(p->key) || misaligned(p->key_rope) || misaligned(p->value) || misaligned(out))
    return fail(CASCADE_ERR_INVALID, "%s: tensors must be 16-byte aligned", op);
  // the stride of a dimension of one is never used, whatever it is
  const bool head = p->num_heads > 1, token = p->num_kv > 1;
  const int64_t key_ts = token ? p->key_token_stride : kPrefillDv, value_ts = token ? p->value_token_stride : kPrefillDv;
  const int64_t rope_ts = token ? p->rope_token_stride : kPrefillDv;
  const int64_t key_hs = head ? p->key_head_stride : 0, value_hs = head ? p->value_head_stride : 0;
  for (int64_t s : {key_ts, value_ts, rope_ts, key_hs, value_hs})
    if (s < 0 || s % 8 || s >= (int64_t(1) << 38))
      return fail(CASCADE_ERR_INVALID, "%s: strides must be non-negative multiples of 8 elements", op);
  if (!key_ts || !value_ts || !rope_ts)
    return fail(CASCADE_ERR_INVALID, "%s: token strides must be positive", op);
  LatentPrefillLaunch L = {};
  L.query = p->query;
  L.key = p->key;
  L.key_rope = p->key_rope;
  L.value = p->value;
  L.cu_q = p->cu_q_seqlens;
  L.cu_kv = p->cu_kv_seqlens;
  L.out = out;
  L.lse = lse;
  L.num_tokens = p->num_tokens;
  L.num_kv = p->num_kv;
  L.key_ts = key_ts;
  L.key_hs = key_hs;
  L.rope_ts = rope_ts;
  L.value_ts = value_ts;
  L.value_hs = value_hs;
  L.num_heads = static_cast<int32_t>(p->num_heads);
  L.batch = static_cast<int32_t>(p->batch);
  L.max_q = static_cast<int32_t>(std::min(p->max_q_seqlen, p->num_tokens));
  L.causal = p->causal != 0;
  L.scale = p->scale;
  L.debug_stall = (p->flags & CASCADE_FLAG_DEBUG_STALL) != 0;
  L.wait_limit_us = L.debug_stall ? 1000 : 0;
  return finish(op, launch_latent_prefill(L, p->dtype == CASCADE_FP16, reinterpret_cast<cudaStream_t>(stream)));
}

int cascade_page_copy(void* const* pools, int64_t num_pools, int64_t num_blocks, int64_t page_bytes,
                      const int64_t* src, const int64_t* dst, int64_t count, cascade_stream_t stream) {
  const char* op = "cascade_page_copy";
  int rc = check_pages(op, pools, num_pools, num_blocks, 1, page_bytes, 0, 0);
  if (rc) return rc;
  if (count < 0) return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (count == 0 || num_pools == 0 || page_bytes == 0) return CASCADE_OK;
  if (!src || !dst) return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  return finish(op, launch_page_copy(pools, num_pools, num_blocks, page_bytes, src, dst, count,
                                     reinterpret_cast<cudaStream_t>(stream)));
}

size_t cascade_page_fork_workspace_size(int64_t num_blocks, int64_t count) {
  return count > 0 && num_blocks >= 0 ? page_fork_workspace(num_blocks, count) : 0;
}

int cascade_page_fork(void* const* pools, int64_t num_pools, int64_t num_blocks, int64_t block_size,
                      int64_t row_bytes, const int32_t* block_table, int64_t rows, int64_t cols,
                      const int64_t* kv_lens, const int32_t* page_refs, const int64_t* parents, int64_t count,
                      int32_t* child_table, int64_t* child_lens, int32_t* refs_out, void* workspace,
                      size_t workspace_bytes, cascade_stream_t stream) {
  const char* op = "cascade_page_fork";
  int rc = check_pages(op, pools, num_pools, num_blocks, block_size, row_bytes, rows, cols);
  if (rc) return rc;
  if (count < 0) return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (count > kI32) return fail(CASCADE_ERR_UNSUPPORTED, "%s: too many children", op);
  const bool ids = num_blocks > 0, kids = count > 0;
  if ((ids && (!page_refs || !refs_out)) || (kids && (!parents || !child_lens)) || (kids && cols && !child_table) ||
      (kids && rows && (!kv_lens || (cols && !block_table))))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  if (refs_out && refs_out == page_refs)
    return fail(CASCADE_ERR_INVALID, "%s: refs_out must not be page_refs", op);
  rc = check_workspace(op, workspace, workspace_bytes, cascade_page_fork_workspace_size(num_blocks, count));
  if (rc) return rc;
  if (!ids && !kids) return CASCADE_OK;
  const PageState s = {block_table, kv_lens, page_refs, child_table, child_lens, refs_out, rows, cols, num_blocks,
                       block_size};
  return finish(op, launch_page_fork(s, pools, num_pools, row_bytes, parents, count, workspace,
                                     reinterpret_cast<cudaStream_t>(stream)));
}

int cascade_page_free(const int32_t* block_table, int64_t rows, int64_t cols, const int64_t* kv_lens,
                      const int32_t* page_refs, int64_t num_blocks, const int64_t* keep_lens, int64_t block_size,
                      int32_t* table_out, int64_t* lens_out, int32_t* refs_out, cascade_stream_t stream) {
  const char* op = "cascade_page_free";
  int rc = check_pages(op, nullptr, 0, num_blocks, block_size, 0, rows, cols);
  if (rc) return rc;
  if ((num_blocks && (!page_refs || !refs_out)) || (rows && (!kv_lens || !keep_lens || !lens_out)) ||
      (rows && cols && (!block_table || !table_out)))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  if (refs_out && refs_out == page_refs)
    return fail(CASCADE_ERR_INVALID, "%s: refs_out must not be page_refs", op);
  if (num_blocks == 0 && rows == 0) return CASCADE_OK;
  const PageState s = {block_table, kv_lens, page_refs, table_out, lens_out, refs_out, rows, cols, num_blocks,
                       block_size};
  return finish(op, launch_page_free(s, keep_lens, reinterpret_cast<cudaStream_t>(stream)));
}

size_t cascade_page_compact_workspace_size(int64_t num_blocks) {
  return num_blocks > 0 ? page_compact_workspace(num_blocks) : 0;
}

int cascade_page_compact(void* const* pools, int64_t num_pools, int64_t num_blocks, int64_t block_size,
                         int64_t row_bytes, const int32_t* block_table, int64_t rows, int64_t cols,
                         const int64_t* kv_lens, const int32_t* page_refs, int32_t* table_out, int32_t* refs_out,
                         int32_t* live_out, void* workspace, size_t workspace_bytes, cascade_stream_t stream) {
  const char* op = "cascade_page_compact";
  int rc = check_pages(op, pools, num_pools, num_blocks, block_size, row_bytes, rows, cols);
  if (rc) return rc;
  if (num_blocks == 0) return fail(CASCADE_ERR_INVALID, "%s: no pages", op);
  if (!page_refs || !refs_out || !live_out || (rows && !kv_lens) || (rows && cols && (!block_table || !table_out)))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  if (refs_out == page_refs) return fail(CASCADE_ERR_INVALID, "%s: refs_out must not be page_refs", op);
  rc = check_workspace(op, workspace, workspace_bytes, cascade_page_compact_workspace_size(num_blocks));
  if (rc) return rc;
  const PageState s = {block_table, kv_lens, page_refs, table_out, nullptr, refs_out, rows, cols, num_blocks,
                       block_size};
  return finish(op, launch_page_compact(s, pools, num_pools, row_bytes, live_out, workspace,
                                        reinterpret_cast<cudaStream_t>(stream)));
}

int cascade_verify_drafts(const int64_t* tokens, const int64_t* draft_lens, const void* draft_probs,
                          const void* target_probs, const float* uniform, const float* noise, int32_t dtype,
                          int64_t batch, int64_t max_drafts, int64_t vocab, int64_t* out_tokens, int64_t* accepted,
                          cascade_stream_t stream) {
  const char* op = "cascade_verify_drafts";
  if (!half_type(dtype) && dtype != CASCADE_FP32)
    return fail(CASCADE_ERR_INVALID, "%s: probabilities must be bf16, fp16 or fp32", op);
  if (batch < 0 || max_drafts < 0) return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (vocab < 1) return fail(CASCADE_ERR_INVALID, "%s: vocabulary must not be empty", op);
  // (the kernel's 32-bit indices step up to two rounds of 16,384 entries past the row)
  if (vocab >= kI32 / 2 || max_drafts > kI32 || batch > kI32 / 8)
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large", op);
  if (batch == 0) return CASCADE_OK;
  if (!draft_lens || !target_probs || !noise || !out_tokens || !accepted || (max_drafts && (!tokens || !uniform)))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  const uintptr_t element = dtype == CASCADE_FP32 ? 4 : 2;
  if (misaligned(target_probs, element) || misaligned(draft_probs, element) || misaligned(noise, 4) ||
      misaligned(uniform, 4) || misaligned(tokens, 8) || misaligned(draft_lens, 8))
    return fail(CASCADE_ERR_INVALID, "%s: tensors must be aligned to their elements", op);
  const VerifyLaunch L = {tokens,  draft_lens, draft_probs, target_probs, uniform, noise, out_tokens,
                          accepted, batch,      max_drafts,  vocab,        dtype};
  return finish(op, launch_verify_drafts(L, reinterpret_cast<cudaStream_t>(stream)));
}

}  // extern "C"
