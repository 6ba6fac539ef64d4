// C ABI entry points of the 4-bit key-value cache and of the log probabilities
// (include/cascade_b200.h): argument checks and launches; nothing here reads
// device memory.
#include <algorithm>

#include "capi_util.h"

namespace cascade {
namespace {

bool page_size(int64_t bs) { return bs >= 16 && bs <= 512 && (bs & (bs - 1)) == 0; }

int check_decode(const cascade_quant_attn_t* p, const char* op) {
  if (!p) return fail(CASCADE_ERR_INVALID, "%s: null argument", op);
  if (!half_type(p->dtype)) return fail(CASCADE_ERR_INVALID, "%s: query must be bf16 or fp16", op);
  if (p->head_dim != kHeadDim) return fail(CASCADE_ERR_UNSUPPORTED, "%s: head_dim must be 128", op);
  const int64_t bs = p->block_size;
  if (!page_size(bs))
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: paged blockSize must be one of 16, 32, 64, 128, 256, 512", op);
  if (p->num_tokens < 0 || p->num_heads < 0 || p->batch < 0 || p->num_blocks < 0 || p->block_cols < 0)
    return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (p->kv_heads < 1 || p->num_heads % p->kv_heads)
    return fail(CASCADE_ERR_INVALID, "%s: num_heads must be a multiple of kv_heads", op);
  if (p->q_seqlen_value < 0)
    return fail(CASCADE_ERR_INVALID, "%s: q_seqlen_value must be >= 0 (0 = per request)", op);
  // their product has to hold in 64 bits, and the kernels' steps from request to request in 32
  if (p->batch > kI32 / 2 || p->q_seqlen_value > kI32)
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large for 32-bit row indices", op);
  if (p->q_seqlen_value > 0 && p->num_tokens != p->batch * p->q_seqlen_value)
    return fail(CASCADE_ERR_INVALID, "%s: with q_seqlen_value=%lld, query.size(0) must equal batch * q_seqlen_value",
                op, static_cast<long long>(p->q_seqlen_value));
  if (p->num_heads > 65535 || p->num_tokens > kI32 || p->num_tokens * p->num_heads > kI32 / 2 ||
      p->block_cols > kI32 || p->num_blocks > kI32 || p->num_blocks * bs > kI32 - 1024 || p->block_cols * bs > kI32 / 2)
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large for 32-bit row indices", op);
  if (!(p->scale > 0.f) || p->scale > 3e38f) return fail(CASCADE_ERR_INVALID, "%s: scale must be positive", op);
  if (p->flags & ~CASCADE_FLAG_DEBUG_STALL) return fail(CASCADE_ERR_INVALID, "%s: unknown flags", op);
  return CASCADE_OK;
}

QuantDecodeLaunch decode_launch(const cascade_quant_attn_t* p, void* out, float* lse) {
  QuantDecodeLaunch L = {};
  L.query = p->query;
  L.key = static_cast<const uint8_t*>(p->key_cache);
  L.value = static_cast<const uint8_t*>(p->value_cache);
  L.block_table = p->block_table;
  L.q_lens = p->q_seqlen_value > 0 ? nullptr : p->actual_q_seqlens;
  L.kv_lens = p->actual_kv_seqlens;
  L.out = out;
  L.lse = lse;
  L.num_tokens = p->num_tokens;
  L.num_heads = static_cast<int32_t>(p->num_heads);
  L.kv_heads = static_cast<int32_t>(p->kv_heads);
  L.group = static_cast<int32_t>(p->num_heads / p->kv_heads);
  L.num_blocks = static_cast<int32_t>(p->num_blocks);
  L.block_size = static_cast<int32_t>(p->block_size);
  L.batch = static_cast<int32_t>(p->batch);
  L.block_cols = static_cast<int32_t>(p->block_cols);
  L.q_len = static_cast<int32_t>(p->q_seqlen_value);
  L.causal = p->causal != 0;
  L.scale = p->scale;
  L.debug_stall = (p->flags & CASCADE_FLAG_DEBUG_STALL) != 0;
  L.wait_limit_us = L.debug_stall ? 1000 : 0;
  return L;
}

// What write and read share.
int check_rows(const char* op, const void* key, const void* value, const void* key_cache, const void* value_cache,
               const int64_t* slots, int64_t num_tokens, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
               int64_t block_size) {
  if (head_dim != kHeadDim) return fail(CASCADE_ERR_UNSUPPORTED, "%s: head_dim must be 128", op);
  if (num_tokens < 0 || kv_heads < 0 || num_blocks < 0) return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (block_size < 1) return fail(CASCADE_ERR_INVALID, "%s: block size must be >= 1", op);
  if (num_tokens > kI32 || kv_heads > 65535 || num_tokens * kv_heads > kI32 / 2 || num_blocks > kI32 || block_size > kI32 ||
      num_blocks * block_size > (int64_t(1) << 40))
    return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large", op);
  if (num_tokens == 0 || kv_heads == 0) return CASCADE_OK;
  if (!key || !value || !slots || (num_blocks && (!key_cache || !value_cache)))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  if (misaligned(key) || misaligned(value) || misaligned(key_cache) || misaligned(value_cache))
    return fail(CASCADE_ERR_INVALID, "%s: tensors must be 16-byte aligned", op);
  return CASCADE_OK;
}

}  // namespace
}  // namespace cascade

using namespace cascade;

extern "C" {

int cascade_quant_write(const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                        int64_t value_token_stride, int64_t value_head_stride, void* key_cache, void* value_cache,
                        const int64_t* slots, int64_t num_tokens, int64_t kv_heads, int64_t head_dim,
                        int64_t num_blocks, int64_t block_size, int32_t dtype, cascade_stream_t stream) {
  const char* op = "cascade_quant_write";
  if (!half_type(dtype)) return fail(CASCADE_ERR_INVALID, "%s: key and value must be bf16 or fp16", op);
  int rc = check_rows(op, key, value, key_cache, value_cache, slots, num_tokens, kv_heads, head_dim, num_blocks, block_size);
  if (rc || num_tokens == 0 || kv_heads == 0) return rc;
  if (key_cache && key_cache == value_cache)
    return fail(CASCADE_ERR_INVALID, "%s: key_cache and value_cache must be two caches", op);
  QuantRowsLaunch L = {};
  L.src[0] = key;
  L.src[1] = value;
  // the stride of a dimension of one is never used, whatever it is
  L.token_stride[0] = num_tokens > 1 ? key_token_stride : 0;
  L.token_stride[1] = num_tokens > 1 ? value_token_stride : 0;
  L.head_stride[0] = kv_heads > 1 ? key_head_stride : 0;
  L.head_stride[1] = kv_heads > 1 ? value_head_stride : 0;
  for (int i = 0; i < 2; ++i)
    for (int64_t s : {L.token_stride[i], L.head_stride[i]})
      if (s < 0 || s % 8 || s >= (int64_t(1) << 31))
        return fail(CASCADE_ERR_INVALID, "%s: strides must be non-negative multiples of 8 elements", op);
  L.cache[0] = static_cast<uint8_t*>(key_cache);
  L.cache[1] = static_cast<uint8_t*>(value_cache);
  L.slots = slots;
  L.num_tokens = num_tokens;
  L.num_slots = num_blocks * block_size;
  L.kv_heads = static_cast<int32_t>(kv_heads);
  return finish(op, launch_quant_write(L, dtype == CASCADE_FP16, reinterpret_cast<cudaStream_t>(stream)));
}

int cascade_quant_read(const void* key_cache, const void* value_cache, const int64_t* slots, void* key, void* value,
                       int64_t num_tokens, int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                       int32_t dtype, cascade_stream_t stream) {
  const char* op = "cascade_quant_read";
  if (!half_type(dtype) && dtype != CASCADE_FP32)
    return fail(CASCADE_ERR_INVALID, "%s: key and value must be bf16, fp16 or fp32", op);
  int rc = check_rows(op, key, value, key_cache, value_cache, slots, num_tokens, kv_heads, head_dim, num_blocks, block_size);
  if (rc || num_tokens == 0 || kv_heads == 0) return rc;
  QuantRowsLaunch L = {};
  L.dst[0] = key;
  L.dst[1] = value;
  L.cache[0] = static_cast<uint8_t*>(const_cast<void*>(key_cache));
  L.cache[1] = static_cast<uint8_t*>(const_cast<void*>(value_cache));
  L.slots = slots;
  L.num_tokens = num_tokens;
  L.num_slots = num_blocks * block_size;
  L.kv_heads = static_cast<int32_t>(kv_heads);
  return finish(op, launch_quant_read(L, dtype, reinterpret_cast<cudaStream_t>(stream)));
}

size_t cascade_quant_decode_workspace_size(const cascade_quant_attn_t* p) {
  if (check_decode(p, "cascade_quant_decode") != CASCADE_OK) return 0;
  if (p->num_tokens == 0 || p->num_heads == 0 || p->batch == 0) return 0;
  return quant_decode_workspace(decode_launch(p, nullptr, nullptr));
}

int cascade_quant_decode(const cascade_quant_attn_t* p, void* out, float* lse, void* workspace, size_t workspace_bytes,
                         cascade_stream_t stream) {
  const char* op = "cascade_quant_decode";
  int rc = check_decode(p, op);
  if (rc) return rc;
  if (p->num_tokens == 0 || p->num_heads == 0) return CASCADE_OK;
  if (p->batch == 0) return fail(CASCADE_ERR_INVALID, "%s: query tokens but no requests", op);
  if (!p->query || !p->actual_kv_seqlens || !out || !lse || (p->block_cols && !p->block_table) ||
      (p->num_blocks && (!p->key_cache || !p->value_cache)) || (p->q_seqlen_value == 0 && !p->actual_q_seqlens))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  if (misaligned(p->query) || misaligned(p->key_cache) || misaligned(p->value_cache) || misaligned(out))
    return fail(CASCADE_ERR_INVALID, "%s: query/caches/out must be 16-byte aligned", op);
  const QuantDecodeLaunch L = decode_launch(p, out, lse);
  rc = check_workspace(op, workspace, workspace_bytes, quant_decode_workspace(L));
  if (rc) return rc;
  return finish(op, launch_quant_decode(L, p->dtype == CASCADE_FP16, workspace,
                                        reinterpret_cast<cudaStream_t>(stream)));
}

int cascade_token_logprobs(const void* logits, int64_t row_stride, const int64_t* tokens, int32_t dtype, int64_t rows,
                           int64_t vocab, int64_t top, float* logprob, float* entropy, int64_t* rank,
                           float* top_logprobs, int64_t* top_tokens, cascade_stream_t stream) {
  const char* op = "cascade_token_logprobs";
  if (!half_type(dtype) && dtype != CASCADE_FP32)
    return fail(CASCADE_ERR_INVALID, "%s: logits must be bf16, fp16 or fp32", op);
  if (rows < 0 || top < 0) return fail(CASCADE_ERR_INVALID, "%s: negative size", op);
  if (vocab < 1) return fail(CASCADE_ERR_INVALID, "%s: vocabulary must not be empty", op);
  if (top > kMaxTop || top > vocab)
    return fail(CASCADE_ERR_INVALID, "%s: top must be at most 32 and at most the vocabulary", op);
  if (vocab >= kI32 / 2 || rows > kI32 / 32) return fail(CASCADE_ERR_UNSUPPORTED, "%s: problem too large", op);
  if (rows == 0) return CASCADE_OK;
  if (rows > 1 && (row_stride < vocab || row_stride >= (int64_t(1) << 40)))
    return fail(CASCADE_ERR_INVALID, "%s: the row stride must hold a row", op);
  if (!logits || !tokens || !logprob || !entropy || !rank || (top && (!top_logprobs || !top_tokens)))
    return fail(CASCADE_ERR_INVALID, "%s: null device pointer", op);
  if (misaligned(logits, dtype == CASCADE_FP32 ? 4 : 2) || misaligned(tokens, 8) || misaligned(rank, 8) ||
      misaligned(top_tokens, 8) || misaligned(logprob, 4) || misaligned(entropy, 4) || misaligned(top_logprobs, 4))
    return fail(CASCADE_ERR_INVALID, "%s: tensors must be aligned to their elements", op);
  const LogprobsLaunch L = {logits,       tokens,     logprob, entropy, rank,
                            top_logprobs, top_tokens, rows,    vocab,   rows > 1 ? row_stride : vocab,
                            static_cast<int32_t>(top), dtype};
  return finish(op, launch_token_logprobs(L, reinterpret_cast<cudaStream_t>(stream)));
}

}  // extern "C"
