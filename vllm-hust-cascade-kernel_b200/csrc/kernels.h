// Internal launch interface between the C ABI (capi.cu) and the kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace cascade {

constexpr int kHeadDim = 128;
constexpr int kNumSMs = 148;

// Stage-1 overlapped with a cascade step's suffix decode (PagedAttnLaunch::
// ov_seg): segment A runs on kOvCtas SMs beside the decode, sized so that its
// runs last about as long as the decode: the suffix's kv bytes at
// kOvDecodeBytesPerNs (the decode's HBM rate on the SMs segment A leaves it:
// the C4 decode took 221 instead of 206 us with 48 SMs held, 254 with 64)
// over kOvTileNs per 128-token KV tile of a two-tile stage-1 CTA (C4: 55
// tiles in ~175 us). Within 40% of that estimate, the segment A whose
// segment-B runs are a whole fraction of a stream (tc >> k tiles, TA = T -
// runs_b * (tc >> k)) is taken instead: no segment-B run then straddles two
// (request, kv head) streams and every segment-B CTA does one piece (C4:
// 343 us at TA = 1,728 tiles, 32-tile runs, against 345-361 us for segments
// whose runs straddle streams). No segment A below kOvMinRunTiles tiles per
// run (16: the 2-rank shard of C4, 4 kv heads, gets a segment A of 864 tiles,
// 203 instead of 206 us serial; with 32 it had none); at most 3/5 of the
// tiles.
constexpr int kOvCtas = 64;
constexpr int64_t kOvMinRunTiles = 16;
constexpr double kOvDecodeBytesPerNs = 6000.0;  // 6 TB/s
constexpr double kOvTileNs = 3300.0;
__host__ __device__ inline int64_t overlap_tiles(int64_t suffix_tokens, int64_t kv_heads, int64_t runs_a,
                                                 int64_t runs_b, int64_t T, int64_t tc) {
  const double t_dec = static_cast<double>(suffix_tokens) * static_cast<double>(kv_heads) * 512.0 /
                       kOvDecodeBytesPerNs;
  int64_t per_run = static_cast<int64_t>(t_dec / kOvTileNs);
  const int64_t cap = (3 * T) / 5 / runs_a;
  if (per_run > cap) per_run = cap;
  if (per_run < kOvMinRunTiles) return 0;
  const int64_t est = per_run * runs_a;
  int64_t best = -1;
  for (int k = 0; k < 4; ++k) {
    const int64_t lb = tc >> k;
    if (lb < 8 || (lb << k) != tc) break;
    const int64_t ta = T - runs_b * lb;
    if (ta < kOvMinRunTiles * runs_a || ta > (3 * T) / 5 || 5 * (ta > est ? ta - est : est - ta) > 2 * est) continue;
    if (best < 0 || (ta > est ? ta - est : est - ta) < (best > est ? best - est : est - best)) best = ta;
  }
  return best >= 0 ? best : est;
}

// ----------------------------------------------------------------------------
// paged attention (decode path: <= 16 query rows per (request, kv head))
// ----------------------------------------------------------------------------
struct PagedAttnLaunch {
  CUtensorMap tmap_k;  // 2-D view [num_blocks*block_size, kv_heads*128], box {64, box_rows}, SW128
  CUtensorMap tmap_v;
  const void* query;
  const int32_t* block_table;
  const int64_t* q_seqlens;
  const int64_t* kv_seqlens;
  void* out;            // final output (nsplit == 1) in out_dtype
  float* lse;           // final lse (nsplit == 1), row stride lse_stride
  float* part_o;        // [nsplit][T*H][128] fp32 (nsplit > 1)
  float* part_lse;      // [nsplit][T*H]
  int32_t num_tokens, num_heads, kv_heads, group;
  int32_t batch, block_cols, block_size, num_blocks;
  int32_t q_seqlen_value;  // > 0 uniform, 0 = per-request (prefix-summed in kernel)
  int32_t max_q_seqlen;
  int32_t split_tokens, num_splits;
  // two-tile stage-1 over equal runs of KV tiles (0 = the split grid): the
  // grid has piece_ctas CTAs; (request, kv head, row-tile pair) units of
  // piece_unit_tiles 128-token tiles are concatenated and cut into piece_ctas
  // equal runs, each CTA taking one run (one or two pieces of units); a
  // piece's partial goes to plane "its index among the unit's pieces"
  int32_t piece_ctas, piece_unit_tiles;
  // Equal runs in two segments around a cascade step's suffix decode
  // (ov_seg 0: one segment of piece_ctas / pairs runs). The first TA tiles
  // are cut into ov_runs_a runs (segment A, launched before the decode on few
  // SMs: ov_seg 1), the rest into ov_runs_b runs (segment B, launched after
  // it: ov_seg 2). Every CTA of both launches computes the same TA from the
  // suffix's kv lengths (ov_lens, ov_nlens requests).
  int32_t ov_seg, ov_runs_a, ov_runs_b, ov_nlens;
  const int64_t* ov_lens;
  int32_t out_dtype;    // 0 bf16, 1 fp16, 2 fp32
  int32_t lse_stride;   // 8 (reference padded rows) or 1 (compact)
  int32_t partial_out;  // 1: always write split partials (a later combine produces the output)
  int32_t pdl;          // launched as a programmatic dependent of the previous kernel in the stream:
                        // 1 = every CTA waits for it before exiting, 2 = only the grid's last CTA does
  int32_t debug_stall;  // 1 (test hook): the consumers first wait on a barrier nothing completes
  uint32_t wait_limit_us;  // limit of one mbarrier wait (0 = the default, kWaitLimitNs)

  float scale_log2;     // softmax scale * log2(e)
  // planned decode (kernel 2): workspace arrays after the partials, or null
  int32_t* plan_items;     // [batch * num_splits] (request << 8) | split of the non-empty items
  int32_t* plan_count;     // number of items
  int32_t* plan_counters;  // [kv_heads] next item per kv head
};

cudaError_t launch_paged_decode(const PagedAttnLaunch& p, bool fp16, cudaStream_t stream);

// Launch `kern` with the programmatic-dependent attribute when `pdl` is set.
template <typename Arg>
cudaError_t launch_maybe_pdl(void (*kern)(Arg), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl,
                             const Arg& arg) {
  if (!pdl) {
    kern<<<grid, block, smem, stream>>>(arg);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, arg);
}


// Stage-1 tensor-core path (tcgen05, > 16 rows per (request, kv head)).
cudaError_t launch_paged_prefix_tc(const PagedAttnLaunch& p, bool fp16, cudaStream_t stream);

// Merge the nsplit partials of every (token, head) row into the final output.
cudaError_t launch_split_combine(const PagedAttnLaunch& p, cudaStream_t stream);

// One combine for a whole cascade step: merges the split partials of stage-1
// and of the suffix for every (token, head) row and writes the final output.
struct CascadeCombineLaunch {
  const float* o1;      // [n1][rows][128]
  const float* l1;      // [n1][rows]
  const float* o2;      // [n2][rows][128]
  const float* l2;      // [n2][rows]
  int32_t n1, n2;
  int64_t rows;
  void* out;            // [rows][128] in out_dtype
  int32_t out_dtype;    // 0 bf16, 1 fp16, 2 fp32
  float* lse_out;       // [rows] or null
  int32_t pdl;          // 1: launched as a programmatic dependent (waits for its primary first)
};

cudaError_t launch_cascade_combine(const CascadeCombineLaunch& p, cudaStream_t stream);

// ----------------------------------------------------------------------------
// LSE merge
// ----------------------------------------------------------------------------
struct LseMergeLaunch {
  const void* o1;
  const void* o2;
  const float* lse1;
  const float* lse2;
  void* out;
  int64_t rows;
  int32_t dim;
  int32_t stride1, stride2;
  int32_t o1_dtype, o2_dtype, out_dtype;  // 0 bf16, 1 fp16, 2 fp32
};

cudaError_t launch_lse_merge(const LseMergeLaunch& p, cudaStream_t stream);

// ----------------------------------------------------------------------------
// gate_up GEMM + epilogue
// ----------------------------------------------------------------------------
struct GateUpLaunch {
  void* ws;            // [M, 2I] bf16 (modes that write C)
  void* d;             // [M, I] bf16
  int64_t d_stride;
  int32_t M, K, I;
  int32_t mode;
};

cudaError_t launch_gateup(const GateUpLaunch& p, const void* a, const void* b, cudaStream_t stream);
// Modes 3/5/7/8: epilogue window traffic on an existing workspace (no GEMM).
cudaError_t launch_gateup_window(const void* ws, void* d, int64_t d_stride, int32_t M, int32_t I, int32_t mode,
                                 cudaStream_t stream);

// ----------------------------------------------------------------------------
// Residual add + RMSNorm statistics
// ----------------------------------------------------------------------------
struct RmsNormLaunch {
  const void* x1;      // [M, K] 16-bit
  const void* x2;      // [M, K] (modes 0 and 2)
  const void* gamma;   // [K] (mode 1)
  const void* beta;    // [K] or nullptr (mode 1)
  void* x_out;         // [M, K] (mode 0)
  float* rstd;         // [m_padded] (rows >= M zeroed)
  void* y;             // [M, K] (mode 1)
  int32_t M, K, m_padded, mode;
  float eps;
};

cudaError_t launch_add_rms_norm_stats(const RmsNormLaunch& p, bool fp16, cudaStream_t stream);

// ----------------------------------------------------------------------------
// Latent attention
// ----------------------------------------------------------------------------
constexpr int kLatentDim = 512;               // latent values of a cache row
constexpr int kLatentRow = kLatentDim + 64;   // with the rotary key values
constexpr int kPrefillDk = 192;               // expanded key: 128 per head + 64 shared
constexpr int kPrefillDv = 128;

struct LatentDecodeLaunch {
  const void* query;
  const void* cache;
  const int32_t* block_table;
  const int64_t* q_lens;   // null when q_len > 0
  const int64_t* kv_lens;
  void* out;               // [num_tokens, num_heads, 512]
  float* lse;              // [num_tokens * num_heads]
  int64_t num_tokens;
  int32_t num_heads, num_blocks, block_size, batch, block_cols;
  int32_t q_len;           // 0 = per request
  int32_t causal;
  float scale;
  uint32_t wait_limit_us;
  int32_t debug_stall;
};
cudaError_t launch_latent_decode(const LatentDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream);
size_t latent_decode_workspace(const LatentDecodeLaunch& p);
cudaError_t launch_latent_decode_pair(const LatentDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream);
size_t latent_decode_pair_workspace(const LatentDecodeLaunch& p);

struct LatentPrefillLaunch {
  const void* query;
  const void* key;
  const void* key_rope;
  const void* value;
  const int64_t* cu_q;
  const int64_t* cu_kv;
  void* out;
  float* lse;
  int64_t num_tokens, num_kv;
  int64_t key_ts, key_hs, rope_ts, value_ts, value_hs;  // strides in elements
  int32_t num_heads, batch, max_q;
  int32_t causal;
  float scale;
  uint32_t wait_limit_us;
  int32_t debug_stall;
};
cudaError_t launch_latent_prefill(const LatentPrefillLaunch& p, bool fp16, cudaStream_t stream);

// ----------------------------------------------------------------------------
// Pages of a cache
// ----------------------------------------------------------------------------
constexpr int kMaxPoolsPerLaunch = 128;  // pool pointers that travel as kernel arguments

struct PageState {
  const int32_t* table;
  const int64_t* kv_lens;
  const int32_t* refs;
  int32_t* table_out;
  int64_t* lens_out;
  int32_t* refs_out;
  int64_t rows, cols, num_blocks, block_size;
};
cudaError_t launch_page_copy(void* const* pools, int64_t num_pools, int64_t num_blocks, int64_t page_bytes,
                             const int64_t* src, const int64_t* dst, int64_t count, cudaStream_t stream);
size_t page_fork_workspace(int64_t num_blocks, int64_t count);
cudaError_t launch_page_fork(const PageState& s, void* const* pools, int64_t num_pools, int64_t row_bytes,
                             const int64_t* parents, int64_t count, void* workspace, cudaStream_t stream);
cudaError_t launch_page_free(const PageState& s, const int64_t* keep_lens, cudaStream_t stream);
size_t page_compact_workspace(int64_t num_blocks);
cudaError_t launch_page_compact(const PageState& s, void* const* pools, int64_t num_pools, int64_t row_bytes,
                                int32_t* live_out, void* workspace, cudaStream_t stream);

// ----------------------------------------------------------------------------
// Verification of drafted tokens
// ----------------------------------------------------------------------------
struct VerifyLaunch {
  const int64_t* tokens;
  const int64_t* draft_lens;
  const void* draft;   // [B, K, V] or null
  const void* target;  // [B, K + 1, V]
  const float* uniform;
  const float* noise;
  int64_t* out_tokens;
  int64_t* accepted;
  int64_t batch, drafts, vocab;
  int32_t dtype;       // 0 bf16, 1 fp16, 2 fp32
};
cudaError_t launch_verify_drafts(const VerifyLaunch& p, cudaStream_t stream);

// ----------------------------------------------------------------------------
// A key-value cache held in 4 bits
// ----------------------------------------------------------------------------
constexpr int kQuantRow = 80;    // bytes of a cache row: 64 of codes, then four groups' (centre, scale) in fp16
constexpr int kQuantCodes = 64;

struct QuantRowsLaunch {
  const void* src[2];    // keys, values (write)
  void* dst[2];          // keys, values (read)
  int64_t token_stride[2], head_stride[2];  // of src, in elements
  uint8_t* cache[2];
  const int64_t* slots;
  int64_t num_tokens, num_slots;
  int32_t kv_heads;
};
cudaError_t launch_quant_write(const QuantRowsLaunch& p, bool fp16, cudaStream_t stream);
cudaError_t launch_quant_read(const QuantRowsLaunch& p, int dtype, cudaStream_t stream);

struct QuantDecodeLaunch {
  const void* query;
  const uint8_t* key;
  const uint8_t* value;
  const int32_t* block_table;
  const int64_t* q_lens;   // null when q_len > 0
  const int64_t* kv_lens;
  void* out;               // [num_tokens, num_heads, 128]
  float* lse;              // [num_tokens * num_heads]
  int64_t num_tokens;
  int32_t num_heads, kv_heads, group, num_blocks, block_size, batch, block_cols;
  int32_t q_len;           // 0 = per request
  int32_t causal;
  float scale;
  uint32_t wait_limit_us;
  int32_t debug_stall;
};
cudaError_t launch_quant_decode(const QuantDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream);
size_t quant_decode_workspace(const QuantDecodeLaunch& p);
// The same on the tensor cores' 128-row tiles, for many query rows per request.
cudaError_t launch_quant_tiles(const QuantDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream);
size_t quant_tiles_workspace(const QuantDecodeLaunch& p);

// ----------------------------------------------------------------------------
// Log probabilities of tokens
// ----------------------------------------------------------------------------
constexpr int kMaxTop = 32;

struct LogprobsLaunch {
  const void* logits;
  const int64_t* tokens;
  float* logprob;
  float* entropy;
  int64_t* rank;
  float* top_logprobs;
  int64_t* top_tokens;
  int64_t rows, vocab, row_stride;
  int32_t top;
  int32_t dtype;           // 0 bf16, 1 fp16, 2 fp32
};
cudaError_t launch_token_logprobs(const LogprobsLaunch& p, cudaStream_t stream);

// Host: raise a kernel's dynamic shared memory limit once per (kernel,
// device) instead of on every launch.
cudaError_t ensure_smem_limit(const void* kernel, int bytes);

// Host: record `msg` as this thread's cascade_last_error() text; returns `code`.
int set_error(int code, const char* msg);

// Host: encode a 2-D bf16/fp16 tiled tensor map (SW128 when inner box is 64).
bool encode_tmap_2d(CUtensorMap* map, const void* base, uint64_t inner, uint64_t rows, uint64_t row_stride_bytes,
                    uint32_t box_inner, uint32_t box_rows, bool swizzle128, CUtensorMapL2promotion promo);

// Host: encode a 3-D tiled tensor map of bytes, no swizzle, innermost extent first;
// the inner extent of tensor and box (up to 1,024), strides and base address are
// multiples of 16.
bool encode_tmap_bytes(CUtensorMap* map, const void* base, const uint64_t (&extent)[3], const uint64_t (&stride_bytes)[2],
                       const uint32_t (&box)[3]);

// Host: encode a tiled tensor map of 16-bit elements, 128-byte swizzle (box[0]
// = 64 elements), rank 2 to 5, innermost extent first; strides of the outer
// rank - 1 dimensions.
bool encode_tmap_nd(CUtensorMap* map, const void* base, int rank, const uint64_t* extent, const uint64_t* stride_bytes,
                    const uint32_t* box);

}  // namespace cascade
