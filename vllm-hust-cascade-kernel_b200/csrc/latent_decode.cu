// Latent attention, absorbed form (cascade_latent_decode).
//
// For a query row x (576 values) of a request: s_t = scale <x, c_t> over the
// request's cache rows c_t, out = sum_t softmax(s)_t c_t[0:512] with the
// running maximum m and sum l of exp(s - m) in fp32. One warp per query row:
// the lanes hold 18 query and 16 output values each, a dot product is one
// warp reduction per cache row.
#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

constexpr int kWarps = 4;

template <bool kFp16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (kFp16) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  } else {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  }
}

// Request and query token of flat token `tok`; returns false past the last.
__device__ bool find_request(const LatentDecodeLaunch& p, int64_t tok, int* b, int64_t* i, int64_t* q_len) {
  if (p.q_len > 0) {
    *b = static_cast<int>(tok / p.q_len);
    *i = tok % p.q_len;
    *q_len = p.q_len;
    return *b < p.batch;
  }
  for (int r = 0; r < p.batch; ++r) {
    const int64_t n = max(p.q_lens[r], static_cast<int64_t>(0));
    if (tok < n) {
      *b = r;
      *i = tok;
      *q_len = n;
      return true;
    }
    tok -= n;
  }
  return false;
}

template <bool kFp16>
__global__ void __launch_bounds__(kWarps * 32) latent_decode_kernel(const LatentDecodeLaunch p) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= p.num_tokens * p.num_heads) return;
  int b = 0;
  int64_t i = 0, q_len = 0, n = 0;
  if (find_request(p, row / p.num_heads, &b, &i, &q_len)) {
    n = min(p.kv_lens[b], static_cast<int64_t>(p.block_cols) * p.block_size);
    if (p.causal) n = min(n, p.kv_lens[b] - q_len + i + 1);
  }
  // pairs of values: lane holds pairs lane + 32 j, j < 9 (the last 32 pairs are the rotary part)
  const uint32_t* q = static_cast<const uint32_t*>(p.query) + row * (kLatentRow / 2);
  float2 x[9], o[8];
#pragma unroll
  for (int j = 0; j < 9; ++j) x[j] = unpack2<kFp16>(q[lane + 32 * j]);
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = make_float2(0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  const int32_t* bt = p.block_table + static_cast<int64_t>(b) * p.block_cols;
  for (int64_t t = 0; t < n; ++t) {
    const int32_t id = bt[t / p.block_size];
    const bool ok = static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks);
    if (!ok && lane == 0) atomicOr(&g_cascade_device_error, kErrBadBlockId);
    const uint32_t* c = static_cast<const uint32_t*>(p.cache) +
                        (static_cast<int64_t>(ok ? id : 0) * p.block_size + t % p.block_size) * (kLatentRow / 2);
    float2 v[9];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 9; ++j) {
      v[j] = unpack2<kFp16>(ok ? c[lane + 32 * j] : 0u);
      s = fmaf(x[j].x, v[j].x, fmaf(x[j].y, v[j].y, s));
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    s *= p.scale;
    const float m_new = fmaxf(m, s);
    const float dm = m == m_new ? 1.f : expf(m - m_new);
    const float e = m_new == -INFINITY ? 0.f : expf(s - m_new);
    l = l * dm + e;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      o[j].x = fmaf(e, v[j].x, o[j].x * dm);
      o[j].y = fmaf(e, v[j].y, o[j].y * dm);
    }
    m = m_new;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint32_t* out = static_cast<uint32_t*>(p.out) + row * (kLatentDim / 2);
#pragma unroll
  for (int j = 0; j < 8; ++j) out[lane + 32 * j] = pack2<kFp16>(o[j].x * inv, o[j].y * inv);
  if (lane == 0) p.lse[row] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace

size_t latent_decode_workspace(const LatentDecodeLaunch&) { return 0; }

cudaError_t launch_latent_decode(const LatentDecodeLaunch& p, bool fp16, void*, cudaStream_t stream) {
  const int64_t rows = p.num_tokens * p.num_heads;
  auto kern = fp16 ? latent_decode_kernel<true> : latent_decode_kernel<false>;
  kern<<<static_cast<unsigned>((rows + kWarps - 1) / kWarps), kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace cascade
