// Latent attention, expanded form (cascade_latent_prefill).
//
// For a query row of head h: s_t = scale (<q[0:128], k_th> + <q[128:192], r_t>)
// over the sequence's keys it may see, out = sum_t softmax(s)_t v_th with the
// running maximum and sum in fp32. One warp per query row.
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

template <bool kFp16>
__global__ void __launch_bounds__(kWarps * 32) latent_prefill_kernel(const LatentPrefillLaunch p) {
  const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t q0 = p.cu_q[b], k0 = p.cu_kv[b];
  const int64_t n = p.cu_q[b + 1] - q0, m_kv = p.cu_kv[b + 1] - k0;
  if (i >= n || q0 < 0 || q0 + n > p.num_tokens || k0 < 0 || k0 + m_kv > p.num_kv) return;
  const int64_t row = (q0 + i) * p.num_heads + h;
  const int64_t last = p.causal ? min(m_kv, m_kv - n + i + 1) : m_kv;
  auto pair = [](const void* base, int64_t element) { return static_cast<const uint32_t*>(base) + element / 2; };
  const uint32_t* q = pair(p.query, row * kPrefillDk);
  const float2 x0 = unpack2<kFp16>(q[lane]), x1 = unpack2<kFp16>(q[lane + 32]), x2 = unpack2<kFp16>(q[lane + 64]);
  float2 o0 = make_float2(0.f, 0.f), o1 = o0;
  float m = -INFINITY, l = 0.f;
  for (int64_t t = 0; t < last; ++t) {
    const uint32_t* k = pair(p.key, (k0 + t) * p.key_ts + h * p.key_hs);
    const uint32_t* r = pair(p.key_rope, (k0 + t) * p.rope_ts);
    const uint32_t* v = pair(p.value, (k0 + t) * p.value_ts + h * p.value_hs);
    const float2 a = unpack2<kFp16>(k[lane]), c = unpack2<kFp16>(k[lane + 32]), d = unpack2<kFp16>(r[lane]);
    float s = x0.x * a.x + x0.y * a.y + x1.x * c.x + x1.y * c.y + x2.x * d.x + x2.y * d.y;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= p.scale;
    const float m_new = fmaxf(m, s);
    const float dm = m == m_new ? 1.f : expf(m - m_new);
    const float e = m_new == -INFINITY ? 0.f : expf(s - m_new);
    const float2 v0 = unpack2<kFp16>(v[lane]), v1 = unpack2<kFp16>(v[lane + 32]);
    l = l * dm + e;
    o0 = make_float2(fmaf(e, v0.x, o0.x * dm), fmaf(e, v0.y, o0.y * dm));
    o1 = make_float2(fmaf(e, v1.x, o1.x * dm), fmaf(e, v1.y, o1.y * dm));
    m = m_new;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint32_t* out = static_cast<uint32_t*>(p.out) + row * (kPrefillDv / 2);
  out[lane] = pack2<kFp16>(o0.x * inv, o0.y * inv);
  out[lane + 32] = pack2<kFp16>(o1.x * inv, o1.y * inv);
  if (lane == 0) p.lse[row] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace

cudaError_t launch_latent_prefill(const LatentPrefillLaunch& p, bool fp16, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.max_q + kWarps - 1) / kWarps), p.num_heads, p.batch);
  auto kern = fp16 ? latent_prefill_kernel<true> : latent_prefill_kernel<false>;
  kern<<<grid, kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace cascade
