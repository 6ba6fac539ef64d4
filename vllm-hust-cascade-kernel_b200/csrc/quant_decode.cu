// Attention over a 4-bit key-value cache (cascade_quant_decode): one warp per
// (query token, head), tokens one after the other, 4 values per lane, fp32.
#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

constexpr int kThreads = 256;

// the lane's 4 values of a cache row: d = 4 lane .. 4 lane + 3
__device__ __forceinline__ float4 row_values(const uint8_t* row, int lane) {
  const int d = 4 * lane;
  const uint16_t code = *reinterpret_cast<const uint16_t*>(row + 16 * (d % 32 / 8) + 4 * (d / 32) + d % 8 / 2);
  const float2 cs = __half22float2(*reinterpret_cast<const __half2*>(row + kQuantCodes + 4 * (d / 32)));
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fmaf(static_cast<float>((code >> (4 * i)) & 15) - 7.5f, cs.y, cs.x);
  return make_float4(x[0], x[1], x[2], x[3]);
}

template <bool kFp16>
__global__ void __launch_bounds__(kThreads) quant_decode_kernel(const __grid_constant__ QuantDecodeLaunch p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / 32;
  if (row >= p.num_tokens * p.num_heads) return;
  const int64_t tok = row / p.num_heads;
  const int h = static_cast<int>(row % p.num_heads) / p.group;
  int64_t b = 0, first = 0, q = p.q_len;
  if (p.q_len > 0) {
    b = tok / p.q_len, first = b * p.q_len;
  } else {
    for (; b < p.batch; ++b) {
      q = min(max(p.q_lens[b], static_cast<int64_t>(0)), p.num_tokens - first);
      if (tok < first + q) break;
      first += q;
    }
    if (b == p.batch) return;  // no request's token
  }
  const int64_t kv = min(max(p.kv_lens[b], static_cast<int64_t>(0)), static_cast<int64_t>(p.block_cols) * p.block_size);
  const int64_t n = p.causal ? max(static_cast<int64_t>(0), kv - q + (tok - first) + 1) : kv;
  const uint2 qw = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.query) + row * kHeadDim + 4 * lane);
  const uint32_t w[2] = {qw.x, qw.y};
  float x[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 f = kFp16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[i]))
                           : make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
  float m = -INFINITY, o[4] = {};
  double sum = 0.;  // (one after the other: n roundings of fp32 would show)
  bool nan = false;
  for (int64_t t = 0; t < n; ++t) {
    const int64_t page = p.block_table[b * p.block_cols + t / p.block_size];
    const bool bad = page < 0 || page >= p.num_blocks;
    if (bad && lane == 0) atomicOr(&g_cascade_device_error, kErrBadBlockId);
    const int64_t at = ((page * p.block_size + t % p.block_size) * p.kv_heads + h) * kQuantRow;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 k = bad ? zero : row_values(p.key + at, lane), v = bad ? zero : row_values(p.value + at, lane);
    float s = x[0] * k.x + x[1] * k.y + x[2] * k.z + x[3] * k.w;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.scale * 1.4426950408889634f;
    nan = nan || !(s < INFINITY);
    if (s > m) {
      const float f = ex2(m - s);
      sum *= f, m = s;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= f;
    }
    const float e = m == -INFINITY ? 0.f : ex2(s - m);
    sum += e;
    o[0] = fmaf(e, v.x, o[0]), o[1] = fmaf(e, v.y, o[1]), o[2] = fmaf(e, v.z, o[2]), o[3] = fmaf(e, v.w, o[3]);
  }
  float l = static_cast<float>(sum);
  if (nan) l = __int_as_float(0x7fffffff);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * kHeadDim + 4 * lane) =
      make_uint2(pack2<kFp16>(o[0] * inv, o[1] * inv), pack2<kFp16>(o[2] * inv, o[3] * inv));
  if (lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
}

}  // namespace

size_t quant_decode_workspace(const QuantDecodeLaunch&) { return 0; }

cudaError_t launch_quant_decode(const QuantDecodeLaunch& p, bool fp16, void*, cudaStream_t stream) {
  const int64_t rows = p.num_tokens * p.num_heads;
  (fp16 ? quant_decode_kernel<true> : quant_decode_kernel<false>)
      <<<static_cast<unsigned>((rows * 32 + kThreads - 1) / kThreads), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace cascade
