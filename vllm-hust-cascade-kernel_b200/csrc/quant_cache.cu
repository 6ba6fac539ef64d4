// Rows of a 4-bit key-value cache: quantised as they are written, and read back
// (cascade_quant_write, cascade_quant_read).
//
// A row of 128 values is four groups of 32 with a centre and a scale (fp16) and a
// 4-bit code each: value = (code - 7.5) scale + centre. 16 threads take a row, 8
// values (a 16-byte load or store of 16-bit values, one 32-bit word of codes)
// each; a group is four neighbouring threads. Both bound by HBM: 512 bytes of
// 16-bit values and 160 of cache per token and kv head.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

constexpr int kThreads = 256;
constexpr int kRowThreads = 16;  // per cache row
constexpr float kLargest = 32768.f;

template <bool kFp16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (kFp16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// slot of token t, or -1 for one that is to be passed by
__device__ __forceinline__ int64_t slot_of(const QuantRowsLaunch& p, int64_t t) {
  const int64_t s = p.slots[t];
  if (s >= p.num_slots) {
    atomicOr(&g_cascade_device_error, kErrBadBlockId);
    return -1;
  }
  return s < 0 ? -1 : s;
}

template <bool kFp16>
__global__ void __launch_bounds__(kThreads) quant_write_kernel(const QuantRowsLaunch p) {
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kRowThreads;
  const int which = blockIdx.y, j = threadIdx.x % kRowThreads;
  const bool live = row < p.num_tokens * p.kv_heads;
  const int64_t t = live ? row / p.kv_heads : 0;
  const int h = live ? static_cast<int>(row % p.kv_heads) : 0;
  const int64_t slot = live ? slot_of(p, t) : -1;
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= 0)
    v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.src[which]) + t * p.token_stride[which] +
                                        h * p.head_stride[which] + j * 8);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float x[8], lo = INFINITY, hi = -INFINITY;
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<kFp16>(w[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
    fine = fine && fabsf(x[i]) <= kLargest;
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    fine = __shfl_xor_sync(0xffffffffu, fine, d) && fine;
  }
  const __half centre = __float2half_rn(__fmul_rn(__fadd_rn(lo, hi), 0.5f));
  const __half scale = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const float c = __half2float(centre), s = __half2float(scale), by = fine && s > 0.f ? __frcp_rn(s) : 0.f;
  uint32_t code = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float u = __fadd_rn(__fmul_rn(__fsub_rn(x[i], c), by), 7.5f);
    code |= static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(fine ? u : 7.5f, 0.f), 15.f))) << (4 * i);
  }
  if (slot < 0) return;
  uint8_t* dst = p.cache[which] + (slot * p.kv_heads + h) * kQuantRow;
  reinterpret_cast<uint32_t*>(dst)[4 * (j & 3) + (j >> 2)] = code;
  if ((j & 3) == 0) {
    const uint32_t par = __half_as_ushort(centre) | static_cast<uint32_t>(__half_as_ushort(scale)) << 16;
    reinterpret_cast<uint32_t*>(dst + kQuantCodes)[j >> 2] = fine ? par : 0x7fff7fffu;
  }
}

template <int kType>
__global__ void __launch_bounds__(kThreads) quant_read_kernel(const QuantRowsLaunch p) {
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kRowThreads;
  const int which = blockIdx.y, j = threadIdx.x % kRowThreads;
  if (row >= p.num_tokens * p.kv_heads) return;
  const int64_t t = row / p.kv_heads;
  const int h = static_cast<int>(row % p.kv_heads);
  const int64_t slot = slot_of(p, t);
  uint32_t code = 0, par = 0;
  if (slot >= 0) {
    const uint8_t* src = p.cache[which] + (slot * p.kv_heads + h) * kQuantRow;
    code = reinterpret_cast<const uint32_t*>(src)[4 * (j & 3) + (j >> 2)];
    par = reinterpret_cast<const uint32_t*>(src + kQuantCodes)[j >> 2];
  }
  const float2 cs = __half22float2(*reinterpret_cast<const __half2*>(&par));
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(static_cast<float>((code >> (4 * i)) & 15u) - 7.5f, cs.y, cs.x);
  if constexpr (kType == 2) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.dst[which]) + row * kHeadDim + j * 8);
    dst[0] = make_float4(x[0], x[1], x[2], x[3]);
    dst[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dst[which]) + row * kHeadDim + j * 8) =
        make_uint4(pack2<kType == 1>(x[0], x[1]), pack2<kType == 1>(x[2], x[3]), pack2<kType == 1>(x[4], x[5]),
                   pack2<kType == 1>(x[6], x[7]));
  }
}

dim3 rows_grid(const QuantRowsLaunch& p) {
  const int64_t rows = p.num_tokens * p.kv_heads;
  return dim3(static_cast<unsigned>((rows * kRowThreads + kThreads - 1) / kThreads), 2);
}

}  // namespace

cudaError_t launch_quant_write(const QuantRowsLaunch& p, bool fp16, cudaStream_t stream) {
  (fp16 ? quant_write_kernel<true> : quant_write_kernel<false>)<<<rows_grid(p), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_quant_read(const QuantRowsLaunch& p, int dtype, cudaStream_t stream) {
  (dtype == 2 ? quant_read_kernel<2> : dtype == 1 ? quant_read_kernel<1> : quant_read_kernel<0>)
      <<<rows_grid(p), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace cascade
