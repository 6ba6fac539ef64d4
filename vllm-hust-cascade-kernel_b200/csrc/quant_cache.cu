// Rows of a 4-bit key-value cache: quantised as they are written, and read back
// (cascade_quant_write, cascade_quant_read).
//
// A row of 128 values is four groups of 32 with a centre and a scale (fp16) and a
// 4-bit code each: value = (code - 7.5) scale + centre. 16 threads take a row, 8
// values (a 16-byte load or store of 16-bit values, one 32-bit word of codes)
// each; a group is four neighbouring threads. Bound by HBM (512 bytes of
// 16-bit values and 160 of cache per token and kv head) and, the write, by its
// instructions, some 135 for eight values. A thread takes the key and
// the value of kUnroll rows at once: its chain slot -> row -> store is two
// latencies long. 60,001 tokens x 4 kv heads: written in 38 us (4.2 TB/s), read back
// in 29.7 us (5.4 TB/s; the same with four rows at once, 32.7 with eight).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

constexpr int kThreads = 256;
constexpr int kRowThreads = 16;  // per cache row
constexpr int kStep = kThreads / kRowThreads;  // rows of a CTA at once
constexpr int kUnroll = 2;
constexpr float kLargest = 32768.f;

template <bool kFp16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (kFp16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// packed 16-bit maximum (NaN if either is) and minimum
template <bool kFp16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (kFp16)
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Where this thread's rows are: output row, and cache row (-1: to be passed by).
struct Place {
  uint32_t row, token, head;
  int64_t at;
  bool live;
};
__device__ __forceinline__ void places(const QuantRowsLaunch& p, Place (&x)[kUnroll]) {
  const uint32_t rows = static_cast<uint32_t>(p.num_tokens) * p.kv_heads;
  int64_t slot[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    x[i].row = blockIdx.x * (kStep * kUnroll) + i * kStep + threadIdx.x / kRowThreads;
    x[i].live = x[i].row < rows;
    x[i].token = x[i].live ? x[i].row / static_cast<uint32_t>(p.kv_heads) : 0;
    x[i].head = x[i].live ? x[i].row - x[i].token * p.kv_heads : 0;
    slot[i] = x[i].live ? __ldg(p.slots + x[i].token) : -1;
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if (slot[i] >= p.num_slots) {
      atomicOr(&g_cascade_device_error, kErrBadBlockId);
      slot[i] = -1;
    }
    x[i].at = slot[i] < 0 ? -1 : slot[i] * p.kv_heads + x[i].head;
  }
}

// x / 15 rounded to nearest: the quotient by the rounded reciprocal, corrected by its remainder (Markstein 1990: the
// result is correctly rounded). For x below 2^-100 it need not be: the scale is 0.
__device__ __forceinline__ float fifteenth(float x) {
  const float by = 1.f / 15.f, q = __fmul_rn(x, by);
  return __fmaf_rn(__fmaf_rn(-15.f, q, x), by, q);
}
// 1 / s, to nearest where a code depends on it (tested with every positive fp16 scale, values next to the codes' borders): one
// Newton step.
__device__ __forceinline__ float reciprocal(float s) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
  return __fmaf_rn(__fmaf_rn(-s, y, 1.f), y, y);
}

// A group's 32 values (8 in each of four threads) as this thread's word of codes and the group's centre and scale.
template <bool kFp16>
__device__ __forceinline__ uint2 quantise(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  // the largest of the values and of their negatives, side by side
  uint32_t hi = max2<kFp16>(max2<kFp16>(w[0], w[1]), max2<kFp16>(w[2], w[3]));
  uint32_t lo = max2<kFp16>(max2<kFp16>(w[0] ^ 0x80008000u, w[1] ^ 0x80008000u), max2<kFp16>(w[2] ^ 0x80008000u, w[3] ^ 0x80008000u));
  uint32_t m = max2<kFp16>(__byte_perm(hi, lo, 0x5410), __byte_perm(hi, lo, 0x7632));
  m = max2<kFp16>(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max2<kFp16>(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const float2 f = unpack2<kFp16>(m);  // highest, -lowest
  const bool fine = f.x <= kLargest && f.y <= kLargest;  // (a NaN is not)
  const __half centre = __float2half_rn(__fmul_rn(__fsub_rn(f.x, f.y), 0.5f));
  const __half scale = __float2half_rn(fifteenth(__fadd_rn(f.x, f.y)));
  const float c = __half2float(centre), s = __half2float(scale), by = fine && s > 0.f ? reciprocal(s) : 0.f;
  // u = (x - c) / s + 7.5, rounded to a whole number (half to even) in the low bits by adding 1.5 * 2^23. It is within +-64 (a
  // spread of values is no less than a step of theirs, and the centre's rounding no more), so two fit a pair of 16 bits, and
  // are cut to 0..15 there.
  uint32_t n[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = unpack2<kFp16>(w[i]);
    float u0 = x.x, u1 = x.y;
    fadd2(u0, u1, -c, -c);
    u0 = __fmul_rn(u0, by), u1 = __fmul_rn(u1, by);  // (a packed product is fused with the sum after it)
    fadd2(u0, u1, 7.5f, 7.5f);
    fadd2(u0, u1, 12582912.f, 12582912.f);
    asm("min.relu.s16x2 %0, %1, %2;" : "=r"(n[i]) : "r"(__byte_perm(__float_as_uint(u0), __float_as_uint(u1), 0x5410)), "r"(0x000f000fu));
  }
  const uint32_t lo4 = n[0] + n[1] * 256u, hi4 = n[2] + n[3] * 256u;  // bytes: first of two pairs, second of two pairs
  const uint32_t code = __byte_perm(lo4 + (lo4 >> 12), hi4 + (hi4 >> 12), 0x5410);
  const uint32_t par = __half_as_ushort(centre) | static_cast<uint32_t>(__half_as_ushort(scale)) << 16;
  return fine ? make_uint2(code, par) : make_uint2(0x88888888u, 0x7fff7fffu);
}

template <bool kFp16>
__global__ void __launch_bounds__(kThreads) quant_write_kernel(const QuantRowsLaunch p) {
  const int j = threadIdx.x % kRowThreads;
  Place x[kUnroll];
  uint4 v[kUnroll][2];
  places(p, x);
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v[i][k] = make_uint4(0u, 0u, 0u, 0u);
      if (x[i].at >= 0)
        v[i][k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.src[k]) + x[i].token * p.token_stride[k] +
                                                       x[i].head * p.head_stride[k] + j * 8));
    }
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint2 q = quantise<kFp16>(v[i][k]);
      if (x[i].at < 0) continue;
      uint32_t* dst = reinterpret_cast<uint32_t*>(p.cache[k] + x[i].at * kQuantRow);
      dst[4 * (j & 3) + (j >> 2)] = q.x;
      if ((j & 3) == 0) dst[kQuantCodes / 4 + (j >> 2)] = q.y;
    }
  }
}

template <int kType>
__global__ void __launch_bounds__(kThreads) quant_read_kernel(const QuantRowsLaunch p) {
  const int j = threadIdx.x % kRowThreads;
  Place x[kUnroll];
  uint32_t code[kUnroll][2], par[kUnroll][2];
  places(p, x);
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      code[i][k] = par[i][k] = 0;
      if (x[i].at >= 0) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.cache[k] + x[i].at * kQuantRow);
        code[i][k] = __ldg(src + 4 * (j & 3) + (j >> 2));
        par[i][k] = __ldg(src + kQuantCodes / 4 + (j >> 2));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if (!x[i].live) continue;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float2 cs = __half22float2(*reinterpret_cast<const __half2*>(&par[i][k]));
      // a nibble at the bits 16..19 of 2^7 (the float's bits 0x43000000) is 128 + code
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t n = (e < 4 ? code[i][k] << (16 - 4 * e) : code[i][k] >> (4 * e - 16)) & 0xf0000u;
        y[e] = fmaf(__uint_as_float(0x43000000u | n) - 135.5f, cs.y, cs.x);
      }
      const int64_t at = static_cast<int64_t>(x[i].row) * kHeadDim + j * 8;
      if constexpr (kType == 2) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.dst[k]) + at);
        dst[0] = make_float4(y[0], y[1], y[2], y[3]);
        dst[1] = make_float4(y[4], y[5], y[6], y[7]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dst[k]) + at) =
            make_uint4(pack2<kType == 1>(y[0], y[1]), pack2<kType == 1>(y[2], y[3]), pack2<kType == 1>(y[4], y[5]),
                       pack2<kType == 1>(y[6], y[7]));
      }
    }
  }
}

unsigned rows_grid(const QuantRowsLaunch& p) {
  return static_cast<unsigned>((p.num_tokens * p.kv_heads + kStep * kUnroll - 1) / (kStep * kUnroll));
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
