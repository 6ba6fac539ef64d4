// Log probabilities of tokens (cascade_token_logprobs): one CTA per row, a pass
// for the maximum, the sums and the rank, and one per alternative.
#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

constexpr int kThreads = 512;

template <int kType>
__device__ __forceinline__ float load(const void* base, int64_t i) {
  if constexpr (kType == 2) return __ldg(static_cast<const float*>(base) + i);
  const uint16_t b = __ldg(static_cast<const uint16_t*>(base) + i);
  if constexpr (kType == 1) return __half2float(__ushort_as_half(b));
  return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

// a logit's place in the order: larger first, lower index first among equals, a NaN as -inf; never 0
__device__ __forceinline__ uint64_t make_key(float x, uint32_t v) {
  const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.f);
  const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (static_cast<uint64_t>(up) << 32) | (0xffffffffu - v);
}

template <class T, class Op>
__device__ __forceinline__ T block_reduce(T v, T* slot, Op op) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, d));
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  v = slot[0];
  for (int w = 1; w < kThreads / 32; ++w) v = op(v, slot[w]);
  __syncthreads();
  return v;
}

template <int kType>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobsLaunch p) {
  __shared__ float slots[kThreads / 32];
  __shared__ uint64_t keys[kThreads / 32];
  const int64_t n = blockIdx.x;
  const void* row = static_cast<const char*>(p.logits) + n * p.row_stride * (kType == 2 ? 4 : 2);
  const int64_t V = p.vocab, token = p.tokens[n];
  const bool given = token >= 0 && token < V;
  const float mine = given ? load<kType>(row, token) : 0.f;
  const uint64_t key = given ? make_key(mine, static_cast<uint32_t>(token)) : 0;
  float top = -INFINITY;
  uint64_t ahead = 0;
  for (int64_t v = threadIdx.x; v < V; v += kThreads) {
    const float x = load<kType>(row, v);
    top = fmaxf(top, x);
    ahead += make_key(x, static_cast<uint32_t>(v)) > key;
  }
  top = block_reduce(top, slots, [](float a, float b) { return fmaxf(a, b); });
  ahead = block_reduce(ahead, keys, [](uint64_t a, uint64_t b) { return a + b; });
  float sum = 0.f, dot = 0.f;
  for (int64_t v = threadIdx.x; v < V; v += kThreads) {
    const float d = load<kType>(row, v) - top, e = expf(d);
    sum += e;
    dot += e > 0.f ? e * d : e != e ? e : 0.f;
  }
  sum = block_reduce(sum, slots, [](float a, float b) { return a + b; });
  dot = block_reduce(dot, slots, [](float a, float b) { return a + b; });
  const float norm = logf(sum);
  if (threadIdx.x == 0) {
    p.logprob[n] = given ? (mine - top) - norm : -INFINITY;
    p.entropy[n] = norm - dot / sum;
    p.rank[n] = given ? static_cast<int64_t>(ahead) : -1;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    uint64_t best = 0;
    for (int64_t v = threadIdx.x; v < V; v += kThreads) {
      const uint64_t a = make_key(load<kType>(row, v), static_cast<uint32_t>(v));
      if (a < last && a > best) best = a;
    }
    last = block_reduce(best, keys, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    if (threadIdx.x == 0) {
      const int64_t v = 0xffffffffu - static_cast<uint32_t>(last);
      p.top_tokens[n * p.top + k] = v;
      p.top_logprobs[n * p.top + k] = (load<kType>(row, v) - top) - norm;
    }
  }
}

}  // namespace

size_t token_logprobs_workspace(const LogprobsLaunch&) { return 0; }

cudaError_t launch_token_logprobs(const LogprobsLaunch& p, void*, cudaStream_t stream) {
  (p.dtype == 2 ? logprobs_kernel<2> : p.dtype == 1 ? logprobs_kernel<1> : logprobs_kernel<0>)
      <<<static_cast<unsigned>(p.rows), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace cascade
