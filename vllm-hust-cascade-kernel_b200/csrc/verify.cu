// Verification of drafted tokens (cascade_verify_drafts).
//
// Draft i of a request is accepted while u_i q_i(x_i) < p_i(x_i); the token
// after the accepted ones is argmax_v r(v) / e(v) with r = max(p - q, 0) at the
// first refused place (p of the row after the last draft if none was), e
// independent exponential variates: P[argmax = v] = r(v) / sum r.
//
// Only one row of p, q and e is read per request, once: HBM-bound for large
// batches, and for small ones bound by the chain draft token -> its two
// probabilities -> the row. A cluster of CTAs shares a request's row; every CTA
// repeats the acceptance (a few gathered loads) instead of waiting for another's,
// and the CTAs' best entries meet in every CTA's shared memory.
//
// Measured: 128 requests x 128,256 entries in fp32 (170 MB, floor 26 us) 33.4 us,
// 5.1 TB/s, in bf16 (about 118 MB, floor 18 us) 26.8 in a graph (41 us with a division per positive entry and single loads); 4
// requests x 32,000 entries 5.7 us, a launch and four dependent loads.
//
// Each value is one rounded product, difference and quotient in fp32, and the
// best entry is the largest (quotient, lowest index), so the answer does not
// depend on how the row was split.
#include <cooperative_groups.h>

#include <type_traits>

#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kPerSm = 4;    // CTAs resident per SM (64 registers); 3 or 5 with the loads that fit: 39, 40 us for 33.5
// loads of each row in flight per thread: single entries, or groups of four (1: 35, 3: 38 us for 33.5)
template <int kW>
constexpr int kUnroll = kW == 1 ? 5 : 2;
constexpr int kMaxCtas = 8;  // CTAs per request

template <int kType>
__device__ __forceinline__ float load(const void* base, int64_t i) {
  if constexpr (kType == 2) return __ldg(static_cast<const float*>(base) + i);
  const uint16_t b = __ldg(static_cast<const uint16_t*>(base) + i);
  if constexpr (kType == 1) return __half2float(__ushort_as_half(b));
  return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

// kW entries from entry i on, i a multiple of kW (four: a load of 16 or 8 bytes).
template <int kType, int kW>
__device__ __forceinline__ void load_group(const void* base, int i, float (&x)[kW]) {
  if constexpr (kW == 1) {
    x[0] = load<kType>(base, i);
  } else if constexpr (kType == 2) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + i));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i));
    const uint32_t w[2] = {v.x, v.y};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
      x[j] = kType == 1 ? __half2float(__ushort_as_half(static_cast<uint16_t>(b))) : __uint_as_float(b << 16);
    }
  }
}

// (quotient, index) as one ordered key: larger quotient first, then lower
// index. Quotients are >= 0, so their bits order as integers. 0 = no entry.
__device__ __forceinline__ uint64_t make_key(float quotient, uint32_t v) {
  return (static_cast<uint64_t>(__float_as_uint(quotient)) << 32) | (0xffffffffu - v);
}

__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <int kType, int kW>
__global__ void __launch_bounds__(kThreads, kPerSm) verify_kernel(const VerifyLaunch p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t b = blockIdx.x / ctas;
  const int64_t K = p.drafts, V = p.vocab;
  const int64_t n = min(max(p.draft_lens[b], static_cast<int64_t>(0)), K);
  __shared__ int64_t s_taken;
  __shared__ uint64_t s_best[kThreads / 32], s_all[kMaxCtas];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  cluster.barrier_arrive();  // waited for before the first write to another CTA: all have started by then

  if (warp == 0) {
    int64_t taken = n;  // the first refused draft
    for (int64_t i0 = 0; i0 < n; i0 += 32) {
      const int64_t i = i0 + lane;
      bool refused = false;
      if (i < n) {
        const int64_t x = p.tokens[b * K + i];
        refused = true;
        if (x >= 0 && x < V) {
          const float q = p.draft ? load<kType>(p.draft, (b * K + i) * V + x) : 1.f;
          const float t = load<kType>(p.target, (b * (K + 1) + i) * V + x);
          refused = !(__fmul_rn(p.uniform[b * K + i], q) < t);
        }
      }
      const uint32_t any = __ballot_sync(0xffffffffu, refused);
      if (any) {
        taken = i0 + __ffs(any) - 1;
        break;
      }
    }
    if (lane == 0) s_taken = taken;
  }
  __syncthreads();
  const int64_t taken = s_taken;
  const bool refused = taken < n;
  // the three rows; the entries are walked with 32-bit indices
  const int element = kType == 2 ? 4 : 2, n_v = static_cast<int>(V);
  const void* prow = static_cast<const char*>(p.target) + (b * (K + 1) + taken) * V * element;
  const void* qrow = refused && p.draft ? static_cast<const char*>(p.draft) + (b * K + taken) * V * element : nullptr;
  const float* erow = p.noise + b * V;
  // the token left out: -1 where it is no entry of the row, before it is narrowed to the entries' 32 bits
  const int64_t token = refused && !p.draft ? p.tokens[b * K + taken] : -1;
  const int out = token >= 0 && token < V ? static_cast<int>(token) : -1;

  // the best entry of this cluster's row: pass 0 over `left`; pass 1, only
  // when left is 0 everywhere, over the target's row
  uint64_t best = 0;
  for (int pass = 0; pass < 2; ++pass) {
    const bool minus = pass == 0 && qrow;
    const int skip = pass == 0 ? out : -1;
    const int stride = ctas * kThreads * kW, block = stride * kUnroll<kW>;
    int v0 = (rank * kThreads + static_cast<int>(threadIdx.x)) * kW;
    // `best` as (quotient, index): the thread meets its indices in ascending order, so a later one has to be larger
    float top = -1.f, bar = -1.f;
    int at = 0;
    // bar: the warp's best of the rounds before. left < fl(bar e) means left / e < bar (rounding keeps order), and
    // what rounds to an equal quotient loses to the lower index: such entries need no division.
    auto take = [&](float t, float q, float e, int v) {
      const float left = __fsub_rn(t, q);
      if (left > 0.f && left >= __fmul_rn(bar, e) && v != skip) {
        const float quotient = __fdiv_rn(left, e);
        if (quotient > top) top = quotient, at = v;
      }
    };
    auto round = [&](auto whole) {
      float t[kUnroll<kW>][kW], q[kUnroll<kW>][kW], e[kUnroll<kW>][kW];
#pragma unroll
      for (int u = 0; u < kUnroll<kW>; ++u) {
        const int v = v0 + u * stride;
        if (whole.value || v < n_v) {  // (groups are whole: the row's length is a multiple of kW)
          load_group<kType, kW>(prow, v, t[u]);
          load_group<2, kW>(erow, v, e[u]);
          if (minus) load_group<kType, kW>(qrow, v, q[u]);
        } else {
#pragma unroll
          for (int j = 0; j < kW; ++j) t[u][j] = 0.f, e[u][j] = 1.f, q[u][j] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll<kW>; ++u) {
#pragma unroll
        for (int j = 0; j < kW; ++j) take(t[u][j], minus ? q[u][j] : 0.f, e[u][j], v0 + u * stride + j);
      }
    };
    // rounds that are whole for the warp's last lane: its lanes stay together, and the rest is at most one round
    for (; v0 + (31 - lane) * kW + (kUnroll<kW> - 1) * stride < n_v; v0 += block) {
      round(std::true_type());
      // (as whole numbers: -1 or quotients that are not negative)
      bar = __int_as_float(__reduce_max_sync(0xffffffffu, __float_as_int(top)));
    }
    round(std::false_type());
    best = top >= 0.f ? make_key(top, static_cast<uint32_t>(at)) : 0;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) best = max_u64(best, __shfl_xor_sync(0xffffffffu, best, d));
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
    if (pass == 0) cluster.barrier_wait();
    if (warp == 0) {
      best = lane < kThreads / 32 ? s_best[lane] : 0;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) best = max_u64(best, __shfl_xor_sync(0xffffffffu, best, d));
      if (lane < ctas) cluster.map_shared_rank(s_all, lane)[rank] = best;
    }
    cluster.sync();
    best = 0;
    for (int r = 0; r < ctas; ++r) best = max_u64(best, s_all[r]);
    if (best != 0) break;
    cluster.sync();  // s_all is written again
  }
  if (rank == 0) {
    // nothing positive in the whole row: index 0, as an argmax over zeros
    const int64_t last = best ? static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(best)) : 0;
    for (int64_t i = threadIdx.x; i <= K; i += kThreads)
      p.out_tokens[b * (K + 1) + i] = i < taken ? p.tokens[b * K + i] : i == taken ? last : -1;
    if (threadIdx.x == 0) p.accepted[b] = taken;
  }
}

}  // namespace

cudaError_t launch_verify_drafts(const VerifyLaunch& p, cudaStream_t stream) {
  // as many CTAs per request as run at once, with at least one unrolled round
  // of the row each
  int ctas = 1;
  while (ctas < kMaxCtas && p.batch * ctas * 2 <= kPerSm * kNumSMs &&
         p.vocab > static_cast<int64_t>(ctas) * kThreads * 8)
    ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.batch * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Groups of four entries where every row starts at a multiple of four and the tensors allow the loads.
  // 128 requests x 128,256 entries: fp32 33.5 us against 35.8 with single entries, bf16 26.6 against 32.9.
  auto on = [](const void* ptr, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes == 0; };
  const uintptr_t bytes = p.dtype == 2 ? 16 : 8;
  const bool four = p.vocab % 4 == 0 && on(p.target, bytes) && on(p.draft, bytes) && on(p.noise, 16);
  auto kern = four ? (p.dtype == 2 ? verify_kernel<2, 4> : p.dtype == 1 ? verify_kernel<1, 4> : verify_kernel<0, 4>)
                   : (p.dtype == 2 ? verify_kernel<2, 1> : p.dtype == 1 ? verify_kernel<1, 1> : verify_kernel<0, 1>);
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace cascade
