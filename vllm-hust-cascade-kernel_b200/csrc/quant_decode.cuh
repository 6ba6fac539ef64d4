// What the kernels over a 4-bit cache share: the units of work, how they are cut
// into equal runs, and the merge of the units that run boundaries cut.
#pragma once
#include <algorithm>

#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

// A unit is a block of query rows of one request and kv head over the tokens its
// last row sees. Per kv head the units lie one after the other on an axis, each
// kSetup + its tiles long; the axis is cut into `runs` equal runs.
template <int kRows, int kTok>
struct QuantUnit {
  const QuantDecodeLaunch& p;
  int cap;
  __device__ explicit QuantUnit(const QuantDecodeLaunch& l) : p(l), cap(l.block_cols * l.block_size) {}
  // query tokens of request b, whose first one is `tok` <= num_tokens: lengths on the device that add up to more than
  // num_tokens are cut there, so that no unit, row or offset lies past the tensors
  __device__ __forceinline__ int q_len(int b, int64_t tok) const {
    return p.q_len > 0 ? p.q_len
                       : static_cast<int>(min(max(p.q_lens[b], static_cast<int64_t>(0)), p.num_tokens - tok));
  }
  // cut to what the block table holds (2^30 - 1 at most), before the causal mask counts from its end
  __device__ __forceinline__ int kv_len(int b) const {
    return static_cast<int>(min(max(p.kv_lens[b], static_cast<int64_t>(0)), static_cast<int64_t>(cap)));
  }
  __device__ __forceinline__ int blocks(int q) const { return (q * p.group + kRows - 1) / kRows; }
  // cached tokens that query token i < q of a request sees
  __device__ __forceinline__ int limit(int q, int kv, int i) const {
    return max(0, p.causal ? kv - q + i + 1 : kv);
  }
  // tiles of a unit: up to what its last row sees, at least one
  __device__ __forceinline__ int tiles(int q, int kv, int block) const {
    if (!p.causal) return max(1, (kv + kTok - 1) / kTok);
    const int last = (min(q * p.group, (block + 1) * kRows) - 1) / p.group;
    return max(1, (limit(q, kv, last) + kTok - 1) / kTok);
  }
};

// Rows of units that were cut: their pieces lie in the slots 2c + 1 (the first
// piece, the last of run c), 2 (c + 1), 2 (c + 2), ... of their kv head.
struct QuantPartials {
  int32_t* row_info;  // [tokens x heads]: how the row's partials are found, 0 = none
  float* o;           // [2 runs][kv heads][rows of a block][128], normalised
  float* lse;         // [2 runs][kv heads][rows of a block]
  int32_t runs;
};
// row r of a unit cut into `count` >= 2 pieces, the first in run c
__device__ __forceinline__ int32_t pack_info(int c, int count, int r) {
  return static_cast<int32_t>(static_cast<uint32_t>(count) << 20 | static_cast<uint32_t>(c) << 8 | static_cast<uint32_t>(r));
}
constexpr int kMaxRuns = 4095, kMaxBlockRows = 256;

// A run, as its first unit and the place in it.
struct QuantRun {
  int64_t begin, end;  // on the axis; no run: end = begin
  int64_t base;        // where the tiles of the first unit begin
  int64_t tok;         // first query token of request b
  int64_t each;        // length of a run; `rest` of the `runs` runs have one more
  int b, block, t0, q, kv;
  int rest, runs;
};

// Start of run c: floor(c total / runs), without a wide division.
__device__ __forceinline__ int64_t run_begin(int c, int64_t each, int rest, int runs) {
  return c * each + static_cast<uint32_t>(c * rest) / static_cast<uint32_t>(runs);
}

// Finds run c of one kv head's axis (the same for every head); one warp.
template <int kRows, int kTok, int kSetup>
__device__ __forceinline__ QuantRun find_run(const QuantUnit<kRows, kTok>& u, int c, int runs) {
  const int lane = threadIdx.x & 31;
  const QuantDecodeLaunch& p = u.p;
  const int per = (p.batch + 31) / 32;
  const int b0 = min(p.batch, lane * per), b1 = min(p.batch, b0 + per);
  auto before = [&](int64_t v) {  // sum over the lanes below
    int64_t s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += a;
    }
    return s - v;
  };
  int64_t tok0 = static_cast<int64_t>(b0) * p.q_len;
  if (p.q_len == 0) {
    int64_t n = 0;
    for (int b = b0; b < b1; ++b) n += u.q_len(b, 0);
    tok0 = min(before(n), p.num_tokens);
  }
  int64_t mine = 0, tok = tok0;
  int last_kv = 0;
  for (int b = b0; b < b1; ++b) {
    const int q = u.q_len(b, tok), kv = last_kv = u.kv_len(b), m = u.blocks(q);
    if (!p.causal)
      mine += static_cast<int64_t>(m) * (kSetup + u.tiles(q, kv, 0));
    else
      for (int i = 0; i < m; ++i) mine += kSetup + u.tiles(q, kv, i);
    tok += q;
  }
  int64_t at = before(mine);
  const int64_t total = __shfl_sync(0xffffffffu, at + mine, 31);
  QuantRun r = {};
  r.runs = runs = static_cast<int>(min(static_cast<int64_t>(runs), total));
  if (c >= runs) return r;
  r.each = total >> 31 ? total / runs : static_cast<uint32_t>(total) / static_cast<uint32_t>(runs);
  r.rest = static_cast<int>(total - r.each * runs);
  r.begin = run_begin(c, r.each, r.rest, runs), r.end = run_begin(c + 1, r.each, r.rest, runs);
  const uint32_t who = __ballot_sync(0xffffffffu, r.begin >= at && r.begin < at + mine);
  const int owner = __ffs(who) - 1;
  if (lane == owner) {
    tok = tok0;
    bool found = false;
    for (int b = b0; b < b1 && !found; ++b) {
      const int q = u.q_len(b, tok), kv = per == 1 ? last_kv : u.kv_len(b), m = u.blocks(q);
      for (int i = 0; i < m; ++i) {
        const int t = kSetup + u.tiles(q, kv, i);
        if (r.begin < at + t) {
          r.base = at + kSetup, r.tok = tok, r.b = b, r.block = i, r.q = q, r.kv = kv;
          r.t0 = static_cast<int>(max(r.begin - r.base, static_cast<int64_t>(0)));
          found = true;
          break;
        }
        at += t;
      }
      tok += q;
    }
  }
  r.base = __shfl_sync(0xffffffffu, r.base, owner);
  r.tok = __shfl_sync(0xffffffffu, r.tok, owner);
  r.b = __shfl_sync(0xffffffffu, r.b, owner);
  r.block = __shfl_sync(0xffffffffu, r.block, owner);
  r.t0 = __shfl_sync(0xffffffffu, r.t0, owner);
  r.q = __shfl_sync(0xffffffffu, r.q, owner);
  r.kv = __shfl_sync(0xffffffffu, r.kv, owner);
  return r;
}

// The walk over a run, piece by piece (a piece: the run's part of a unit). The next request's lengths are loaded a piece ahead.
template <int kRows, int kTok, int kSetup>
struct QuantWalk {
  QuantUnit<kRows, kTok> u;
  int b, block, t0, n, q, kv;  // the current piece: tiles t0 .. t0 + n of its unit
  int64_t tok, base;
  bool starts, ends;
  int64_t next_base, end;
  int next_t0, next_b, next_q;
  int64_t next_kv;  // as loaded: not used, and so not waited for, until the next piece
  bool fresh;       // the next piece is the first block of request next_b
  __device__ QuantWalk(const QuantDecodeLaunch& l, const QuantRun& r)
      : u(l), b(r.b), block(r.block - 1), t0(0), n(0), q(r.q), kv(r.kv), tok(r.tok), base(0), starts(false), ends(false),
        next_base(r.base), end(r.end), next_t0(r.t0), next_b(0), next_q(0), next_kv(0), fresh(false) {}
  __device__ __forceinline__ bool next() {
    if (next_base + next_t0 >= end) return false;
    if (fresh) {
      block = 0, tok += q, b = next_b, q = next_q;
      kv = static_cast<int>(min(max(next_kv, static_cast<int64_t>(0)), static_cast<int64_t>(u.cap)));
    } else {
      ++block;
    }
    base = next_base;
    const int all = u.tiles(q, kv, block);
    t0 = next_t0;
    n = static_cast<int>(min(static_cast<int64_t>(all), end - base)) - t0;
    starts = t0 == 0;
    ends = t0 + n == all;
    next_base = base + all + kSetup;
    next_t0 = 0;
    fresh = false;
    if (next_base < end && block + 1 >= u.blocks(q)) {
      fresh = true;
      for (next_b = b + 1;; ++next_b) {  // requests without query tokens have no units
        if (next_b >= u.p.batch) {
          next_base = end;
          break;
        }
        next_q = u.q_len(next_b, tok + q);
        if (next_q > 0) break;
      }
      if (next_base < end) next_kv = u.p.kv_lens[next_b];
    }
    return true;
  }
};

// centre or scale NaN (or infinite) in either half
__device__ __forceinline__ bool odd_par(uint32_t x) { return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u; }
// bit i: group i of the value of token `tok` (below the request's length) is NaN
__device__ __forceinline__ uint32_t odd_groups(const QuantDecodeLaunch& p, int b, int tok, int shift, int h) {
  const int32_t id = p.block_table[static_cast<int64_t>(b) * p.block_cols + (tok >> shift)];
  if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.num_blocks)) return 0;
  const int64_t row = (static_cast<int64_t>(id) * p.block_size + (tok & (p.block_size - 1))) * p.kv_heads + h;
  const uint4 par = __ldg(reinterpret_cast<const uint4*>(p.value + row * kQuantRow + kQuantCodes));
  return odd_par(par.x) | odd_par(par.y) << 1 | odd_par(par.z) << 2 | odd_par(par.w) << 3;
}

// row_info of a unit whose first piece is run c's and whose last tile is at `last` of the axis, without its row
__device__ __forceinline__ int32_t cut_info(const QuantRun& run, int c, int64_t last) {
  const float total = static_cast<float>(run.each * run.runs + run.rest);
  int hi = max(c, min(run.runs - 1, static_cast<int>(static_cast<float>(last) / total * static_cast<float>(run.runs))));
  while (hi + 1 < run.runs && run_begin(hi + 1, run.each, run.rest, run.runs) <= last) ++hi;
  while (hi > c && run_begin(hi, run.each, run.rest, run.runs) > last) --hi;
  return pack_info(c, hi - c + 1, 0);
}

// Merges the pieces of the rows whose unit was cut, in the pieces' order, weights
// exp(lse_i - max): kWarps warps per row take every kWarps-th piece, eight in
// flight each, and their sums meet in shared memory. Bound by the chain row info
// -> partials. Few rows (with up to a piece per run) get many warps.
template <bool kFp16, int kBlockRows, int kWarps>
__global__ void __launch_bounds__(kWarps == 1 ? 256 : 32 * kWarps)
    quant_combine_kernel(const __grid_constant__ QuantDecodeLaunch L, const __grid_constant__ QuantPartials P) {
  constexpr int kDepth = 8;
  __shared__ float4 part[kWarps == 1 ? 1 : kWarps][32];
  __shared__ float part_sum[kWarps], part_top[kWarps];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = kWarps == 1 ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  if (row >= L.num_tokens * L.num_heads) return;
  const uint32_t info = static_cast<uint32_t>(P.row_info[row]);
  const int count = static_cast<int>(info >> 20), c0 = static_cast<int>(info >> 8) & kMaxRuns, r = static_cast<int>(info) & (kMaxBlockRows - 1);
  // (an aborted run may have left its rows' info as the workspace held it: nothing past the slots is read for them)
  if (count < 2 || c0 + count > P.runs || r >= kBlockRows) return;
  const int h = static_cast<int>(row % L.num_heads) / L.group;
  auto slot = [&](int i) {
    return (static_cast<int64_t>(i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * L.kv_heads + h) * kBlockRows + r;
  };
  const int step = kWarps == 1 ? 1 : kWarps, begin = kWarps == 1 ? 0 : warp;
  float top = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = begin; i0 < count; i0 += kDepth * step) {
    float4 v[kDepth];
    float lse[kDepth], most = top;
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int i = i0 + d * step;
      lse[d] = i < count ? P.lse[slot(i)] : -INFINITY;
      v[d] = i < count ? reinterpret_cast<const float4*>(P.o + slot(i) * kHeadDim)[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) most = fmaxf(most, lse[d]);
    if (most == -INFINITY) {  // (nothing seen so far, or NaN alone, which the sum keeps)
#pragma unroll
      for (int d = 0; d < kDepth; ++d) sum += lse[d] != lse[d] ? lse[d] : 0.f;
      continue;
    }
    const float f = __expf(top - most);
    top = most;
    sum *= f, acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (i0 + d * step >= count) break;
      const float w = __expf(lse[d] - top);
      sum += w;
      acc.x = fmaf(w, v[d].x, acc.x), acc.y = fmaf(w, v[d].y, acc.y);
      acc.z = fmaf(w, v[d].z, acc.z), acc.w = fmaf(w, v[d].w, acc.w);
    }
  }
  if constexpr (kWarps > 1) {
    part[warp][lane] = acc;
    if (lane == 0) part_sum[warp] = sum, part_top[warp] = top;
    __syncthreads();
    if (warp > 0) return;
    float w = lane < kWarps ? part_top[lane] : -INFINITY;
    top = w;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    w = w == -INFINITY ? 0.f : __expf(w - top);
    sum = lane < kWarps ? (w == 0.f && part_sum[lane] == part_sum[lane] ? 0.f : part_sum[lane] * (w == 0.f ? 1.f : w)) : 0.f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const float4 a = part[i][lane];
      acc.x = fmaf(wi, a.x, acc.x), acc.y = fmaf(wi, a.y, acc.y);
      acc.z = fmaf(wi, a.z, acc.z), acc.w = fmaf(wi, a.w, acc.w);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  reinterpret_cast<uint2*>(static_cast<uint16_t*>(L.out) + row * kHeadDim)[lane] =
      make_uint2(pack2<kFp16>(acc.x * inv, acc.y * inv), pack2<kFp16>(acc.z * inv, acc.w * inv));
  if (lane == 0) L.lse[row] = sum == 0.f ? -INFINITY : top + logf(sum);
}

inline size_t quant_info_bytes(const QuantDecodeLaunch& p) {
  return (static_cast<size_t>(p.num_tokens) * p.num_heads * sizeof(int32_t) + 255) / 256 * 256;
}
inline size_t quant_partial_bytes(const QuantDecodeLaunch& p, int runs, int block_rows) {
  if (runs == 1) return quant_info_bytes(p);  // (no unit is cut)
  return quant_info_bytes(p) + static_cast<size_t>(runs) * 2 * p.kv_heads * block_rows * (kHeadDim + 1) * sizeof(float);
}
inline QuantPartials quant_partials(const QuantDecodeLaunch& p, int runs, int block_rows, void* workspace) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* o = reinterpret_cast<float*>(ws + quant_info_bytes(p));
  return {reinterpret_cast<int32_t*>(ws), o, o + static_cast<size_t>(runs) * 2 * p.kv_heads * block_rows * kHeadDim, runs};
}

template <bool kFp16, int kBlockRows>
cudaError_t launch_quant_combine(const QuantDecodeLaunch& p, const QuantPartials& parts, cudaStream_t stream) {
  const int64_t rows = p.num_tokens * p.num_heads;
  const bool many = rows > 2048;
  cudaLaunchConfig_t cc = {};
  cc.gridDim = dim3(static_cast<unsigned>(many ? (rows + 7) / 8 : rows));
  cc.blockDim = dim3(256);
  cc.stream = stream;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cc.attrs = pdl;
  cc.numAttrs = 1;
  if (many) return cudaLaunchKernelEx(&cc, quant_combine_kernel<kFp16, kBlockRows, 1>, p, parts);
  if (rows > 256) return cudaLaunchKernelEx(&cc, quant_combine_kernel<kFp16, kBlockRows, 8>, p, parts);
  cc.blockDim = dim3(1024);
  return cudaLaunchKernelEx(&cc, quant_combine_kernel<kFp16, kBlockRows, 32>, p, parts);
}

}  // namespace
}  // namespace cascade
