// What the two latent decode kernels share: how the work is cut into equal runs
// (one per CTA or cluster), the walk over a run, and the merge of the units that
// run boundaries cut. kRows: query rows per tile, kTok: cache rows per tile.
#pragma once
#include <algorithm>

#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

struct Partials {
  int32_t* row_info;  // [tokens x heads]: how the row's partials are found, 0 = none
  float* o;           // [2 runs][kRows][512]
  float* lse;         // [2 runs][kRows]
};

struct Sched {
  // A unit takes kSetup + its tiles on the axis that the runs divide, the tiles last.
  int64_t begin, end;  // this run
  int64_t base;        // where the tiles of its first unit begin
  int64_t each;        // length of a run; `rest` runs of all have one more
  int64_t tok;         // first query token of request b
  int b, mt, t0;       // the first unit, and the run's first tile of it
  int q, kv;           // request b's lengths
  int rest, runs;
};

// row_info of a unit cut into `count` >= 2 pieces, the first in run `c`: row r
// of the slots 2c + 1 (first piece), 2 (c + 1), 2 (c + 2), ...
__device__ __forceinline__ int32_t pack_info(int c, int count, int r) { return (count << 17) | (c << 7) | r; }

// The (request, row tile) units' geometry, and the walk over a cluster's run.
template <int kRows, int kTok>
struct Unit {
  const LatentDecodeLaunch& p;
  int cap;
  __device__ explicit Unit(const LatentDecodeLaunch& l) : p(l), cap(l.block_cols * l.block_size) {}
  // query tokens of request b, whose first one is `tok` <= num_tokens: lengths on the device that add up to more than
  // num_tokens are cut there, so that no unit, row or offset lies past the tensors
  __device__ __forceinline__ int q_len(int b, int64_t tok) const {
    return p.q_len > 0 ? p.q_len
                       : static_cast<int>(min(max(p.q_lens[b], static_cast<int64_t>(0)), p.num_tokens - tok));
  }
  // cut to what the block table holds (2^30 - 1 at most), before the causal mask counts from its end
  __device__ __forceinline__ int kv_len(int64_t n) const {
    return static_cast<int>(min(max(n, static_cast<int64_t>(0)), static_cast<int64_t>(cap)));
  }
  __device__ __forceinline__ int row_tiles(int q) const {
    return static_cast<int>((static_cast<int64_t>(q) * p.num_heads + kRows - 1) / kRows);
  }
  // cache rows that query token i < q of a request sees
  __device__ __forceinline__ int limit(int q, int kv, int i) const {
    return max(0, p.causal ? kv - q + i + 1 : kv);
  }
  // tiles of a unit: up to what its last row sees, at least one
  __device__ __forceinline__ int tiles(int q, int kv, int mt) const {
    // (find_run adds these up tile by tile: with the division below, 256 tokens x 128 heads take 30 us more in all)
    if (!p.causal) return max(1, (kv + kTok - 1) / kTok);
    const int last = static_cast<int>(min(static_cast<int64_t>(q) * p.num_heads, static_cast<int64_t>(mt + 1) * kRows) - 1) /
                     p.num_heads;
    return max(1, (limit(q, kv, last) + kTok - 1) / kTok);
  }
};

template <int kRows, int kTok, int kSetup>
struct Walk {
  Unit<kRows, kTok> u;
  // the current piece
  int b, mt, t0, n, q, kv;
  int64_t tok, base;
  bool starts, ends, last;  // last: of the run
  int unit_tiles;

  int next_b, next_mt, next_t0, nq;
  int64_t next_tok, nkv, next_base, end;  // (nkv as loaded: not used, and so not waited for, until the next piece)

  __device__ Walk(const LatentDecodeLaunch& l, const Sched& s)
      : u(l), next_b(s.b), next_mt(s.mt), next_t0(s.t0), nq(s.q), next_tok(s.tok), nkv(s.kv), next_base(s.base), end(s.end) {}
  __device__ __forceinline__ void load() {
    nq = u.q_len(next_b, next_tok);
    nkv = u.p.kv_lens[next_b];
  }
  __device__ __forceinline__ bool next() {
    if (next_base + next_t0 >= end) return false;
    b = next_b, mt = next_mt, t0 = next_t0, q = nq, kv = u.kv_len(nkv), tok = next_tok, base = next_base;
    unit_tiles = u.tiles(q, kv, mt);
    n = static_cast<int>(min(static_cast<int64_t>(unit_tiles), end - base)) - t0;
    starts = t0 == 0;
    ends = t0 + n == unit_tiles;
    next_base = base + unit_tiles + kSetup;
    next_t0 = 0;
    last = next_base >= end;
    if (!last) {  // the next unit's lengths, loaded a piece ahead
      if (++next_mt == u.row_tiles(q)) {
        next_mt = 0;
        do {
          next_tok += nq;
          ++next_b;
          if (next_b >= u.p.batch) {
            last = true;
            next_base = end;
            break;
          }
          load();
        } while (nq == 0);
      }
    }
    return true;
  }
};

// Start of run c: floor(c total / runs), without a wide division.
__device__ __forceinline__ int64_t run_begin(int c, int64_t each, int rest, int runs) {
  return c * each + static_cast<uint32_t>(c * rest) / static_cast<uint32_t>(runs);
}

// row_info of row r of a unit whose first piece is this run's and whose last
// tile is at `last`: finds the run that holds it.
__device__ __forceinline__ int32_t cut_info(const Sched& s, int run, int64_t last, int r) {
  int hi = run + static_cast<int>(min(static_cast<float>(s.runs - 1 - run),
                                      static_cast<float>(last - s.begin) / static_cast<float>(s.each + (s.rest > 0))));
  while (hi + 1 < s.runs && run_begin(hi + 1, s.each, s.rest, s.runs) <= last) ++hi;
  while (hi > run && run_begin(hi, s.each, s.rest, s.runs) > last) --hi;
  return pack_info(run, hi - run + 1, r);
}

// Finds this cluster's run: the block sums the query tokens (if their lengths are on
// the device) and the units' lengths on the axis per contiguous chunk of requests, then
// the thread whose chunk holds the run's start walks to it. A run that ends in a unit's set-up has none of its
// tiles, one that starts there has them from the first on; a few runs may be empty.
// The walk over a request's row tiles is one thread's, in every CTA and before any
// load: 256 query tokens x 128 heads over 64 cache rows take 37 us, 4,096 tokens x 128
// heads 437 us (floors 11 and 177; in a graph).
// Rows past the requests' tokens (lengths on the device may add up to less than
// num_tokens) belong to no unit: their row_info is cleared here, for the merge to pass them by.
template <int kRows, int kTok, int kSetup, int kThreads>
__device__ __forceinline__ void find_run(const LatentDecodeLaunch& p, int32_t* row_info, int cluster, int clusters,
                                         int64_t (*scan)[kThreads / 32], Sched* sched) {
  const Unit<kRows, kTok> u(p);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  // the sum over this thread and those before it in `sum`, over all in the result
  auto scan_sum = [&](int64_t& sum, int64_t* slot) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += a;
    }
    if (lane == 31) slot[warp] = sum;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) sum += slot[w];
      all += slot[w];
    }
    return all;
  };
  int64_t tok0 = static_cast<int64_t>(b0) * p.q_len;  // the first query token of request b0
  const int64_t kv0 = b0 < b1 ? p.kv_lens[b0] : 0;     // (on its way during the scan)
  if (p.q_len == 0) {
    int64_t toks = 0;
    for (int b = b0; b < b1; ++b) toks += u.q_len(b, 0);
    tok0 = -toks;
    const int64_t own = min(scan_sum(toks, scan[1]), p.num_tokens);  // tokens that belong to requests
    tok0 = min(tok0 + toks, p.num_tokens);
    for (int64_t i = own * p.num_heads + cluster * kThreads + tid; i < p.num_tokens * p.num_heads; i += clusters * kThreads)
      row_info[i] = 0;
  }
  int64_t tiles = 0, tok = tok0;
  for (int b = b0; b < b1; ++b) {
    const int q = u.q_len(b, tok), kv = u.kv_len(b == b0 ? kv0 : p.kv_lens[b]), m = u.row_tiles(q);
    for (int mt = 0; mt < m; ++mt) tiles += kSetup + u.tiles(q, kv, mt);
    tok += q;
  }
  int64_t st = tiles;
  if (tid == 0) sched->base = sched->end = 0, sched->t0 = 0;  // no run
  const int64_t total = scan_sum(st, scan[0]);
  const int64_t runs = min(static_cast<int64_t>(clusters), total);
  if (cluster < runs) {
    const int n_runs = static_cast<int>(runs);
    const int64_t each = total >> 31 ? total / runs : static_cast<uint32_t>(total) / static_cast<uint32_t>(n_runs);
    const int rest = static_cast<int>(total - each * runs);
    const int64_t begin = run_begin(cluster, each, rest, n_runs), end = run_begin(cluster + 1, each, rest, n_runs);
    int64_t at = st - tiles;
    if (begin >= at && begin < st) {
      tok = tok0;
      for (int b = b0; b < b1; ++b) {
        const int q = u.q_len(b, tok), kv = u.kv_len(p.kv_lens[b]), m = u.row_tiles(q);
        for (int mt = 0; mt < m; ++mt) {
          const int t = kSetup + u.tiles(q, kv, mt);
          if (begin < at + t) {
            *sched = {begin, end, at + kSetup, each, tok, b, mt, static_cast<int>(max(begin - at - kSetup, static_cast<int64_t>(0))),
                      q, kv, rest, n_runs};
            b = b1;
            break;
          }
          at += t;
        }
        tok += q;
      }
    }
  }
  __syncthreads();
}

// Merges the partials of the rows whose unit was cut, in run order, weights
// exp(lse_i - max): kWarps warps per row take every kWarps-th piece, four in
// flight each, and their sums meet in shared memory. Bound by the chain row info
// -> partials and log-sum-exps. Few rows (they may have a piece per run) get eight
// warps, many rows, with two or three pieces each, one.
constexpr int64_t kFewRows = 1024;
template <bool kFp16, int kRows, int kWarps>
__global__ void __launch_bounds__(256) latent_combine_kernel(const __grid_constant__ LatentDecodeLaunch L,
                                                             const __grid_constant__ Partials P, int clusters) {
  constexpr int kDepth = 4, kVec = 4;  // pieces in flight, float4 of a piece per lane
  __shared__ float4 part[kWarps == 1 ? 1 : 8][kLatentDim / 4];
  __shared__ float part_sum[8];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 8 + warp) / kWarps;
  if (row >= L.num_tokens * L.num_heads) return;
  const int32_t info = P.row_info[row];
  const int count = info >> 17, c0 = (info >> 7) & 1023, r = info & 127;
  // (an aborted run may have left its rows' info as the workspace held it: nothing past the slots is read for them)
  if (count < 2 || c0 + count > clusters || r >= kRows) return;
  auto slot = [&](int i) { return static_cast<int64_t>(i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * kRows + r; };
  const int first = kWarps == 1 ? 0 : warp;
  float4 v[kDepth][kVec];
  float lse[kDepth];
  auto read = [&](int i0) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int i = i0 + d * kWarps;
      if (i >= count) break;
      lse[d] = P.lse[slot(i)];
      const float4* src = reinterpret_cast<const float4*>(P.o + slot(i) * kLatentDim) + lane;
#pragma unroll
      for (int k = 0; k < kVec; ++k) v[d][k] = src[32 * k];
    }
  };
  read(first);
  float top = -INFINITY;
  for (int i = lane; i < count; i += 32) top = fmaxf(top, P.lse[slot(i)]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float4 acc[kVec] = {};
  float sum = 0.f;
  for (int i0 = first; i0 < count; i0 += kDepth * kWarps) {
    if (i0 > first) read(i0);
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (i0 + d * kWarps >= count) break;
      const float wgt = lse[d] == -INFINITY ? 0.f : __expf(lse[d] - top);
      sum += wgt;
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        acc[k].x = fmaf(wgt, v[d][k].x, acc[k].x);
        acc[k].y = fmaf(wgt, v[d][k].y, acc[k].y);
        acc[k].z = fmaf(wgt, v[d][k].z, acc[k].z);
        acc[k].w = fmaf(wgt, v[d][k].w, acc[k].w);
      }
    }
  }
  uint2* out = reinterpret_cast<uint2*>(static_cast<uint16_t*>(L.out) + row * kLatentDim);
  auto write = [&](int at, float4 a, float inv) {
    out[at] = make_uint2(pack2<kFp16>(a.x * inv, a.y * inv), pack2<kFp16>(a.z * inv, a.w * inv));
  };
  if constexpr (kWarps == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < kVec; ++k) write(32 * k + lane, acc[k], inv);
  } else {  // (the block has one row, all its warps are here)
#pragma unroll
    for (int k = 0; k < kVec; ++k) part[warp][32 * k + lane] = acc[k];
    if (lane == 0) part_sum[warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += part_sum[i];
    if (threadIdx.x < kLatentDim / 4) {
      float4 a = part[0][threadIdx.x];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        const float4 b = part[i][threadIdx.x];
        a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w;
      }
      write(threadIdx.x, a, sum == 0.f ? 0.f : 1.f / sum);
    }
  }
  if (threadIdx.x % (32 * kWarps) == 0) L.lse[row] = sum == 0.f ? -INFINITY : top + __logf(sum);
}

inline size_t info_bytes(const LatentDecodeLaunch& p) {
  return (static_cast<size_t>(p.num_tokens) * p.num_heads * sizeof(int32_t) + 255) / 256 * 256;
}

template <int kRows>
size_t partial_bytes(const LatentDecodeLaunch& p, int runs) {
  return info_bytes(p) + static_cast<size_t>(runs) * 2 * kRows * (kLatentDim + 1) * sizeof(float);
}

template <int kRows>
Partials partials(const LatentDecodeLaunch& p, int runs, void* workspace) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* o = reinterpret_cast<float*>(ws + info_bytes(p));
  return {reinterpret_cast<int32_t*>(ws), o, o + static_cast<size_t>(runs) * 2 * kRows * kLatentDim};
}

// Runs of a launch: more would stay empty, whatever the lengths.
template <int kRows, int kTok, int kSetup>
int run_bound(const LatentDecodeLaunch& p, int most) {
  const int64_t rows = p.num_tokens * p.num_heads;
  const int64_t units = p.batch + rows / kRows;
  const int64_t tiles = std::max<int64_t>(1, (static_cast<int64_t>(p.block_cols) * p.block_size + kTok - 1) / kTok);
  return static_cast<int>(std::min<int64_t>(most, std::min<int64_t>(units, 1 << 20) * (kSetup + tiles)));
}

template <bool kFp16, int kRows, int kTok>
cudaError_t launch_combine(const LatentDecodeLaunch& p, const Partials& parts, int runs, cudaStream_t stream) {
  // one run, or units of one tile: none is cut
  if (runs == 1 || static_cast<int64_t>(p.block_cols) * p.block_size <= kTok) return cudaSuccess;
  const int64_t rows = p.num_tokens * p.num_heads;
  const bool few = rows <= kFewRows;
  cudaLaunchConfig_t cc = {};
  cc.gridDim = dim3(static_cast<unsigned>(few ? rows : (rows + 7) / 8));
  cc.blockDim = dim3(256);
  cc.stream = stream;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cc.attrs = pdl;
  cc.numAttrs = 1;
  return few ? cudaLaunchKernelEx(&cc, latent_combine_kernel<kFp16, kRows, 8>, p, parts, runs)
             : cudaLaunchKernelEx(&cc, latent_combine_kernel<kFp16, kRows, 1>, p, parts, runs);
}

}  // namespace
}  // namespace cascade
