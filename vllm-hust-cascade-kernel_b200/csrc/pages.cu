// Pages of a cache: copy, fork, free, compact (cascade_page_*).
//
// The index work (counts, ranks of free pages, new tables) is one launch of
// one cluster of eight CTAs: each CTA owns an eighth of the page ids, and the
// cluster barrier stands where a grid-wide one would be needed (counts known
// -> ranks written -> references and tables updated). It moves a few hundred
// KB at most and is bound by the latency of its three or four dependent
// rounds. The page contents are moved by a second launch, a programmatic
// dependent, that spreads 16 KB pieces of all pools' pages over the GPU and is
// bound by HBM (read + write).
//
// Measured: moving 450 MB of pages in 8 pools 160 us (5.6 TB/s read and written,
// floor 140 us); 192 children of 64 rows with 41 MB of last pages 20 us on the
// device (floor 13 us, the index work about 7); freeing over 256 rows 5.4 us.
//
// Ranks are prefix sums and reference counts are integer atomics, so the
// results do not depend on the order in which threads run.
#include <cooperative_groups.h>

#include <algorithm>

#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

namespace cg = cooperative_groups;

constexpr int kPlanCtas = 8;      // portable cluster size
constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kCopyPerSm = 4;     // CTAs per SM: 64 KB of loads in flight (6: 179, 4: 159, 3: 162 us on 8 pools x 1,500 pages of 37 KB)
constexpr int kPieceBytes = kCopyThreads * kCopyUnroll * 16;

struct Pools {
  void* ptr[kMaxPoolsPerLaunch];
  int32_t count;
};

// ---------------------------------------------------------------- copies ----

// Pages to copy: src[i] -> dst[i], the first rows[i] rows of each (whole pages
// when rows is null), i < *count_dev (or `count` when that is null).
template <typename Id>
struct CopyJobs {
  const Id* src;
  const Id* dst;
  const int32_t* rows;
  const int32_t* count_dev;
  int64_t count;
  int64_t num_blocks, row_bytes, page_bytes;
};

template <typename Id>
__global__ void __launch_bounds__(kCopyThreads, kCopyPerSm) page_copy_kernel(const CopyJobs<Id> j, const Pools pools) {
  pdl_wait();  // the jobs come from the launch before this one (returns at once without one)
  const int64_t count = j.count_dev ? *j.count_dev : j.count;
  const int pieces = static_cast<int>((j.page_bytes + kPieceBytes - 1) / kPieceBytes);
  const int64_t piece_bytes = ((j.page_bytes + pieces - 1) / pieces + 15) / 16 * 16;  // equal pieces
  const int64_t tasks = count * pools.count * pieces;
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    // consecutive CTAs: the pieces of one page, then the pools
    const uint32_t per_job = static_cast<uint32_t>(pools.count) * pieces;
    const int64_t i = task / per_job;
    const uint32_t rest = static_cast<uint32_t>(task - i * per_job);
    const int64_t bytes = j.rows ? j.rows[i] * j.row_bytes : j.page_bytes;
    const int64_t src = static_cast<int64_t>(j.src[i]), dst = static_cast<int64_t>(j.dst[i]);
    const int64_t begin = static_cast<int64_t>(rest % pieces) * piece_bytes;
    if (begin >= bytes) continue;
    if (src < 0 || src >= j.num_blocks || dst < 0 || dst >= j.num_blocks) {
      if (threadIdx.x == 0) atomicOr(&g_cascade_device_error, kErrBadBlockId);
      continue;
    }
    uint8_t* base = static_cast<uint8_t*>(pools.ptr[rest / pieces]);
    const uint4* from = reinterpret_cast<const uint4*>(base + src * j.page_bytes + begin) + threadIdx.x;
    uint4* to = reinterpret_cast<uint4*>(base + dst * j.page_bytes + begin) + threadIdx.x;
    const int words = static_cast<int>(min(piece_bytes, bytes - begin) / 16) - threadIdx.x;
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (u * kCopyThreads < words) v[u] = from[u * kCopyThreads];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (u * kCopyThreads < words) to[u * kCopyThreads] = v[u];
  }
}

template <typename Id>
cudaError_t launch_copy(const CopyJobs<Id>& j, void* const* pools, int64_t num_pools, bool after_plan,
                        cudaStream_t stream) {
  const int64_t pieces = (j.page_bytes + kPieceBytes - 1) / kPieceBytes;
  for (int64_t first = 0; first < num_pools; first += kMaxPoolsPerLaunch) {
    Pools args = {};
    args.count = static_cast<int32_t>(std::min<int64_t>(kMaxPoolsPerLaunch, num_pools - first));
    for (int32_t i = 0; i < args.count; ++i) args.ptr[i] = pools[first + i];
    const int64_t tasks = j.count * args.count * pieces;
    if (tasks == 0) continue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(tasks, kNumSMs * kCopyPerSm)));
    cfg.blockDim = dim3(kCopyThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = after_plan && first == 0 ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, page_copy_kernel<Id>, j, args);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// ------------------------------------------------------------ index work ----

// Exclusive prefix sum over the CTA's threads; *total gets the CTA's sum.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* total) {
  __shared__ uint64_t warp_sum[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t s = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t t = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += t;
  }
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  if (warp == 0) {
    uint64_t w = warp_sum[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint64_t t = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += t;
    }
    warp_sum[lane] = w;
  }
  __syncthreads();
  const uint64_t before = warp ? warp_sum[warp - 1] : 0;
  *total = warp_sum[kPlanThreads / 32 - 1];
  __syncthreads();
  return before + s - v;
}

// The half-open run of [0, n) that thread `tid` of cluster rank `rank` owns:
// consecutive per thread, and consecutive over the threads and ranks.
struct Run {
  int64_t begin, end;
};
__device__ __forceinline__ Run own_run(int64_t n, unsigned rank) {
  const int64_t per = (n + kPlanCtas * kPlanThreads - 1) / (kPlanCtas * kPlanThreads);
  const int64_t begin = min(n, (static_cast<int64_t>(rank) * kPlanThreads + threadIdx.x) * per);
  return {begin, min(n, begin + per)};
}

// Sums the CTAs' totals: what the ranks before this one hold, and all of them.
// Ends with no CTA reading another's shared memory only after the next
// cluster barrier.
__device__ __forceinline__ void cluster_totals(cg::cluster_group& cluster, uint64_t* slot, uint64_t* before,
                                               uint64_t* all) {
  const unsigned rank = cluster.block_rank();
  uint64_t b = 0, a = 0;
  for (unsigned r = 0; r < kPlanCtas; ++r) {
    const uint64_t v = *cluster.map_shared_rank(slot, r);
    if (r < rank) b += v;
    a += v;
  }
  *before = b;
  *all = a;
}

__device__ __forceinline__ int64_t pages_of(int64_t len, int64_t block_size) {
  return len > 0 ? (len - 1) / block_size + 1 : 0;  // (no sum that a length near 2^63 makes negative)
}

struct ForkWork {
  int64_t* len;                               // [count]: a child's length, -1 if it cannot be made
  int32_t *fresh, *rank, *src, *dst, *rows;  // [count] each
};

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads)
    fork_plan_kernel(const PageState s, const int64_t* parents, int64_t count, const ForkWork w) {
  pdl_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank();
  __shared__ uint64_t slot;
  const int64_t bs = s.block_size;

  // the parent's length if child i can be made at all (its table holds the length), else -1
  auto length = [&](int64_t i) -> int64_t {
    const int64_t p = parents[i];
    if (p < 0 || p >= s.rows) return -1;
    const int64_t n = s.kv_lens[p];  // (negative: the parent could not be made itself)
    return n >= 0 && pages_of(n, bs) <= s.cols ? n : -1;
  };

  // counts: free pages (high half) and children that need one (low half)
  const Run ids = own_run(s.num_blocks, rank), kids = own_run(count, rank);
  uint64_t mine = 0;
  for (int64_t id = ids.begin; id < ids.end; ++id) {
    const int32_t r = s.refs[id];
    s.refs_out[id] = r;
    mine += static_cast<uint64_t>(r == 0) << 32;
  }
  for (int64_t i = kids.begin; i < kids.end; ++i) {
    const int64_t n = length(i);
    w.len[i] = n;
    mine += n > 0 && n % bs ? 1 : 0;
  }
  uint64_t total, before, all;
  uint64_t at = block_scan(mine, &total);
  if (threadIdx.x == 0) slot = total;
  cluster.sync();
  cluster_totals(cluster, &slot, &before, &all);
  at += before;
  const int64_t num_free = static_cast<int64_t>(all >> 32);

  // ranks: the first `count` free pages, and each child's place among those that need one
  int64_t f = static_cast<int64_t>(at >> 32), k = static_cast<int64_t>(at & 0xffffffffu);
  for (int64_t id = ids.begin; id < ids.end && f < count; ++id)
    if (s.refs[id] == 0) w.fresh[f++] = static_cast<int32_t>(id);
  for (int64_t i = kids.begin; i < kids.end; ++i) {
    const int64_t n = w.len[i];  // this thread's own
    w.rank[i] = static_cast<int32_t>(k);
    k += n > 0 && n % bs ? 1 : 0;
  }
  cluster.sync();

  // one warp per child: its table row, its references, its copy job
  const int lane = threadIdx.x & 31;
  const int64_t warps = kPlanCtas * (kPlanThreads / 32);
  for (int64_t i = static_cast<int64_t>(rank) * (kPlanThreads / 32) + (threadIdx.x >> 5); i < count; i += warps) {
    int64_t n = w.len[i];
    const int64_t parent = parents[i];
    const int32_t place = w.rank[i];
    const bool tail = n > 0 && n % bs;
    if (tail && place >= num_free) n = -1;
    const int64_t full = n > 0 ? n / bs : 0;
    const int32_t* from = s.table + (n >= 0 ? parent : 0) * s.cols;
    const bool job = tail && n > 0;
    const int32_t page = job ? w.fresh[place] : 0;
    for (int64_t c = lane; c < s.cols; c += 32) {
      int32_t id = -1;
      if (c < full) {
        id = from[c];
        if (static_cast<uint64_t>(static_cast<int64_t>(id)) < static_cast<uint64_t>(s.num_blocks))
          atomicAdd(s.refs_out + id, 1);
        else
          atomicOr(&g_cascade_device_error, kErrBadBlockId);
      } else if (c == full && tail && n > 0) {
        id = page;
        s.refs_out[id] = 1;
      }
      s.table_out[i * s.cols + c] = id;
    }
    if (lane == 0) {
      s.lens_out[i] = n;
      w.src[i] = job ? from[full] : 0;
      w.dst[i] = page;
      w.rows[i] = job ? static_cast<int32_t>(n % bs) : 0;
    }
  }
}

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads)
    free_kernel(const PageState s, const int64_t* keep_lens) {
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank();
  const int64_t tid = static_cast<int64_t>(rank) * kPlanThreads + threadIdx.x;
  for (int64_t id = tid; id < s.num_blocks; id += kPlanCtas * kPlanThreads) s.refs_out[id] = s.refs[id];
  cluster.sync();
  const int lane = threadIdx.x & 31;
  const int64_t warps = kPlanCtas * (kPlanThreads / 32);
  for (int64_t r = tid >> 5; r < s.rows; r += warps) {
    const int64_t n = max(s.kv_lens[r], static_cast<int64_t>(0));
    const int64_t keep = min(max(keep_lens[r], static_cast<int64_t>(0)), n);
    const int64_t have = pages_of(n, s.block_size), hold = pages_of(keep, s.block_size);
    for (int64_t c = lane; c < s.cols; c += 32) {
      const int32_t id = s.table[r * s.cols + c];
      if (c >= hold && c < have) {
        if (static_cast<uint64_t>(static_cast<int64_t>(id)) < static_cast<uint64_t>(s.num_blocks))
          atomicSub(s.refs_out + id, 1);
        else
          atomicOr(&g_cascade_device_error, kErrBadBlockId);
      }
      s.table_out[r * s.cols + c] = c < hold ? id : -1;
    }
    if (lane == 0) s.lens_out[r] = keep;
  }
}

struct CompactWork {
  int32_t *live, *holes, *to, *src, *count;  // [num_blocks] x 4, [1]
};

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads)
    compact_plan_kernel(const PageState s, const CompactWork w, int32_t* live_out) {
  pdl_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank();
  __shared__ uint64_t slot[2];
  const Run ids = own_run(s.num_blocks, rank);

  uint64_t mine = 0, total, before, all;
  for (int64_t id = ids.begin; id < ids.end; ++id) mine += s.refs[id] > 0;
  const uint64_t at = block_scan(mine, &total);
  if (threadIdx.x == 0) slot[0] = total;
  cluster.sync();
  cluster_totals(cluster, &slot[0], &before, &all);
  const int64_t n = static_cast<int64_t>(all);  // live pages
  // by rank: the live page ids, and the free ids below n
  int64_t k = static_cast<int64_t>(at + before);
  uint64_t holes = 0;
  for (int64_t id = ids.begin; id < ids.end; ++id) {
    const int32_t r = s.refs[id];
    w.to[id] = static_cast<int32_t>(id);
    s.refs_out[id] = id < n && r > 0 ? r : 0;
    if (r > 0) {
      w.live[k++] = static_cast<int32_t>(id);
    } else if (id < n) {
      w.holes[id - k] = static_cast<int32_t>(id);
      ++holes;
    }
  }
  block_scan(holes, &total);
  if (threadIdx.x == 0) slot[1] = total;
  cluster.sync();
  // as many live pages lie at or past n as there are holes below it: the last ones
  cluster_totals(cluster, &slot[1], &before, &all);
  const int64_t moves = static_cast<int64_t>(all);
  const int64_t tid = static_cast<int64_t>(rank) * kPlanThreads + threadIdx.x;
  for (int64_t i = tid; i < moves; i += kPlanCtas * kPlanThreads) {
    const int32_t src = w.live[n - moves + i], dst = w.holes[i];
    w.src[i] = src;
    w.to[src] = dst;
    s.refs_out[dst] = s.refs[src];
  }
  if (tid == 0) {
    *w.count = static_cast<int32_t>(moves);
    *live_out = static_cast<int32_t>(n);
  }
  cluster.sync();
  const int lane = threadIdx.x & 31;
  for (int64_t r = tid >> 5; r < s.rows; r += kPlanCtas * (kPlanThreads / 32)) {
    const int64_t have = pages_of(s.kv_lens[r], s.block_size);
    for (int64_t c = lane; c < s.cols; c += 32) {
      int32_t id = -1;
      if (c < have) {
        id = s.table[r * s.cols + c];
        if (static_cast<uint64_t>(static_cast<int64_t>(id)) < static_cast<uint64_t>(s.num_blocks))
          id = w.to[id];
        else
          atomicOr(&g_cascade_device_error, kErrBadBlockId);
      }
      s.table_out[r * s.cols + c] = id;
    }
  }
}

}  // namespace

cudaError_t launch_page_copy(void* const* pools, int64_t num_pools, int64_t num_blocks, int64_t page_bytes,
                             const int64_t* src, const int64_t* dst, int64_t count, cudaStream_t stream) {
  const CopyJobs<int64_t> j = {src, dst, nullptr, nullptr, count, num_blocks, page_bytes, page_bytes};
  return launch_copy(j, pools, num_pools, false, stream);
}

size_t page_fork_workspace(int64_t, int64_t count) {
  return static_cast<size_t>(count) * (sizeof(int64_t) + 5 * sizeof(int32_t));
}

cudaError_t launch_page_fork(const PageState& s, void* const* pools, int64_t num_pools, int64_t row_bytes,
                             const int64_t* parents, int64_t count, void* workspace, cudaStream_t stream) {
  int64_t* len = static_cast<int64_t*>(workspace);
  int32_t* w = reinterpret_cast<int32_t*>(len + count);
  const ForkWork work = {len, w, w + count, w + 2 * count, w + 3 * count, w + 4 * count};
  fork_plan_kernel<<<kPlanCtas, kPlanThreads, 0, stream>>>(s, parents, count, work);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const CopyJobs<int32_t> j = {work.src, work.dst, work.rows, nullptr, count, s.num_blocks, row_bytes,
                               row_bytes * s.block_size};
  return launch_copy(j, pools, num_pools, true, stream);
}

cudaError_t launch_page_free(const PageState& s, const int64_t* keep_lens, cudaStream_t stream) {
  free_kernel<<<kPlanCtas, kPlanThreads, 0, stream>>>(s, keep_lens);
  return cudaGetLastError();
}

size_t page_compact_workspace(int64_t num_blocks) {
  return (static_cast<size_t>(num_blocks) * 4 + 1) * sizeof(int32_t);
}

cudaError_t launch_page_compact(const PageState& s, void* const* pools, int64_t num_pools, int64_t row_bytes,
                                int32_t* live_out, void* workspace, cudaStream_t stream) {
  int32_t* w = static_cast<int32_t*>(workspace);
  const int64_t N = s.num_blocks;
  const CompactWork work = {w, w + N, w + 2 * N, w + 3 * N, w + 4 * N};
  compact_plan_kernel<<<kPlanCtas, kPlanThreads, 0, stream>>>(s, work, live_out);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // at most half the pages move: as many as there are free ones below the live count
  const CopyJobs<int32_t> j = {work.src, work.holes, nullptr, work.count, (N + 1) / 2, N, row_bytes * s.block_size,
                               row_bytes * s.block_size};
  return launch_copy(j, pools, num_pools, true, stream);
}

}  // namespace cascade
