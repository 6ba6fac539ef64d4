// Log probabilities of tokens (cascade_token_logprobs).
//
// One pass over a row's logits keeps, per thread, the running maximum m, the sum of
// e = exp(x - m) and of e (x - m): ln p(x) = x - m - ln sum, and the entropy is
// ln sum - (sum of e (x - m)) / sum, differences of small numbers whatever the
// logits' size. The maximum of a thread's batch of 32 (16 in fp32) logits is kept
// in shared memory for the alternatives.
//
// The `top` first entries: with w full warps, the lowest of the warps'
// ceil(top / w)-th largest thread maxima is a bound that at least `top` entries
// reach. The batches whose maximum reaches it are read again (from L2, a few more
// than `top` of them, a lane per entry), their entries that reach it are ordered by
// counting. A bound is a (logit, index) pair, so equal logits need no care but
// where a thread hides very many entries, or fewer are above -inf (or a mask's lowest
// value) than the bound asks of each warp: then the CTA takes one maximum after the
// other (50 entries left of 128,256, 20 alternatives: 4 rows 76 us, 128 rows 656).
// A batch with a -inf is summed twice, and a row whose token is -inf is read by single
// logits: 128 rows without alternatives 40 to 44 us for 14.
//
// Bound by HBM in fp32 (1,500 rows of 128,256 without alternatives: 125 us, 6.2
// TB/s) and by instructions in 16 bits (some ten per logit, one for the special
// function unit: 74 us, 5.2 TB/s); an alternative adds 9 us there, 20 add 14. Few
// rows are shared by a cluster of CTAs, which meet in the first one's shared memory
// (128 rows with 20 alternatives 18.2 us, 4 of 32,000 with 5 8.4).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

namespace cg = cooperative_groups;

constexpr int kVecs = 4;       // vectors of a batch per thread, 32 apart
// Threads of a CTA: 256, and 128 for rows of 16 bits that have a CTA each. Its warps wait for one another to find the
// alternatives, its SM's other CTAs do not: 1,500 rows with one alternative 82 us with 128, 92 with 256, 133 with 512; but a row
// that has eight CTAs is done in 9.1 us with 256 and 10.0 with 128. fp32 rows have HBM to wait for: 125 us with 256, 154 with 128.
// Threads per SM: 768 in 16 bits (1,024 with 64 registers: 94 us for 77), 1,024 in fp32.
template <int kType>
constexpr int kSmThreads = kType == 2 ? 1024 : 768;
constexpr int kMaxCtas = 8;    // per row
constexpr int kSlots = 32;     // of batches per thread whose maxima are kept
constexpr int kList = 1024;    // entries, or batches, that may reach the bound
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int kType>
struct Vec {  // 16 bytes of logits
  static constexpr int kW = kType == 2 ? 4 : 8;
};

template <int kType>
__device__ __forceinline__ float load_one(const void* row, int i) {
  if constexpr (kType == 2) return __ldg(static_cast<const float*>(row) + i);
  const uint16_t b = __ldg(static_cast<const uint16_t*>(row) + i);
  if constexpr (kType == 1) return __half2float(__ushort_as_half(b));
  return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

template <int kType>
__device__ __forceinline__ void unpack(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kType == 2) {
      x[i] = __uint_as_float(w[i]);
    } else if constexpr (kType == 1) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// maximum of a batch; NaN does not count
template <int kType>
__device__ __forceinline__ float batch_max(const uint4 (&v)[kVecs]) {
  if constexpr (kType == 2) {
    float m = __uint_as_float(v[0].x);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      m = fmax3f(m, __uint_as_float(v[i].x), __uint_as_float(v[i].y));
      m = fmax3f(m, __uint_as_float(v[i].z), __uint_as_float(v[i].w));
    }
    return m;
  } else if constexpr (kType == 1) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    __half2 m[4] = {h[0], h[1], h[2], h[3]};
#pragma unroll
    for (int i = 4; i < 4 * kVecs; ++i) m[i & 3] = __hmax2(m[i & 3], h[i]);
    m[0] = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
    return __half2float(__hmax(__low2half(m[0]), __high2half(m[0])));
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    __nv_bfloat162 m[4] = {h[0], h[1], h[2], h[3]};
#pragma unroll
    for (int i = 4; i < 4 * kVecs; ++i) m[i & 3] = __hmax2(m[i & 3], h[i]);
    m[0] = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
    return __bfloat162float(__hmax(__low2bfloat16(m[0]), __high2bfloat16(m[0])));
  }
}

// how many of a batch's logits are above `bar`, which the type holds
template <int kType, int kN>
__device__ __forceinline__ int count_above(const uint4 (&v)[kN], float bar) {
  if constexpr (kType == 2) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i)
      n += (__uint_as_float(v[i].x) > bar) + (__uint_as_float(v[i].y) > bar) + (__uint_as_float(v[i].z) > bar) +
           (__uint_as_float(v[i].w) > bar);
    return n;
  } else if constexpr (kType == 1) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 b = __float2half2_rn(bar);
    __half2 n[2] = {__hgt2(h[0], b), __hgt2(h[1], b)};
#pragma unroll
    for (int i = 2; i < 4 * kN; ++i) n[i & 1] = __hadd2(n[i & 1], __hgt2(h[i], b));
    n[0] = __hadd2(n[0], n[1]);  // (whole numbers up to 32)
    return static_cast<int>(__low2float(n[0]) + __high2float(n[0]));
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 b = __float2bfloat162_rn(bar);
    __nv_bfloat162 n[2] = {__hgt2(h[0], b), __hgt2(h[1], b)};
#pragma unroll
    for (int i = 2; i < 4 * kN; ++i) n[i & 1] = __hadd2(n[i & 1], __hgt2(h[i], b));
    n[0] = __hadd2(n[0], n[1]);
    return static_cast<int>(__low2float(n[0]) + __high2float(n[0]));
  }
}

// -inf (and what lies below -1e38) as a finite number; NaN stays. fp16 has no number that far below all others: there the
// differences are cut (below).
template <int kType>
__device__ __forceinline__ uint4 clamp_low(uint4 v) {
  if constexpr (kType == 0) {
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], __float2bfloat162_rn(-1e38f));
  }
  if constexpr (kType == 2) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(fmax3f_nan(__uint_as_float(w[i]), -1e38f, -1e38f));
  }
  return v;
}

// the largest number of the type below x (x finite or +infinity)
template <int kType>
__device__ __forceinline__ float next_below(float x) {
  if (x == 0.f) return kType == 2 ? __int_as_float(0x80000001) : kType == 1 ? -0x1p-24f : __int_as_float(0x80010000);
  if constexpr (kType == 1) {
    const uint16_t b = __half_as_ushort(__float2half_rn(x));
    return __half2float(__ushort_as_half(static_cast<uint16_t>(x > 0.f ? b - 1 : b + 1)));
  }
  const int step = kType == 2 ? 1 : 0x10000;
  return __int_as_float(x > 0.f ? __float_as_int(x) - step : __float_as_int(x) + step);
}

// A logit's place in the order: larger first, lower index first among equals, a NaN as -inf; never 0, nor all ones.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t make_key(float x, uint32_t v) {
  return (static_cast<uint64_t>(order_bits(x)) << 32) | (0xffffffffu - v);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xffffffffu - static_cast<uint32_t>(k); }

struct Stats {  // of a thread, a CTA, a row
  float m, sum, dot;  // dot: of e log2(e); sums relative to m
  int ahead;
  int nan;
};

// sums relative to the larger maximum
__device__ __forceinline__ void rebase(Stats& s, float m) {
  if (s.m == m) return;
  if (s.m == -INFINITY) {
    s.m = m;  // (nothing but zeros so far)
    return;
  }
  const float d = (s.m - m) * kLog2e, f = ex2(d);  // d <= 0; -inf only if m is +inf: the row is NaN
  s.dot = f == 0.f ? 0.f : f * fmaf(s.sum, d, s.dot);
  s.sum *= f;
  s.m = m;
}
__device__ __forceinline__ void add(Stats& s, Stats o) {
  const float m = fmaxf(s.m, o.m);
  rebase(s, m);
  rebase(o, m);
  s.sum += o.sum, s.dot += o.dot, s.ahead += o.ahead, s.nan |= o.nan;
}

__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

template <int kThreads>
struct Shared {
  static constexpr int kWarps = kThreads / 32;
  float batch_max[kSlots][kThreads];
  uint64_t list[kList];
  uint32_t hits[kList];  // slot, thread
  uint64_t sorted[kMaxTop];
  uint64_t gather[kMaxCtas * kMaxTop];  // the first CTA's: every CTA's `sorted`
  Stats cta[kMaxCtas];                  // the first CTA's: every CTA's sums
  Stats warp[kWarps];
  uint64_t bound[kWarps];
  int count, hit_count;
};

template <int kType, int kThreads>
__global__ void __launch_bounds__(kThreads, kSmThreads<kType> / kThreads) logprobs_kernel(const LogprobsLaunch p) {
  constexpr int kW = Vec<kType>::kW, kWarps = kThreads / 32;
  constexpr int kBatch = kVecs * kW;         // a thread's logits per batch
  constexpr int kSpan = 32 * kVecs;          // a warp's vectors per batch
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared<kThreads>& sh = *reinterpret_cast<Shared<kThreads>*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  cluster.barrier_arrive();  // waited for before the first write to another CTA: all have started by then
  const int64_t n = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, V = static_cast<int>(p.vocab), top = p.top;
  const char* row = static_cast<const char*>(p.logits) + n * p.row_stride * (kType == 2 ? 4 : 2);
  const int64_t token = p.tokens[n];
  const bool given = token >= 0 && token < V;
  // vectors at 16-byte boundaries: vector v holds the entries v kW - shift .. + kW; those at the ends may be cut
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16) / (kType == 2 ? 4 : 2);
  const int vectors = (V + shift + kW - 1) / kW;
  const int batches = (vectors + kSpan - 1) / kSpan;
  const int first = static_cast<int>(static_cast<int64_t>(batches) * rank / ctas);        // this CTA's batches
  const int last = static_cast<int>(static_cast<int64_t>(batches) * (rank + 1) / ctas);
  const int per_slot = ((last - first + kWarps - 1) / kWarps + kSlots - 1) / kSlots;
  const float mine = given ? load_one<kType>(row, static_cast<int>(token)) : INFINITY;
  const uint64_t key = given ? make_key(mine, static_cast<uint32_t>(token)) : ~0ull;
  // The entries ahead of the token: those above its logit, and its equals before it, which are above the next lower number.
  // (For a logit of -inf or NaN, equal here, by their keys.)
  const float above = given ? mine : INFINITY, above_before = given ? next_below<kType>(mine) : INFINITY;
  const int token_batch = given ? static_cast<int>((token + shift) / (kSpan * kW)) : -1;
  const int at = given ? static_cast<int>(token) : 0;
  const bool odd = given && !(mine > -INFINITY);
  const int whole_from = shift > 0, whole_to = (V + shift) / (kSpan * kW);  // batches of whole vectors alone

  const uint4* vecs = reinterpret_cast<const uint4*>(row - shift * (16 / kW));
  auto index_of = [&](int v, int j) { return (v + j / kW * 32) * kW - shift + j % kW; };  // entry j of a thread's batch from v on

  // ------------------------------------------------------------- the pass
  Stats s = {-INFINITY, 0.f, 0.f, 0, 0};
  int best_at = first + warp;  // batch of the maximum
  float slot_max = -INFINITY;
  int slot = 0, in_slot = 0;
  auto note = [&](float most, int b) {
    if (most > s.m) {
      rebase(s, most);
      best_at = b;
    }
    slot_max = fmaxf(slot_max, most);
    if (++in_slot == per_slot) {
      sh.batch_max[slot++][threadIdx.x] = slot_max;
      slot_max = -INFINITY, in_slot = 0;
    }
  };
  // Batches that the row's ends cut, with logits of any size: sums of e and e y, y = (x - m) log2(e).
  auto careful = [&](int b) {
    const int v = b * kSpan + lane;
    float most = -INFINITY;
    auto load = [&](int q, float (&x)[kW]) {
#pragma unroll
      for (int j = 0; j < kW; ++j) {
        const int i = index_of(v, q * kW) + j;
        x[j] = i >= 0 && i < V ? load_one<kType>(row, i) : -INFINITY;
      }
    };
#pragma unroll 1
    for (int q = 0; q < kVecs; ++q) {
      float x[kW];
      load(q, x);
#pragma unroll
      for (int j = 0; j < kW; ++j) {
        const int i = index_of(v, q * kW) + j;
        most = fmaxf(most, x[j]);
        s.ahead += odd ? i >= 0 && i < V && make_key(x[j], static_cast<uint32_t>(i)) > key : x[j] > (i < at ? above_before : above);
      }
    }
    note(most, b);
    const float neg = s.m == -INFINITY ? 0.f : -s.m;
#pragma unroll 1
    for (int q = 0; q < kVecs; ++q) {
      float x[kW];
      load(q, x);
#pragma unroll
      for (int j = 0; j < kW; ++j) {
        const float y = fmaxf((x[j] + neg) * kLog2e, -200.f), e = ex2(y);  // (2^-200 is 0 next to the sum's 1)
        s.sum += x[j] != x[j] ? x[j] : e, s.dot = fmaf(e, y, s.dot);
      }
    }
  };
  // The others, with a maximum below 1e37 in size: a finite number can stand in for -inf (0 times infinity would be NaN).
  auto batch = [&](const uint4 (&raw)[kVecs], int b) {
    const float most = batch_max<kType>(raw), bar = b < token_batch ? above_before : above;
    const bool ahead = __any_sync(0xffffffffu, most > bar);
    if (!(fabsf(fmaxf(s.m, most)) < 1e37f)) return false;
    note(most, b);
    if (b != token_batch) {
      if (ahead) s.ahead += count_above<kType>(raw, bar);
    } else {
#pragma unroll
      for (int q = 0; q < kVecs; ++q) {
        const int i = index_of(b * kSpan + lane, q * kW);
        const uint4 one[1] = {raw[q]};
        s.ahead += count_above<kType>(one, i + kW <= at ? above_before : above);
        if (i <= at && at < i + kW)  // the equals before the token in its own vector
          for (int j = i; j < at; ++j) s.ahead += load_one<kType>(row, j) == mine;
      }
    }
    const float neg = -s.m;
    float sum = 0.f, dot = 0.f;
    auto sums = [&](auto low) {
      float sum0 = 0.f, sum1 = 0.f, dot0 = 0.f, dot1 = 0.f;
#pragma unroll
      for (int q = 0; q < kVecs; ++q) {
        float x[kW];
        unpack<kType>(low ? clamp_low<kType>(raw[q]) : raw[q], x);
#pragma unroll
        for (int j = 0; j < kW; j += 2) {
          float y0 = x[j], y1 = x[j + 1];
          fadd2(y0, y1, neg, neg);
          fmul2(y0, y1, kLog2e);
          if constexpr (kType == 1 && decltype(low)::value) y0 = fmax3f_nan(y0, -1e30f, -1e30f), y1 = fmax3f_nan(y1, -1e30f, -1e30f);
          const float e0 = ex2(y0), e1 = ex2(y1);
          fadd2(sum0, sum1, e0, e1);
          ffma2(dot0, dot1, e0, e1, y0, y1);
        }
      }
      sum = sum0 + sum1, dot = dot0 + dot1;
    };
    // In 16 bits, where instructions count, first as if there were no -inf; then 0 times infinity is a NaN. (In fp32, 130 us for
    // 1,500 rows, the second form costs registers: 173.)
    if constexpr (kType != 2) sums(std::false_type());
    if (kType == 2 || dot != dot) sums(std::true_type());
    s.sum += sum, s.dot += dot;
    return true;
  };
  int b = first + warp;
  const int stop = odd ? b : min(last, whole_to);
  for (; b < last && (odd || b < whole_from); b += kWarps) careful(b);
  uint4 next[kVecs];
  auto read = [&](int b) {
#pragma unroll
    for (int q = 0; q < kVecs; ++q) next[q] = __ldg(vecs + b * kSpan + q * 32 + lane);
  };
  if (b < stop) read(b);
  for (; b < stop; b += kWarps) {
    uint4 raw[kVecs];
#pragma unroll
    for (int q = 0; q < kVecs; ++q) raw[q] = next[q];
    if (b + kWarps < stop) read(b + kWarps);
    if (!batch(raw, b)) careful(b);
  }
  for (; b < last; b += kWarps) careful(b);
  if (in_slot > 0) sh.batch_max[slot++][threadIdx.x] = slot_max;
  s.nan = s.sum != s.sum;
  // the thread's maximum, with an index that it is not behind
  const uint64_t best =
      best_at >= last ? 0 : make_key(s.m, static_cast<uint32_t>(min(V - 1, max(0, index_of(best_at * kSpan + lane, kBatch - 1)))));

  // ------------------------------------------------------------- the sums
  const float thread_max = s.m;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    Stats o;
    o.m = __shfl_xor_sync(0xffffffffu, s.m, d);
    o.sum = __shfl_xor_sync(0xffffffffu, s.sum, d);
    o.dot = __shfl_xor_sync(0xffffffffu, s.dot, d);
    o.ahead = __shfl_xor_sync(0xffffffffu, s.ahead, d);
    o.nan = __shfl_xor_sync(0xffffffffu, s.nan, d);
    add(s, o);
  }
  if (lane == 0) sh.warp[warp] = s;
  if (top == 0) __syncthreads();

  // ------------------------------------------------------------- the alternatives
  if (top > 0) {
    // warps whose first batch is whole: all lanes have entries (a cut vector has one at least)
    const int full = min(kWarps, max(0, min(last, vectors / kSpan) - first));
    // the lowest of the warps' nth largest, nth = top / warps, or (where that leaves too many: equal logits) the highest of
    // their `top`-th
    auto find_bound = [&](bool one) {
      const int nth = one ? top : full > 0 ? (top + full - 1) / full : 0;
      uint64_t k = best, at = 0;
      for (int i = 0; i < nth; ++i) {
        at = warp_max(k);
        if (k == at) k = 0;
      }
      if (lane == 0) sh.bound[warp] = warp < full ? at : one ? 0 : ~0ull;
      if (threadIdx.x == 0) sh.count = sh.hit_count = 0;
      __syncthreads();
      uint64_t bound = sh.bound[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) bound = one ? max(bound, sh.bound[w]) : min(bound, sh.bound[w]);
      return full > 0 ? bound : 0;
    };
    int count = 0;
    for (int round = 0; round < 2; ++round) {
      const uint64_t bound = find_bound(round > 0);
      const uint32_t bound_hi = static_cast<uint32_t>(bound >> 32);
      if (order_bits(thread_max) >= bound_hi) {
        uint32_t reach = 0;
#pragma unroll 8
        for (int i = 0; i < slot; ++i) reach |= static_cast<uint32_t>(order_bits(sh.batch_max[i][threadIdx.x]) >= bound_hi) << i;
        int to = atomicAdd(&sh.hit_count, __popc(reach));
        for (; reach; reach &= reach - 1, ++to)
          if (to < kList) sh.hits[to] = static_cast<uint32_t>(__ffs(reach) - 1) << 16 | threadIdx.x;
      }
      __syncthreads();
      const int hits = sh.hit_count;
      if (hits <= kList) {
        // a lane per entry (fp32: two batches at once), a warp's next loads under way before it looks at these
        constexpr int kAtOnce = 32 / kBatch, kAhead = 4;
        for (int i = warp * kAtOnce + lane / kBatch; i < hits; i += kWarps * kAtOnce * kAhead) {
          int b[kAhead], v[kAhead];
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const uint32_t hit = i + k * kWarps * kAtOnce < hits ? sh.hits[i + k * kWarps * kAtOnce] : 0xffffu;
            const int who = hit & 0xffff;
            b[k] = who == 0xffff ? last : first + (who >> 5) + static_cast<int>(hit >> 16) * per_slot * kWarps;
            v[k] = who & 31;
          }
          for (int j = 0; j < per_slot; ++j) {
            float x[kAhead];
            int idx[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
              idx[k] = b[k] < last ? index_of(b[k] * kSpan + v[k], lane % kBatch) : -1;
              if (idx[k] >= V) idx[k] = -1;
              x[k] = idx[k] >= 0 ? load_one<kType>(row, idx[k]) : 0.f;
              b[k] += kWarps;
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
              const uint64_t a = make_key(x[k], static_cast<uint32_t>(idx[k]));
              if (idx[k] >= 0 && a >= bound) {
                const int to = atomicAdd(&sh.count, 1);
                if (to < kList) sh.list[to] = a;
              }
            }
          }
        }
      } else if (threadIdx.x == 0) {
        sh.count = kList + 1;
      }
      __syncthreads();
      count = sh.count;
      if (count <= kList) break;
      __syncthreads();  // (all have read the count)
    }
    if (count <= kList) {
      for (int i = threadIdx.x; i < max(count, top); i += kThreads) {
        if (i >= count) {
          sh.sorted[i] = 0;  // (fewer entries than `top` in this CTA's part)
          continue;
        }
        const uint64_t a = sh.list[i];
        int before = 0;
#pragma unroll 4
        for (int j = 0; j < count; ++j) before += sh.list[j] > a;
        if (before < top) sh.sorted[before] = a;
      }
    } else {
      // a thread hides more than the list holds: one maximum after the other
      uint64_t limit = ~0ull;
      for (int k = 0; k < top; ++k) {
        uint64_t most = 0;
        for (int i = first * kSpan * kW + static_cast<int>(threadIdx.x); i < last * kSpan * kW; i += kThreads) {
          const int idx = i - shift;
          if (idx < 0 || idx >= V) continue;
          const uint64_t a = make_key(load_one<kType>(row, idx), static_cast<uint32_t>(idx));
          if (a < limit && a > most) most = a;
        }
        most = warp_max(most);
        if (lane == 0) sh.bound[warp] = most;
        __syncthreads();
        limit = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) limit = max(limit, sh.bound[w]);
        if (threadIdx.x == 0) sh.sorted[k] = limit;
        __syncthreads();
      }
    }
    __syncthreads();
  }

  // ------------------------------------------------------------- the row
  if (warp == 0) {
    s = sh.warp[0];
    for (int w = 1; w < kWarps; ++w) add(s, sh.warp[w]);
  }
  cluster.barrier_wait();
  if (ctas > 1) {
    Shared<kThreads>& root = *cluster.map_shared_rank(&sh, 0);
    if (threadIdx.x == 0) root.cta[rank] = s;
    if (threadIdx.x < top) root.gather[rank * top + threadIdx.x] = sh.sorted[threadIdx.x];
    cluster.sync();
    if (rank > 0) return;
    if (warp == 0) {
      s = sh.cta[0];
      for (int c = 1; c < ctas; ++c) add(s, sh.cta[c]);
    }
    const int all = ctas * top;
    for (int i = threadIdx.x; i < all; i += kThreads) {
      const uint64_t a = sh.gather[i];
      int before = 0;
      for (int j = 0; j < all; ++j) before += sh.gather[j] > a;
      if (a != 0 && before < top) sh.sorted[before] = a;
    }
    __syncthreads();
  }
  if (warp == 0) {
    const bool nan = s.nan || !(s.m < INFINITY) || s.m == -INFINITY;
    const float norm = nan ? __int_as_float(0x7fffffff) : logf(s.sum);
    if (lane == 0) {
      p.logprob[n] = given ? (mine - s.m) - norm : -INFINITY;
      p.entropy[n] = norm - s.dot / s.sum * kLn2;
      p.rank[n] = given ? s.ahead : -1;
    }
    if (lane < top) {
      const uint64_t a = sh.sorted[lane];
      const uint32_t idx = key_index(a);
      p.top_tokens[n * top + lane] = idx;
      p.top_logprobs[n * top + lane] = (load_one<kType>(row, static_cast<int>(idx)) - s.m) - norm;
    }
  }
}

}  // namespace

template <int kType, int kThreads>
static cudaLaunchConfig_t config(int64_t rows, int ctas, cudaStream_t stream, cudaLaunchAttribute& attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared<kThreads>);
  cfg.stream = stream;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cfg;
}

template <int kType, int kThreads>
static cudaError_t launch(const LogprobsLaunch& p, int ctas, cudaStream_t stream) {
  auto kern = logprobs_kernel<kType, kThreads>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), sizeof(Shared<kThreads>));
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = config<kType, kThreads>(p.rows, ctas, stream, attr);
  return cudaLaunchKernelEx(&cfg, kern, p);
}

// Rows that run at once with `ctas` = 2, 4 or 8 CTAs each. Fewer than the SMs hold: a cluster lies within a part of the GPU whose
// SMs need not divide by it (16 bits: 48 rows of 8, 104 of 4; one more takes a second round, 16.5 us for 13.2).
template <int kType>
static int resident_rows(int ctas) {
  static std::atomic<int> known[kMaxCtas + 1];
  int n = known[ctas].load(std::memory_order_relaxed);
  if (n == 0) {
    auto kern = logprobs_kernel<kType, 256>;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = config<kType, 256>(1, ctas, nullptr, attr);
    if (ensure_smem_limit(reinterpret_cast<const void*>(kern), sizeof(Shared<256>)) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess)
      return 0;
    known[ctas].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int kType>
static cudaError_t launch(const LogprobsLaunch& p, cudaStream_t stream) {
  // as many CTAs per row as run at once, with a batch for each of their warps
  constexpr int kMost = kSmThreads<kType> / 256 * kNumSMs, kSpan = 256 * kVecs * Vec<kType>::kW;
  int ctas = 1;
  while (ctas < kMaxCtas && p.rows * ctas * 2 <= kMost && p.vocab >= 2 * ctas * kSpan && p.rows <= resident_rows<kType>(2 * ctas))
    ctas *= 2;
  if (kType != 2 && ctas == 1) return launch<kType, 128>(p, 1, stream);
  return launch<kType, 256>(p, ctas, stream);
}

cudaError_t launch_token_logprobs(const LogprobsLaunch& p, cudaStream_t stream) {
  return p.dtype == 2 ? launch<2>(p, stream) : p.dtype == 1 ? launch<1>(p, stream) : launch<0>(p, stream);
}

}  // namespace cascade
