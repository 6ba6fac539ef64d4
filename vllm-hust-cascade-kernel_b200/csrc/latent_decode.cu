// Latent attention, absorbed form (cascade_latent_decode), on the tensor cores,
// for more than 32 query rows per request (latent_decode_few.cu has the rest).
//
// For a query row x (576 values) of a request: s_t = scale <x, c_t> over the
// request's cache rows c_t (576 values), out = sum_t softmax(s)_t c_t[0:512].
// A cache row of 1,152 bytes meets 2 x 1,088 flops per query row, so 128 rows
// (one token x 128 heads) sit where the tensor cores and HBM take equally
// long (0.168 against 0.179 ns per cache row and GPU), and fewer rows are
// bound by HBM: the kernel has to keep both busy at once.
//
// A cluster of two CTAs computes one tile of 128 query rows (the request's
// [token x head] rows in memory order) against 64 cache rows at a time:
//   * the output of 128 x 512 fp32 would fill a CTA's tensor memory, so each CTA
//     owns 256 of the 512 output columns (256 TMEM columns);
//   * each CTA computes the scores of its own 32 of the 64 cache rows for all
//     128 query rows, so no score is computed twice;
//   * the row maxima of a tile are exchanged (st.async), so both CTAs scale by
//     the same maximum, and each CTA's half of P (128 x 32, 16-bit) is copied
//     to the other by the bulk-copy engine. One way takes 410 and 590 cycles
//     (remote stores with a release held the softmax warps for about 4,000 a
//     tile), so three tiles are in flight: scores of tile n + 2, maxima of
//     n + 1, exponentials and P of n.
// Per 64 cache rows a CTA loads its own 32 rows in full (keys, and its columns
// of V) and its columns of the other 32: 52 KB for 36 KB from HBM.
// Six of the query tile's nine groups of 64 dims live in TMEM (192 columns),
// three in shared memory: with A in shared memory a 128 x 32 x 16 MMA takes 43
// cycles (A's 4 KB), in TMEM 19.
//
// Softmax: running maximum m in the log2 domain that moves only when a score
// exceeds it by more than 2^8 (the exponentials stay below 256, exact in
// relative terms in both types), so the accumulator is rescaled rarely. P is
// rounded to the inputs' type, which the second product needs; the row's sum is
// of the unrounded exponentials, in fp32.
//
// Work: the 64-row tiles of all (request, row tile) units, concatenated, are
// cut into one run of equal cost per cluster, computed on the device from the lengths.
// A unit cut by a run boundary leaves fp32 partials that a second, dependent
// launch merges in run order; all others are written directly.
//
// Measured (128 requests x 128 heads over 1,500-8,200 tokens: 754 MB, 174
// GFLOP, floor 117 us): 250 us per call in a loop, 3.0 TB/s and 695 TFLOP/s; 210
// replayed in a graph. A tile takes about
// 2,100 cycles of a pair; its MMAs take 1,430 (960 for the scores, 43-cycle
// shared-memory and 19-cycle TMEM steps; 530 for P V, less overlap), its 52 KB
// per SM from L2 1,390 at the measured 37 bytes per clock and SM. The rest is
// the chain P -> other CTA -> P V -> buffer free, two deep: with neither MMAs nor
// loads the waits alone take 1,600 cycles a tile. A third P buffer would have to
// come out of the ring of own columns, whose fourth stage is worth more (three
// stages 296 us, four 231, in a graph); fetching the keys into L2 ahead of their load changes nothing.
//
// Warps: 0-7 softmax (two threads per row = TMEM lane, 16 of the CTA's 32 cache
// rows each: with one, its 1,900 cycles a tile set the pace) and output, 8-11 query
// tile, 12 keys (TMA), 13 MMA issue (one issuer: the two kinds of MMA
// interleaved from two take a fifth longer), 14 the other CTA's rows (TMA).
#include <algorithm>
#include <atomic>

#include "latent_decode.cuh"

namespace cascade {
namespace {

constexpr int kRows = 128;     // query rows per tile
constexpr int kTok = 64;       // cache rows per tile
constexpr int kHalfTok = 32;   // per CTA
// What going from one unit to the next costs, in tiles (about 10,000 cycles), for cutting the work into equal runs.
// In a graph, 24 requests x 4 tokens x 128 heads over 4-5,003 tokens: 0 137 us, 4, 5 and 6 all 94 to 105 from run to
// run; 128 requests x 128 heads over 1,500-8,200 tokens: 0 217 us, 4 210.9, 5 210.5, 6 211.3.
constexpr int kSetup = 5;
constexpr int kThreads = 15 * 32;
constexpr int kMaxClusters = kNumSMs / 2;

constexpr int kStagesA = 2, kStagesB = 4, kStagesC = 2;  // keys outside the own columns; own columns; the other rows
constexpr int kPBuf = 2;
static_assert(kStagesA == 2 && kStagesB == 4 && kStagesC <= 4, "the barriers that free the stages");
constexpr int kGroup = kHalfTok * 128;    // 32 cache rows x 64 dims
constexpr int kBytesA = 5 * kGroup;       // keys outside the CTA's own columns
constexpr int kBytesV = 4 * kGroup;       // the CTA's own columns
constexpr int kQGroup = kRows * 128;      // 128 query rows x 64 dims
constexpr int kQTmem = 6;                 // groups of 64 dims in TMEM, the last three in shared memory
constexpr int kPPart = kRows * 16 * 2;        // P of 16 cache rows: one K step of the second product
constexpr int kOffQ = 0;
constexpr int kOffP = kOffQ + (9 - kQTmem) * kQGroup;
constexpr int kOffA = kOffP + kPBuf * 4 * kPPart;
constexpr int kOffB = kOffA + kStagesA * kBytesA;
constexpr int kOffC = kOffB + kStagesB * kBytesV;
constexpr int kTiles = kOffC + kStagesC * kBytesV;  // bytes from the first 1 KB boundary after Aux

constexpr uint32_t kColO = 0, kColQ = 256, kColS = 448;  // TMEM columns: O 256, Q 192, S 2 x 32

struct __align__(16) Aux {
  // What the four threads of a row (two per CTA) tell one another, in both CTAs: their maxima of a tile, their sums of
  // a piece. Three slots: a thread tells the maximum of tile n + 3 when its scores are there; they were computed after
  // P V of tile n, which needed the partners' P of tile n, written after they had read exchange n.
  union {
    float shared[3][4][kRows];
    int64_t scan[2][kThreads / 32];  // find_run only
  };
  // One commit per MMA batch serves all that wait for it (a commit costs the
  // tensor pipe 60 to 100 cycles): s_full[it % 2] = scores of tile it done (the
  // softmax, and the keys' next load), pv_done[it % 4] = P V of tile it done in
  // both CTAs (P, own columns, other rows). A waiter is never two phases behind:
  // the next phase needs what it is about to do.
  // What an MMA batch needs meets on one barrier too (a wait that is over costs
  // 120 cycles): kv_full[it % 4] = tile it's keys loaded, and its score buffer
  // read by the eight softmax warps; p_full[it % 2] = P of both CTAs, and the
  // other CTA's rows loaded. The rows of a tile that ends in unused cache rows
  // come over tail_full[it % 2] instead: the softmax clears those rows first.
  uint64_t kv_full[kStagesB], p_full[kPBuf], tail_full[kPBuf], s_full[2], pv_done[4], x_full[3];
  uint64_t q_full, q_empty, o_empty;
  uint64_t qs_full[3], qs_empty[3];
  uint64_t stall, drain;
  uint32_t tmem_base;
  Sched sched;
};
constexpr int kStaticBytes = 32;  // the wait state comes first
constexpr int kSmemBytes = (kStaticBytes + static_cast<int>(sizeof(Aux)) + 1023) / 1024 * 1024 + kTiles - kStaticBytes;
static_assert(kSmemBytes + kStaticBytes <= 227 * 1024, "shared memory per CTA");

struct Params {
  LatentDecodeLaunch L;
  CUtensorMap map4, map1;  // boxes of 64 dims x kR cache rows x 4 groups (1 group)
  CUtensorMap map_q;       // 64 dims x 128 query rows
  Partials parts;
};

// Loads one box column of a tile: kR cache rows x groups per load, for the 32
// rows that start at cache row `first`. The warp's lanes hold the pool rows of
// the next loads (`rows`, refilled every 32 loads).
template <int kR>
struct PageRows {
  static constexpr int kPer = kHalfTok / kR;  // loads (pages at most) per tile
  const LatentDecodeLaunch& p;
  const int32_t* bt;
  int base, pages, half, row;

  __device__ PageRows(const LatentDecodeLaunch& l, int half_) : p(l), half(half_) {}
  // tiles [t, ...) of request b with kv valid cache rows
  __device__ __forceinline__ void start(int b, int kv) {
    bt = p.block_table + static_cast<int64_t>(b) * p.block_cols;
    pages = (kv + p.block_size - 1) / p.block_size;
    base = -(1 << 30);
  }
  // pool row of load i of tile t (called by the whole warp)
  __device__ __forceinline__ int get(int t, int i, int lane) {
    constexpr int kTiles = 32 / kPer;
    if (t >= base + kTiles || t < base) {
      base = t;
      const int tok = (t + lane / kPer) * kTok + half * kHalfTok + (lane % kPer) * kR;
      const int page = tok / p.block_size, oob = max(1, p.num_blocks * p.block_size);
      row = page < pages ? paged_row(bt[page], tok, p.block_size, p.num_blocks, oob) : oob;
    }
    return __shfl_sync(0xffffffffu, row, (t - base) * kPer + i);
  }
};

// Writes columns [32 g0, 32 g1) of the CTA's 256 of a piece's output, 32 rows per
// warp: divided by the sums to `out` when the piece is its whole unit, else as
// an fp32 partial. They go through shared memory, so that a store instruction
// writes whole sectors: kWide, 128 bytes per row at a time (4 KB of `stage`,
// 16-byte chunk q of row r at q ^ (r % 8)), else 32 (1 KB, half h at
// h ^ (r / 4 % 2)); no bank conflicts either way. `released` (if given) gets an
// arrival per warp once the accumulator has been read.
template <bool kFp16, bool kWide>
__device__ __forceinline__ void write_rows(const Params& P, const Walk<kRows, kTok, kSetup>& x, int cluster, int c, float inv, uint32_t tmem,
                                           uint8_t* stage, int g0, int g1, uint64_t* released) {
  const LatentDecodeLaunch& p = P.L;
  const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3;
  const bool whole = x.starts && x.ends;
  const int row0 = x.mt * kRows + quarter * 32;  // this warp's first row of the unit
  const int64_t grow0 = x.tok * p.num_heads + row0;
  const int rows = static_cast<int>(min(static_cast<int64_t>(32), min(static_cast<int64_t>(x.q) * p.num_heads - row0,
                                                                      p.num_tokens * p.num_heads - grow0)));
  const int64_t slot = 2 * cluster + (x.starts ? 1 : 0);
  uint8_t* dst = whole ? static_cast<uint8_t*>(p.out) + grow0 * (kLatentDim * 2) + 512 * c
                       : reinterpret_cast<uint8_t*>(P.parts.o) + (slot * kRows + quarter * 32) * (kLatentDim * 4) + 1024 * c;
  const int pitch = whole ? kLatentDim * 2 : kLatentDim * 4;
  constexpr int kPerRow = kWide ? 8 : 2;  // 16-byte chunks staged per row
  auto place = [&](int chunk) -> uint4* {
    const int swap = kWide ? lane & 7 : (lane >> 2) & 1;
    return reinterpret_cast<uint4*>(stage + lane * (kPerRow * 16) + ((chunk ^ swap) << 4));
  };
  auto flush = [&](int part) {
    __syncwarp();
#pragma unroll
    for (int q = 0; q < kPerRow; ++q) {
      const int rr = q * (32 / kPerRow) + lane / kPerRow, chunk = lane % kPerRow;
      const int swap = kWide ? rr & 7 : (rr >> 2) & 1;
      const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * (kPerRow * 16) + ((chunk ^ swap) << 4));
      if (rr < rows)
        *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(rr) * pitch + part * (kPerRow * 16) + chunk * 16) = v;
    }
    __syncwarp();
  };
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    uint32_t o[32];
    tmem_ld_32x32b_x32(tmem + kColO + g * 32, o);
    tmem_wait_ld();
    if (released && g + 1 == g1) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(released);
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = inv == 0.f ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
    if (whole) {  // 64 bytes per row
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        auto two = [&](int e) { return pack2<kFp16>(__uint_as_float(o[e]), __uint_as_float(o[e + 1])); };
        const int e = q * 8;
        *place(kWide ? (g & 1) * 4 + q : q & 1) = make_uint4(two(e), two(e + 2), two(e + 4), two(e + 6));
        if (!kWide && (q & 1)) flush(g * 2 + (q >> 1));
      }
      if (kWide && (g & 1)) flush(g >> 1);
    } else {  // 128 bytes per row
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        *place(kWide ? q : q & 1) = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        if (!kWide && (q & 1)) flush(g * 4 + (q >> 1));
      }
      if (kWide) flush(g);
    }
  }
}

// Four groups of 64 dims of kR cache rows, each group kGroup bytes apart: at once
// when a page gives all 32 rows, group by group when two pages share them.
template <int kR>
__device__ __forceinline__ void load_groups(uint8_t* dst, const Params& P, uint64_t* bar, int row, int group) {
  if constexpr (kR == kHalfTok) {
    tma_load_3d(dst, &P.map4, bar, 0, row, group);
  } else {
#pragma unroll
    for (int g = 0; g < 4; ++g) tma_load_3d(dst + g * kGroup, &P.map1, bar, 0, row, group + g);
  }
}

template <bool kFp16, int kR>
__global__ void __launch_bounds__(kThreads, 1) latent_decode_kernel(const __grid_constant__ Params P) {
  pdl_launch_dependents();
  const LatentDecodeLaunch& p = P.L;
  extern __shared__ uint8_t smem_raw[];
  Aux* aux = reinterpret_cast<Aux*>(smem_raw);
  uint8_t* smem = smem_raw + sizeof(Aux) + ((0u - (smem_u32(smem_raw) + static_cast<uint32_t>(sizeof(Aux)))) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c = static_cast<int>(cluster_cta_rank());
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (tid == 0) {
    cta_wait_init(static_cast<uint64_t>(p.wait_limit_us) * 1000);
    for (int s = 0; s < kStagesB; ++s) mbar_init(&aux->kv_full[s], 9);
    for (int s = 0; s < 3; ++s) mbar_init(&aux->x_full[s], 1);
    for (int s = 0; s < kPBuf; ++s) mbar_init(&aux->p_full[s], 9), mbar_init(&aux->tail_full[s], 1), mbar_init(&aux->s_full[s], 1);
    for (int s = 0; s < 4; ++s) mbar_init(&aux->pv_done[s], 2);
    mbar_init(&aux->q_full, 128);
    mbar_init(&aux->q_empty, 1);
    mbar_init(&aux->o_empty, 8);
    for (int s = 0; s < 3; ++s) mbar_init(&aux->qs_full[s], 1), mbar_init(&aux->qs_empty[s], 4);
    mbar_init(&aux->stall, 1);
    mbar_init(&aux->drain, 1);
    fence_mbar_init();
  }
  if (tid == 32) {
    tma_prefetch_desc(&P.map_q);
    tma_prefetch_desc(&P.map4);
    tma_prefetch_desc(&P.map1);
  }
  if (warp == 13) {
    tmem_alloc(&aux->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  find_run<kRows, kTok, kSetup, kThreads>(p, P.parts.row_info, cluster, clusters, aux->scan, &aux->sched);  // (with CTA barriers)
  tc_fence_after();
  // Both CTAs' barriers are initialised once this barrier is passed; only the roles that reach into the other CTA
  // wait for it first, the loads start before.
  cluster_arrive();
  const bool remote = warp < 8 || warp == 13;
  if (remote) cluster_wait();
  const uint32_t tbase = aux->tmem_base;
  Walk<kRows, kTok, kSetup> w(p, aux->sched);

  if (warp == 12 || warp == 14) {
    // ------------------------------------------------------------ producers
    // 12: this CTA's 32 rows; 14: the other CTA's 32 rows, own columns
    const bool keys = warp == 12;
    PageRows<kR> rows(p, keys ? c : 1 - c);
    int it = 0;
    bool live = true;
    while (live && w.next()) {
      rows.start(w.b, w.kv);
      for (int t = w.t0; t < w.t0 + w.n; ++t, ++it) {
        int y[PageRows<kR>::kPer];
#pragma unroll
        for (int i = 0; i < PageRows<kR>::kPer; ++i) y[i] = rows.get(t, i, lane);
        const int stages = keys ? kStagesB : kStagesC, st = it % stages;
        live = it < stages || mbar_wait_warp(&aux->pv_done[(it - stages) & 3], ((it - stages) >> 2) & 1);
        if (keys) live = live && (it < 2 || mbar_wait_warp(&aux->s_full[it & 1], ((it >> 1) - 1) & 1));
        if (!live) break;
        const bool tail = !keys && (t + 1) * kTok > w.kv;
        if (lane == 0) {
          uint64_t* full = keys ? &aux->kv_full[st] : tail ? &aux->tail_full[it & 1] : &aux->p_full[it & 1];
          uint8_t* dst = smem + (keys ? kOffB : kOffC) + st * kBytesV;
          uint8_t* dsta = smem + kOffA + (it & 1) * kBytesA;
          mbar_arrive_expect_tx(full, keys ? kBytesA + kBytesV : kBytesV);
          if (tail) mbar_arrive(&aux->p_full[it & 1]);
#pragma unroll
          for (int i = 0; i < PageRows<kR>::kPer; ++i) {
            const int at = i * kR * 128;  // 32 rows per group, from one page or two
            if (keys) {
              load_groups<kR>(dsta + at, P, full, y[i], 4 * (1 - c));
              tma_load_3d(dsta + 4 * kGroup + at, &P.map1, full, 0, y[i], 8);
            }
            load_groups<kR>(dst + at, P, full, y[i], 4 * c);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 13) {
    // ----------------------------------------------------------- MMA issuer
    // the whole warp walks and waits; one elected lane issues. Scores run two
    // tiles ahead of P V, within a piece.
    const uint32_t idesc_s = make_idesc_f16(kRows, kHalfTok, kFp16 ? 0u : 1u, 0, 0);
    const uint32_t idesc_pv = make_idesc_f16(kRows, 256, kFp16 ? 0u : 1u, 0, 1);
    const uint32_t tm = uniform(tbase), rank = uniform(static_cast<uint32_t>(c)), s0 = uniform(smem_u32(smem));
    const uint64_t dq = make_smem_desc(s0 + kOffQ, 16, 1024, 2);
    int pieces = 0;
    auto scores = [&](int it, bool first, bool last) -> bool {
      const uint32_t u = uniform(it), sa = u & 1, sb = u & 3;
      if ((first && !mbar_wait_warp(&aux->q_full, pieces & 1)) || !mbar_wait_warp(&aux->kv_full[sb], (u >> 2) & 1))
        return false;
      tc_fence_after();
      const uint64_t da = make_smem_desc(s0 + kOffA + sa * kBytesA, 16, 1024, 2);
      const uint64_t db = make_smem_desc(s0 + kOffB + sb * kBytesV, 16, 1024, 2);
      const uint32_t d = tm + kColS + sa * 32;
      __syncwarp();
      if (elect_one()) {
#pragma unroll
        for (int g = 0; g < 9; ++g) {
          const uint64_t k0 = (g < 4 ? db + g * kGroup / 16 : da + (g - 4) * kGroup / 16);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (g < kQTmem)
              umma_f16_ts(d, tm + kColQ + g * 32 + k * 8, k0 + k * 2, idesc_s, g + k > 0);
            else
              umma_f16_ss(d, dq + ((g - kQTmem) * kQGroup + k * 32) / 16, k0 + k * 2, idesc_s, 1u);
          }
        }
        umma_commit(&aux->s_full[sa]);
        if (last) umma_commit(&aux->q_empty);
      }
      __syncwarp();
      return true;
    };
    auto values = [&](int it, bool first, bool last) -> bool {
      const uint32_t u = uniform(it), sb = u & 3, sc = u % kStagesC, pb = u & 1;
      if ((first && pieces > 0 && !mbar_wait_warp(&aux->o_empty, (pieces - 1) & 1)) ||
          !mbar_wait_warp(&aux->p_full[pb], (u >> 1) & 1))
        return false;
      tc_fence_after();
      const uint32_t own = s0 + kOffB + sb * kBytesV, other = s0 + kOffC + sc * kBytesV;
      // P: rows of 32 bytes, 32-byte swizzle; V: 64-column groups kGroup bytes apart
      const uint64_t dp = make_smem_desc(s0 + kOffP + pb * 4 * kPPart, 16, 256, 6);
      const uint64_t dv0 = make_smem_desc(rank == 0 ? own : other, kGroup, 1024, 2);
      const uint64_t dv1 = make_smem_desc(rank == 0 ? other : own, kGroup, 1024, 2);
      __syncwarp();
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            umma_f16_ss(tm + kColO, dp + (h * 2 + k) * kPPart / 16,
                        (h ? dv1 : dv0) + k * 2048 / 16, idesc_pv, !first || h + k > 0);
        }
        umma_commit_cluster(&aux->pv_done[sb], 3);
      }
      __syncwarp();
      return true;
    };
    int it = 0;
    bool live = true;
    while (live && w.next()) {
      live = scores(it, true, w.n == 1) && (w.n == 1 || scores(it + 1, false, w.n == 2));
      for (int j = 0; live && j < w.n; ++j, ++it)
        live = (j + 2 >= w.n || scores(it + 2, false, j + 3 == w.n)) && values(it, j == 0, j + 1 == w.n);
      ++pieces;
    }
    if (!live && lane == 0) {
      umma_commit(&aux->drain);
      mbar_wait_drain(&aux->drain, 0);
    }
  } else if (warp < 8) {
    // -------------------------------------------------------------- softmax
    const int r = tid & 127, hh = tid >> 7, part = 2 * c + hh;  // row, 16 of the CTA's 32 cache rows, of the tile's 64
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float sl2 = p.scale * 1.4426950408889634f;
    const uint32_t peer = static_cast<uint32_t>(1 - c);
    // P of this warp's 32 rows and 16 cache rows: 1 KB, 16-byte half h of row r at h ^ (r / 4 % 2)
    uint8_t* mine = smem + kOffP + part * kPPart + (warp & 3) * 1024;
    const uint32_t peer_mine = mapa_shared(smem_u32(mine), peer);
    const uint32_t peer_bar_p = mapa_shared(smem_u32(&aux->p_full[0]), peer);
    uint32_t to[2], to_bar[2];  // this CTA's and the other's
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      to[k] = mapa_shared(smem_u32(&aux->shared[0][part][r]), k);
      to_bar[k] = mapa_shared(smem_u32(&aux->x_full[0]), k);
    }
    // both score buffers are free
    if (lane == 0) mbar_arrive(&aux->kv_full[0]), mbar_arrive(&aux->kv_full[1]);
    int told = 0, heard = 0;
    auto tell = [&](float v) {
      const int slot = told % 3;
      if (tid == 0) mbar_arrive_expect_tx(&aux->x_full[slot], 4 * kRows * 4);
#pragma unroll
      for (int k = 0; k < 2; ++k) st_async_f32(to[k] + slot * 4 * kRows * 4, v, to_bar[k] + slot * 8);
      ++told;
    };
    auto hear = [&](float (&v)[4]) -> bool {
      const int slot = heard % 3;
      if (!mbar_wait_warp(&aux->x_full[slot], (heard / 3) & 1)) return false;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = aux->shared[slot][k][r];
      ++heard;
      return true;
    };
    if (p.debug_stall) mbar_wait(&aux->stall, 0);  // test hook: runs into the wait limit
    int it = 0, pieces = 0, tails = 0;  // tails: phase bit per buffer
    bool live = true;
    while (live && w.next()) {
      const int row = w.mt * kRows + r;
      const int valid = w.kv;  // cache rows that hold anything
      const int lim = w.u.limit(w.q, w.kv, min(row / p.num_heads, w.q - 1));
      // tiles below this one are seen in full by every row (the first row sees the least)
      const int clean = w.u.limit(w.q, w.kv, w.mt * kRows / p.num_heads) / kTok;
      float m = -INFINITY, l = 0.f;
      float s[16], s_next[16];
      // scores of a tile from TMEM, masked, and their maximum on its way
      auto fetch = [&](int i, int t, float (&x)[16]) {
        tc_fence_after();
        uint32_t sv[16];
        tmem_ld_32x32b_x16(tbase + lane_off + kColS + (i & 1) * 32 + hh * 16, sv);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux->kv_full[(i + 2) & 3]);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(sv[e]);
        if (t >= clean) {
          const int seen = lim - t * kTok - part * 16;
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = e < seen ? x[e] : -INFINITY;
        }
        float a = fmax3f(x[0], x[1], x[2]), b = fmax3f(x[3], x[4], x[5]);
        a = fmax3f(a, x[6], x[7]), b = fmax3f(b, x[8], x[9]);
        a = fmax3f(a, x[10], x[11]), b = fmax3f(b, x[12], x[13]);
        a = fmax3f(a, b, fmaxf(x[14], x[15]));
        tell(a);
      };
      live = mbar_wait_warp(&aux->s_full[it & 1], (it >> 1) & 1);
      if (!live) break;
      fetch(it, w.t0, s);
      for (int j = 0; live && j < w.n; ++j, ++it) {
        const int t = w.t0 + j, pb = it & 1;
        // the next tile's scores, and its maximum on its way: now if they are there, which hides the
        // exchange behind this tile's exponentials, else after this tile's P, which may be what they wait for
        const bool early =
            j + 1 < w.n && __all_sync(0xffffffffu, mbar_test(&aux->s_full[(it + 1) & 1], ((it + 1) >> 1) & 1));
        if (early) fetch(it + 1, t + 1, s_next);
        float of[4];
        live = hear(of);
        if (!live) break;
        const float mx = fmax3f(of[0], of[1], fmaxf(of[2], of[3])) * sl2;
        // all four threads of the row take the same decision from the same maxima
        const bool move = mx > m + 8.f;
        const float dm = move ? ex2(m - mx) : 1.f;  // 0 while nothing has been seen
        if (move) m = mx;
        const float neg = m == -INFINITY ? 0.f : -m;
        float r0 = 0.f, r1 = 0.f;
        uint32_t pk[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float y0, y1;
          ffma2_bcast(y0, y1, s[e], s[e + 1], sl2, neg);
          y0 = ex2(y0), y1 = ex2(y1);
          fadd2(r0, r1, y0, y1);
          pk[e >> 1] = pack2<kFp16>(y0, y1);
        }
        l = l * dm + (r0 + r1);
        if (j > 0 && __any_sync(0xffffffffu, move)) {
          live = mbar_wait_warp(&aux->pv_done[(it - 1) & 3], ((it - 1) >> 2) & 1);  // O holds every tile before this one
          if (!live) break;
          tc_fence_after();
#pragma unroll 1
          for (int g = 4 * hh; g < 4 * hh + 4; ++g) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(tbase + lane_off + kColO + g * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * dm);
            tmem_st_32x32b_x32(tbase + lane_off + kColO + g * 32, o);
          }
          tmem_wait_st();
          tc_fence_before();
        }
        // this buffer's last P has been read by both CTAs (and copied)
        live = it < kPBuf || mbar_wait_warp(&aux->pv_done[(it - kPBuf) & 3], ((it - kPBuf) >> 2) & 1);
        if (!live) break;
        uint8_t* dst = mine + pb * 4 * kPPart;
#pragma unroll
        for (int q = 0; q < 2; ++q)
          *reinterpret_cast<uint4*>(dst + lane * 32 + ((q ^ ((lane >> 2) & 1)) << 4)) =
              make_uint4(pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
        if ((t + 1) * kTok > valid) {
          // rows past the request's length may hold NaN: weight 0 does not hide
          // them from the product, so they are cleared
          live = mbar_wait_warp(&aux->tail_full[pb], (tails >> pb) & 1);
          tails ^= 1 << pb;
          if (!live) break;
          if (t * kTok + hh * kHalfTok + lane >= valid) {
            uint8_t* stage = smem + (hh == c ? kOffB + it % kStagesB * kBytesV : kOffC + it % kStagesC * kBytesV);
            uint4* v = reinterpret_cast<uint4*>(stage + (warp & 3) * kGroup + lane * 128);
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q ^ (lane & 7)] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          bulk_copy_cluster(peer_mine + pb * 4 * kPPart, dst, 1024, peer_bar_p + pb * 8);
          mbar_arrive_expect_tx(&aux->p_full[pb], 1024);
        }
        if (j + 1 < w.n && !early) {
          live = mbar_wait_warp(&aux->s_full[(it + 1) & 1], ((it + 1) >> 1) & 1);
          if (!live) break;
          fetch(it + 1, t + 1, s_next);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = s_next[e];
      }
      if (!live) break;
      // the row's sum over the four threads, added in one order by all
      float of[4];
      tell(l);
      live = hear(of);
      if (!live) break;
      l = (of[0] + of[1]) + (of[2] + of[3]);
      const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN among the scores stays one
      const bool last = w.last;  // of the run
      const int64_t grow = w.tok * p.num_heads + row;
      if (c == 0 && hh == 0 && row < w.q * p.num_heads && grow < p.num_tokens * p.num_heads) {
        const float lse = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
        if (w.starts && w.ends)
          p.lse[grow] = lse;
        else
          P.parts.lse[(2 * cluster + (w.starts ? 1 : 0)) * kRows + r] = lse;
        if (w.starts) {
          P.parts.row_info[grow] =
              w.ends ? 0 : cut_info(aux->sched, cluster, w.base + w.unit_tiles - 1, r);
        }
      }
      // P V of the last tile is done in both CTAs: this warp's own P is free, 1 KB to stage its half of the columns,
      // while warps 8-11 place the next query tile; at the end of the run the query's shared memory, 4 KB
      live = mbar_wait_warp(&aux->pv_done[(it - 1) & 3], ((it - 1) >> 2) & 1);
      if (!live) break;
      tc_fence_after();
      if (last)
        write_rows<kFp16, true>(P, w, cluster, c, inv, tbase + lane_off, smem + kOffQ + warp * 4096, 4 * hh, 4 * hh + 4,
                                nullptr);
      else
        write_rows<kFp16, false>(P, w, cluster, c, inv, tbase + lane_off, mine, 4 * hh, 4 * hh + 4, &aux->o_empty);
      ++pieces;
    }
    // the other CTA's last commits (and with them its copies of this CTA's P) have arrived
    // before this CTA may leave
    for (int i = max(0, it - kPBuf); live && i < it; ++i)
      live = mbar_wait_warp(&aux->pv_done[i & 3], (i >> 2) & 1);
  } else {
    // --------------------------------------------------------- query loads
    const int r = tid - 256;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    // Query tile: the nine groups of 64 dims come by TMA, group g into slot g % 3 of 16 KB; six
    // move on to TMEM, the last three stay. (Loads of a row per thread touch 32 lines per
    // instruction: 14,000 cycles in which the softmax stood still too.)
    auto load_group = [&](const Walk<kRows, kTok, kSetup>& x, int g) {
      // group order: the CTA's own columns, the other latent ones, the rotary part
      const int col = g < 4 ? 4 * c + g : g < 8 ? 4 * (1 - c) + g - 4 : 8;
      mbar_arrive_expect_tx(&aux->qs_full[g % 3], kQGroup);
      tma_load_3d(smem + kOffQ + g % 3 * kQGroup, &P.map_q, &aux->qs_full[g % 3], 0,
                  static_cast<int>(x.tok * p.num_heads + x.mt * kRows), col);
    };
    auto prefetch_q = [&](const Walk<kRows, kTok, kSetup>& x) {
      if (tid == 256)
        for (int g = 0; g < 9; ++g)
          tma_prefetch_3d(&P.map_q, 0, static_cast<int>(x.tok * p.num_heads + x.mt * kRows), g);
    };
    auto place_q = [&](const Walk<kRows, kTok, kSetup>& x, int piece) -> bool {
      if (tid == 256)
        for (int g = 0; g < 3; ++g) load_group(x, g);
      for (int g = 0; g < 9; ++g) {
        bool ok = mbar_wait_warp(&aux->qs_full[g % 3], (piece * 3 + g / 3) & 1);
        if (ok && g < kQTmem) {
          uint32_t x32[32];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint4 v = *reinterpret_cast<const uint4*>(smem + kOffQ + g % 3 * kQGroup + sw128(r, k));
            x32[4 * k] = v.x;
            x32[4 * k + 1] = v.y;
            x32[4 * k + 2] = v.z;
            x32[4 * k + 3] = v.w;
          }
          tmem_st_32x32b_x32(tbase + lane_off + kColQ + g * 32, x32);
          __syncwarp();
          if (lane == 0) mbar_arrive(&aux->qs_empty[g % 3]);
          if (warp == 8) {
            ok = mbar_wait_warp(&aux->qs_empty[g % 3], (piece * 2 + g / 3) & 1);
            if (ok && lane == 0) load_group(x, g + 3);
            __syncwarp();
          }
        }
        if (!ok) return false;
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&aux->q_full);
      return true;
    };
    // the next piece's query goes in as soon as the last scores of this one are computed
    bool live = true;
    for (int piece = 0; live && w.next(); ++piece) {
      prefetch_q(w);
      if (piece > 0) {
        live = mbar_wait_warp(&aux->q_empty, (piece - 1) & 1);
        if (!live) break;
        tc_fence_after();
      }
      live = place_q(w, piece);
    }
  }
  __syncwarp();
  if (!remote) cluster_wait();
  if (cta_aborted()) {
    // loads into this CTA and copies into the other one may be in flight (a few hundred KB): they get a millisecond,
    // hundreds of times what they take, before either CTA leaves
    for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 1000 * 1000;) {
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // no more stores or arrivals to the other CTA
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

template <bool kFp16, int kR>
cudaError_t launch(Params& P, cudaStream_t stream) {
  auto kern = latent_decode_kernel<kFp16, kR>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), kSmemBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // as many clusters as run at once: their runs are equal, a second wave would double the time
  static std::atomic<int> resident[64] = {};
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int n = resident[dev & 63];
  if (n == 0) {
    int found = 0;
    cfg.gridDim = dim3(2 * kMaxClusters);
    if (cudaOccupancyMaxActiveClusters(&found, reinterpret_cast<const void*>(kern), &cfg) != cudaSuccess || found <= 0) {
      cudaGetLastError();
      found = kMaxClusters;
    }
    n = std::min(found, kMaxClusters);
    resident[dev & 63] = n;
  }
  const int clusters = std::min(n, run_bound<kRows, kTok, kSetup>(P.L, kMaxClusters));
  cfg.gridDim = dim3(2 * clusters);
  e = cudaLaunchKernelEx(&cfg, kern, P);
  if (e != cudaSuccess) return e;
  return launch_combine<kFp16, kRows, kTok>(P.L, P.parts, clusters, stream);
}

}  // namespace

size_t latent_decode_pair_workspace(const LatentDecodeLaunch& p) {
  return partial_bytes<kRows>(p, run_bound<kRows, kTok, kSetup>(p, kMaxClusters));
}

cudaError_t launch_latent_decode_pair(const LatentDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream) {
  Params P;
  P.L = p;
  P.parts = partials<kRows>(p, run_bound<kRows, kTok, kSetup>(p, kMaxClusters), workspace);
  // cache rows as 9 groups of 64 dims; a load is the rows of one page (at most 32) x 4 groups (or 1).
  // A cache without pages: a map over one row that nothing in bounds reads.
  const uint32_t rows = p.block_size < kHalfTok ? 16 : 32;
  const uint64_t pool_rows = std::max<uint64_t>(1, static_cast<uint64_t>(p.num_blocks) * p.block_size);
  const void* base = p.num_blocks > 0 ? p.cache : p.query;
  const uint64_t extent[3] = {64, pool_rows, 9}, stride[2] = {kLatentRow * 2, 128};
  const uint64_t extent_q[3] = {64, static_cast<uint64_t>(p.num_tokens) * p.num_heads, 9};
  const uint32_t box4[3] = {64, rows, 4}, box1[3] = {64, rows, 1}, box_q[3] = {64, kRows, 1};
  if (!encode_tmap_nd(&P.map4, base, 3, extent, stride, box4) ||
      !encode_tmap_nd(&P.map1, base, 3, extent, stride, box1) ||
      !encode_tmap_nd(&P.map_q, p.query, 3, extent_q, stride, box_q))
    return cudaErrorInvalidValue;
  if (rows == 16) return fp16 ? launch<true, 16>(P, stream) : launch<false, 16>(P, stream);
  return fp16 ? launch<true, 32>(P, stream) : launch<false, 32>(P, stream);
}

}  // namespace cascade
