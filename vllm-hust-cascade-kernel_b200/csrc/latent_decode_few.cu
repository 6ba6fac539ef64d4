// Latent attention, absorbed form (cascade_latent_decode), for requests of up to
// 32 query rows (a few heads per GPU): bound by reading the cache, 1,152 bytes
// per token. The rows that a tensor-core tile has go to the cache:
//   S^T [64 tokens x kN rows]     = C [64 x 576] X^T
//   O^T [4 x 128 values x kN rows] += V^T [512 x 64] P
// with kN = 16 or 32 query rows as the MMA's N, so a CTA holds a whole output
// (4 kN TMEM columns) and needs no other. Both products read the cache tile from
// shared memory as it was loaded (K-major, then M-major).
//
// Measured: 296 requests x 16 heads over 3,000 tokens (1.02 GB) 171 us, 6.0 TB/s
// (0.93 of the copy rate); 48 requests x 16 heads over 119-5,885 tokens (158 MB) 42
// us on the device: 24 us of HBM, the rest the start (find_run, page ids, query,
// 10,000 cycles to the first scores), the merge and the launches.
//
// Softmax: a thread per token. The rows' running maxima are the same in every
// thread; they move only when some score exceeds its row's by more than 2^8 (a
// vote per tile), so the columns' maxima over 128 lanes are rarely needed. The
// sums stay per thread and row until the piece ends, in fp32, of the unrounded
// exponentials. P is rounded to the inputs' type, which the second product needs.
//
// Shared memory: a tile's eight boxes of 8 tokens x 576 values (page sizes are
// multiples of 16) each come in two parts, six (four) groups of 64 values in a ring of
// three slots and the rest in one of two, so that 1.7 (1.5) tiles are on their way
// while one is worked on: it takes about 2,300 cycles from the last load to the free
// slot, an SM's share of HBM 3,250 for its 74 KB. (Tiles of 128 tokens leave
// 48 KB to be on their way: 61 against 48 us on the 48 requests. Scores of the next
// tile before P V of this one hold the slots longer: 182 against 174 on the 296.)
//
// Warps: 0-3 softmax and output (a piece's after the next one's first tile: the
// products go on meanwhile), 4 cache loads, 5 MMA issue, 6 query loads.
#include <algorithm>
#include <climits>

#include "latent_decode.cuh"

namespace cascade {
namespace {

constexpr int kTok = 64;
constexpr int kSetup = 1;  // what a new unit costs, in tiles (see find_run): 48 requests x 16 heads 0 47.1 us, 1 42.1, 2 42.7
constexpr int kThreads = 7 * 32;
constexpr int kBox = 8;  // cache rows per load
constexpr int kBoxes = kTok / kBox;
constexpr int kAtom = kBox * 128;  // 8 rows x 64 values

template <int kN>
struct Few {
  // a tile's nine groups of 64 values in two parts, with rings of their own
  static constexpr int kGroupsA = kN == 16 ? 6 : 4, kGroupsB = 9 - kGroupsA;
  static constexpr int kSlotsA = 3, kSlotsB = 2;
  static constexpr int kBytesA = kBoxes * kGroupsA * kAtom, kBytesB = kBoxes * kGroupsB * kAtom;
  static constexpr int kQGroup = kN * 128;
  static constexpr int kRowBytes = kN * 2;  // of P: a token's weights
  static constexpr int kOffQ = 0;
  static constexpr int kOffP = kOffQ + 9 * kQGroup;
  static constexpr int kBytesP = kTok * kRowBytes;
  static constexpr int kOffA = kOffP + kBytesP;
  static constexpr int kOffB = kOffA + kSlotsA * kBytesA;
  static constexpr int kTiles = kOffB + kSlotsB * kBytesB;
  static constexpr int kColS = 0, kColO = kN;  // TMEM columns: scores, outputs of two pieces
  static constexpr int kTmem = kN == 16 ? 256 : 512;
  static_assert(kColO + 8 * kN <= kTmem && kOffP % 1024 == 0 && kOffA % 1024 == 0, "layout");
  static_assert(kGroupsA % 2 == 0, "an M block of the second product lies in one part");

  struct __align__(16) Aux {
    union {
      float top[4][kN];  // columns' maxima per warp
      int64_t scan[2][kThreads / 32];  // find_run only
    };
    float sum[4][kN];
    float inv[kN];  // 1 / the rows' sums
    int lim[kN];  // tokens that a row sees
    uint64_t a_full[kSlotsA], b_full[kSlotsB], pv_done[kSlotsA];
    uint64_t q_full, q_free, s_full, p_full, o_full[2], stall, drain;
    uint32_t tmem_base;
    Sched sched;
  };
  static constexpr int kStatic = 32;  // the wait state comes first
  static constexpr int kSmem = (kStatic + static_cast<int>(sizeof(Aux)) + 1023) / 1024 * 1024 + kTiles - kStatic;
  static_assert(kSmem + kStatic <= 227 * 1024, "shared memory per CTA");
};

struct Params {
  LatentDecodeLaunch L;
  CUtensorMap map_a, map_b;  // 64 values x 8 cache rows x the part's groups
  CUtensorMap map_q;         // 64 values x kN query rows x 9 groups
  Partials parts;
};

// v[j] of all 32 lanes combined per j: a lane returns the one of column `col`.
template <int kN, class Op>
__device__ __forceinline__ float reduce_columns(float (&v)[kN], int lane, int& col, Op op) {
  col = 0;
  int d = 16;
#pragma unroll
  for (int half = kN / 2; half >= 1; half >>= 1, d >>= 1) {
    const bool up = lane & d;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float send = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
      v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, d));
    }
    if (up) col += half;
  }
  if (kN == 16) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], 1));
  return v[0];
}

// the four softmax warps meet; true if any thread says so
__device__ __forceinline__ bool meet_any(bool v) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(v))
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void meet() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

template <int kN>
__device__ __forceinline__ void tmem_ld_row(uint32_t addr, uint32_t (&x)[kN]) {
  if constexpr (kN == 16)
    tmem_ld_32x32b_x16(addr, x);
  else
    tmem_ld_32x32b_x32(addr, x);
}
template <int kN>
__device__ __forceinline__ void tmem_st_row(uint32_t addr, const uint32_t (&x)[kN]) {
  if constexpr (kN == 16)
    tmem_st_32x32b_x16(addr, x);
  else
    tmem_st_32x32b_x32(addr, x);
}

template <bool kFp16, int kN>
__global__ void __launch_bounds__(kThreads, 1) latent_decode_few_kernel(const __grid_constant__ Params P) {
  using F = Few<kN>;
  using Aux = typename F::Aux;
  pdl_launch_dependents();
  const LatentDecodeLaunch& p = P.L;
  extern __shared__ uint8_t smem_raw[];
  Aux* aux = reinterpret_cast<Aux*>(smem_raw);
  uint8_t* smem = smem_raw + sizeof(Aux) + ((0u - (smem_u32(smem_raw) + static_cast<uint32_t>(sizeof(Aux)))) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int run = blockIdx.x, runs = gridDim.x;

  if (tid == 0) {
    cta_wait_init(static_cast<uint64_t>(p.wait_limit_us) * 1000);
    for (int s = 0; s < F::kSlotsA; ++s) mbar_init(&aux->a_full[s], 1), mbar_init(&aux->pv_done[s], 1);
    for (int s = 0; s < F::kSlotsB; ++s) mbar_init(&aux->b_full[s], 1);
    mbar_init(&aux->q_full, 1);
    mbar_init(&aux->q_free, 1);
    for (int s = 0; s < 2; ++s) mbar_init(&aux->o_full[s], 1);
    mbar_init(&aux->s_full, 1);
    mbar_init(&aux->p_full, 4);
    mbar_init(&aux->stall, 1);
    mbar_init(&aux->drain, 1);
    fence_mbar_init();
  }
  if (tid == 32) tma_prefetch_desc(&P.map_a), tma_prefetch_desc(&P.map_b);
  if (tid == 64) tma_prefetch_desc(&P.map_q);
  if (warp == 5) {
    tmem_alloc(&aux->tmem_base, F::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  find_run<kN, kTok, kSetup, kThreads>(p, P.parts.row_info, run, runs, aux->scan, &aux->sched);  // (with CTA barriers)
  tc_fence_after();
  const uint32_t tbase = aux->tmem_base;
  Walk<kN, kTok, kSetup> w(p, aux->sched);

  if (warp == 4) {
    // ---------------------------------------------------------- cache loads
    // Lane i takes care of the i-th eight rows of four tiles; their page ids are read four tiles (or a piece) ahead.
    const int oob = max(1, p.num_blocks * p.block_size);
    constexpr int kNoPage = INT_MIN;
    auto first_row = [&](int t) { return t * kTok + lane * kBox; };
    auto page_id = [&](const Walk<kN, kTok, kSetup>& x, int t) {
      const int pages = (x.kv + p.block_size - 1) / p.block_size, page = first_row(t) / p.block_size;
      return page < pages ? p.block_table[static_cast<int64_t>(x.b) * p.block_cols + page] : kNoPage;
    };
    int it = 0, id_next = kNoPage, y = oob;
    bool live = true, more = w.next();
    if (more) id_next = page_id(w, w.t0);
    while (live && more) {
      const int t0 = w.t0, t1 = w.t0 + w.n;
      const Walk<kN, kTok, kSetup> now = w;
      more = false;
      for (int t = t0; t < t1; ++t, ++it) {
        const int ahead = (t - t0) & 3;
        if (ahead == 0) y = id_next == kNoPage ? oob : paged_row(id_next, first_row(t), p.block_size, p.num_blocks, oob);
        const int row = __shfl_sync(0xffffffffu, y, ahead * kBoxes + (lane & (kBoxes - 1)));
        const int sa = it % F::kSlotsA, sb = it % F::kSlotsB;
        // P V of the tile that had the slot is done
        auto freed = [&](int slots) {
          const int old = it - slots;
          return old < 0 || mbar_wait_warp(&aux->pv_done[old % F::kSlotsA], (old / F::kSlotsA) & 1);
        };
        live = freed(F::kSlotsA);
        if (!live) break;
        if (lane == 0) mbar_arrive_expect_tx(&aux->a_full[sa], F::kBytesA);
        __syncwarp();
        if (lane < kBoxes)
          tma_load_3d(smem + F::kOffA + sa * F::kBytesA + lane * F::kGroupsA * kAtom, &P.map_a, &aux->a_full[sa], 0, row, 0);
        live = freed(F::kSlotsB);
        if (!live) break;
        if (lane == 0) mbar_arrive_expect_tx(&aux->b_full[sb], F::kBytesB);
        __syncwarp();
        if (lane < kBoxes)
          tma_load_3d(smem + F::kOffB + sb * F::kBytesB + lane * F::kGroupsB * kAtom, &P.map_b, &aux->b_full[sb], 0, row,
                      F::kGroupsA);
        __syncwarp();
        if (ahead == 0) {
          if (t + 4 < t1)
            id_next = page_id(now, t + 4);
          else if ((more = w.next()))
            id_next = page_id(w, w.t0);
        }
      }
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issue
    const uint32_t idesc_s = make_idesc_f16(kTok, kN, kFp16 ? 0u : 1u, 0, 0);
    const uint32_t idesc_o = make_idesc_f16(128, kN, kFp16 ? 0u : 1u, 1, 1);
    const uint32_t tm = uniform(tbase), s0 = uniform(smem_u32(smem));
    const uint64_t dq = make_smem_desc(s0 + F::kOffQ, 16, 1024, 2);
    // P: a token's kN weights in a row of 32 (64) bytes, swizzled in as many
    const uint64_t dp = make_smem_desc(s0 + F::kOffP, 16, 8 * F::kRowBytes, kN == 16 ? 6 : 4);
    int it = 0, piece = 0;
    bool live = true;
    while (live && w.next()) {
      live = mbar_wait_warp(&aux->q_full, piece & 1);
      for (int t = 0; live && t < w.n; ++t, ++it) {
        const uint32_t u = uniform(it), sa = u % F::kSlotsA, sb = u % F::kSlotsB, o = uniform(piece & 1);
        const uint32_t a = s0 + F::kOffA + sa * F::kBytesA, b = s0 + F::kOffB + sb * F::kBytesB;
        const bool last = t + 1 == w.n;
        // groups [g0, g1) of a part whose boxes are `pitch` bytes apart
        auto scores = [&](uint32_t part, int pitch, int g0, int g1) {
          const uint64_t da = make_smem_desc(part, 16, pitch, 2);
          tc_fence_after();
          __syncwarp();
          if (elect_one()) {
#pragma unroll 1
            for (int g = g0; g < g1; ++g) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16_ss(tm + F::kColS, da + (g - g0) * kAtom / 16 + k * 2, dq + g * F::kQGroup / 16 + k * 2, idesc_s,
                            g + k > 0);
            }
            if (g1 == 9) {
              umma_commit(&aux->s_full);
              if (last) umma_commit(&aux->q_free);
            }
          }
          __syncwarp();
        };
        live = mbar_wait_warp(&aux->a_full[sa], (u / F::kSlotsA) & 1);
        if (!live) break;
        scores(a, F::kGroupsA * kAtom, 0, F::kGroupsA);
        live = mbar_wait_warp(&aux->b_full[sb], (u / F::kSlotsB) & 1);
        if (!live) break;
        scores(b, F::kGroupsB * kAtom, F::kGroupsA, 9);
        live = mbar_wait_warp(&aux->p_full, u & 1);
        if (!live) break;
        tc_fence_after();
        __syncwarp();
        if (elect_one()) {
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            const bool in_a = 2 * j < F::kGroupsA;
            const int pitch = (in_a ? F::kGroupsA : F::kGroupsB) * kAtom;
            const uint64_t dv = make_smem_desc((in_a ? a + 2 * j * kAtom : b + (2 * j - F::kGroupsA) * kAtom), kAtom, pitch, 2);
#pragma unroll
            for (int k = 0; k < kTok / 16; ++k)
              umma_f16_ss(tm + F::kColO + (o * 4 + j) * kN, dv + k * 2 * pitch / 16, dp + k * 16 * F::kRowBytes / 16, idesc_o,
                          t + k > 0);
          }
          umma_commit(&aux->pv_done[sa]);
          if (last) umma_commit(&aux->o_full[o]);
        }
        __syncwarp();
      }
      ++piece;
    }
    if (!live && lane == 0) {
      umma_commit(&aux->drain);
      mbar_wait_drain(&aux->drain, 0);
    }
  } else if (warp == 6) {
    // ---------------------------------------------------------- query loads
    for (int piece = 0; w.next(); ++piece) {
      if (piece > 0) {
        if (lane == 0) tma_prefetch_3d(&P.map_q, 0, static_cast<int>(w.tok * p.num_heads + w.mt * kN), 0);
        if (!mbar_wait_warp(&aux->q_free, (piece - 1) & 1)) break;
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(&aux->q_full, 9 * F::kQGroup);
        tma_load_3d(smem + F::kOffQ, &P.map_q, &aux->q_full, 0, static_cast<int>(w.tok * p.num_heads + w.mt * kN), 0);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------ softmax, output
    // The four warps meet in every tile; none leaves the loop early (an aborted CTA's waits return at once), so none
    // is waited for in vain.
    const uint32_t tl = tbase + (static_cast<uint32_t>(warp * 32) << 16);
    const float sl2 = p.scale * 1.4426950408889634f;
    const int mine = warp * 16 + lane;  // token of the tile: 64 rows of scores lie in the first 16 lanes of each quarter
    const int my_col = tid & (kN - 1);
    if (p.debug_stall) mbar_wait_warp(&aux->stall, 0);  // test hook: runs into the wait limit
    float m[kN], l[kN], my_m = -INFINITY;  // my_m: row my_col's
    // A piece's output is written after the next piece's first P: the products go on meanwhile, into the other
    // accumulator.
    struct {
      int64_t grow0, slot, last_tile;
      int rows;
      bool starts, ends;
      float m;
    } done = {};
    int it = 0, piece = 0, t = 0;
    int valid = 0, clean = 0;  // tokens that hold anything; tiles below `clean` are seen in full by every row
    bool more = w.next(), start = true, pending = false;
    while (true) {
      if (more) {
        if (start) {
          const int row0 = w.mt * kN;
          valid = w.kv;
          clean = w.u.limit(w.q, w.kv, row0 / p.num_heads) / kTok;
          if (tid < kN) aux->lim[tid] = w.u.limit(w.q, w.kv, min((row0 + tid) / p.num_heads, w.q - 1));
          meet();
#pragma unroll
          for (int j = 0; j < kN; ++j) m[j] = -INFINITY, l[j] = 0.f;
          my_m = -INFINITY;
          t = w.t0;
        }
        mbar_wait_warp(&aux->s_full, it & 1);
        tc_fence_after();
        uint32_t x[kN];
        tmem_ld_row<kN>(tl + F::kColS, x);
        tmem_wait_ld();
        const int tok = t * kTok + mine;
        if (lane >= 16) {
#pragma unroll
          for (int j = 0; j < kN; ++j) x[j] = 0xff800000u;
        }
        if (t >= clean) {
#pragma unroll
          for (int j = 0; j < kN; ++j) x[j] = tok < aux->lim[j] ? x[j] : 0xff800000u;
        }
        bool move = false;
#pragma unroll
        for (int j = 0; j < kN; ++j) move |= __uint_as_float(x[j]) * sl2 > m[j] + 8.f;
        if (meet_any(move)) {
          float v[kN];
#pragma unroll
          for (int j = 0; j < kN; ++j) v[j] = __uint_as_float(x[j]);
          int col;
          const float top = reduce_columns<kN>(v, lane, col, [](float a, float b) { return fmaxf(a, b); });
          aux->top[warp][col] = top;
          meet();
          auto top_of = [&](int j) {
            return sl2 * fmaxf(fmaxf(aux->top[0][j], aux->top[1][j]), fmaxf(aux->top[2][j], aux->top[3][j]));
          };
          if (top_of(my_col) > my_m + 8.f) my_m = top_of(my_col);
          float dm[kN];
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            const float mx = top_of(j);
            const bool up = mx > m[j] + 8.f;
            dm[j] = up ? ex2(m[j] - mx) : 1.f;  // 0 while nothing has been seen
            if (up) m[j] = mx;
            l[j] *= dm[j];
          }
          if (!start) {  // the scores came after the last tile's P V: the output is at rest
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {
              uint32_t o[kN];
              tmem_ld_row<kN>(tl + F::kColO + ((piece & 1) * 4 + b) * kN, o);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < kN; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * dm[j]);
              tmem_st_row<kN>(tl + F::kColO + ((piece & 1) * 4 + b) * kN, o);
            }
            tmem_wait_st();
          }
        }
        // P over the last tile's, whose product came before these scores
        uint32_t pk[kN / 2];
#pragma unroll
        for (int j = 0; j < kN; j += 2) {
          float y[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float neg = m[j + i] == -INFINITY ? 0.f : -m[j + i];
            y[i] = ex2(fmaf(__uint_as_float(x[j + i]), sl2, neg));
            l[j + i] += y[i];
          }
          pk[j / 2] = pack2<kFp16>(y[0], y[1]);
        }
        if (lane < 16) {
          uint8_t* dst = smem + F::kOffP + mine * F::kRowBytes;
          const int swap = kN == 16 ? (mine >> 2) & 1 : (mine >> 1) & 3;
#pragma unroll
          for (int q = 0; q < kN / 8; ++q)
            *reinterpret_cast<uint4*>(dst + ((q ^ swap) << 4)) =
                make_uint4(pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
        }
        if ((t + 1) * kTok > valid) {
          // rows past the request's length may hold NaN: weight 0 does not hide
          // them from the product, so they are cleared (the scores have read them);
          // two lanes per row, eight rows' 16-byte chunks in different banks
          const int r = warp * 16 + (lane & 15);
          if (t * kTok + r >= valid) {
#pragma unroll 1
            for (int g = lane >> 4; g < 8; g += 2) {
              uint8_t* at = g < F::kGroupsA
                                ? smem + F::kOffA + it % F::kSlotsA * F::kBytesA + ((r >> 3) * F::kGroupsA + g) * kAtom
                                : smem + F::kOffB + it % F::kSlotsB * F::kBytesB +
                                      ((r >> 3) * F::kGroupsB + g - F::kGroupsA) * kAtom;
#pragma unroll
              for (int q = 0; q < 8; ++q)
                *reinterpret_cast<uint4*>(at + (r & 7) * 128 + ((q ^ (r & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux->p_full);
        ++it;
      }
      if (pending) {
        pending = false;
        const bool whole = done.starts && done.ends;
        meet();
        if (tid < kN) {  // the rows' sums, added in one order
          const float s = (aux->sum[0][tid] + aux->sum[1][tid]) + (aux->sum[2][tid] + aux->sum[3][tid]);
          aux->inv[tid] = s == 0.f ? 0.f : 1.f / s;  // a NaN among the scores stays one
          if (tid < done.rows && !cta_aborted()) {
            const float lse = s == 0.f ? -INFINITY : (done.m + __log2f(s)) * 0.6931471805599453f;
            (whole ? p.lse + done.grow0 : P.parts.lse + done.slot)[tid] = lse;
            if (done.starts)
              P.parts.row_info[done.grow0 + tid] =
                  done.ends ? 0 : cut_info(aux->sched, run, done.last_tile, tid);
          }
        }
        meet();
        const int o_buf = more ? (piece & 1) ^ 1 : piece & 1, at = more ? piece - 1 : piece;
        const bool write = mbar_wait_warp(&aux->o_full[o_buf], (at >> 1) & 1);
        tc_fence_after();
        // (few instructions: they run once or twice, fetching them is what takes time)
#pragma unroll 1
        for (int j0 = 0; j0 < kN && j0 < done.rows && write; j0 += 4) {
          uint32_t o[4][4];
#pragma unroll
          for (int b = 0; b < 4; ++b) tmem_ld_32x32b_x4(tl + F::kColO + (o_buf * 4 + b) * kN + j0, o[b]);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float inv = aux->inv[j0 + j];
            if (j0 + j >= done.rows) break;
            uint16_t* to = static_cast<uint16_t*>(p.out) + (done.grow0 + j0 + j) * kLatentDim + tid;
            float* part = P.parts.o + (done.slot + j0 + j) * kLatentDim + tid;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const float v = inv == 0.f ? 0.f : __uint_as_float(o[b][j]) * inv;
              if (whole)
                to[b * 128] = static_cast<uint16_t>(pack2<kFp16>(v, 0.f));
              else
                part[b * 128] = v;
            }
          }
        }
        tc_fence_before();
      }
      if (!more) break;
      start = ++t == w.t0 + w.n;
      if (start) {
        int col;
        const float sum = reduce_columns<kN>(l, lane, col, [](float a, float b) { return a + b; });
        aux->sum[warp][col] = sum;
        pending = true;
        done.grow0 = w.tok * p.num_heads + w.mt * kN;
        done.slot = (2 * run + (w.starts ? 1 : 0)) * kN;
        done.last_tile = w.base + w.unit_tiles - 1;
        done.rows = static_cast<int>(min(static_cast<int64_t>(kN), min(static_cast<int64_t>(w.q) * p.num_heads - w.mt * kN,
                                                                      p.num_tokens * p.num_heads - done.grow0)));
        done.starts = w.starts, done.ends = w.ends;
        done.m = my_m;
        more = w.next();
        if (more) ++piece;
      }
    }
  }
  if (cta_aborted()) {
    // loads may be in flight (at most 213 KB): they get a millisecond before the CTA leaves
    for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 1000 * 1000;) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tbase, F::kTmem);
  }
}

template <bool kFp16, int kN>
cudaError_t launch(const LatentDecodeLaunch& p, void* workspace, cudaStream_t stream) {
  const int bound = run_bound<kN, kTok, kSetup>(p, kNumSMs);
  Params P;
  P.L = p;
  P.parts = partials<kN>(p, bound, workspace);
  // cache rows as 9 groups of 64 values; a load is eight rows of one page and a part's groups. A cache without pages:
  // a map over one row that nothing in bounds reads.
  const uint64_t pool_rows = std::max<uint64_t>(1, static_cast<uint64_t>(p.num_blocks) * p.block_size);
  const void* base = p.num_blocks > 0 ? p.cache : p.query;
  const uint64_t extent[3] = {64, pool_rows, 9}, stride[2] = {kLatentRow * 2, 128};
  const uint64_t extent_q[3] = {64, static_cast<uint64_t>(p.num_tokens) * p.num_heads, 9};
  const uint32_t box_a[3] = {64, kBox, Few<kN>::kGroupsA}, box_b[3] = {64, kBox, Few<kN>::kGroupsB}, box_q[3] = {64, kN, 9};
  if (!encode_tmap_nd(&P.map_a, base, 3, extent, stride, box_a) || !encode_tmap_nd(&P.map_b, base, 3, extent, stride, box_b) ||
      !encode_tmap_nd(&P.map_q, p.query, 3, extent_q, stride, box_q))
    return cudaErrorInvalidValue;
  auto kern = latent_decode_few_kernel<kFp16, kN>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), Few<kN>::kSmem);
  if (e != cudaSuccess) return e;
  kern<<<bound, kThreads, Few<kN>::kSmem, stream>>>(P);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_combine<kFp16, kN, kTok>(p, P.parts, bound, stream);
}

// Query rows per request, on average (the lengths may be on the device). Up to 16 and up to 32 rows this kernel is
// the faster one (48 requests, in a graph: 16 rows 42 against 69 us, 32 rows 48 against 70), above, where it would read
// the cache once per 32 rows, the pair kernel (48 rows 90 against 71, 64 rows 95 against 73).
int64_t mean_rows(const LatentDecodeLaunch& p) { return (p.num_tokens + p.batch - 1) / p.batch * p.num_heads; }

}  // namespace

size_t latent_decode_workspace(const LatentDecodeLaunch& p) {
  const int64_t rows = mean_rows(p);
  return rows <= 16   ? partial_bytes<16>(p, run_bound<16, kTok, kSetup>(p, kNumSMs))
         : rows <= 32 ? partial_bytes<32>(p, run_bound<32, kTok, kSetup>(p, kNumSMs))
                      : latent_decode_pair_workspace(p);
}

cudaError_t launch_latent_decode(const LatentDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream) {
  const int64_t rows = mean_rows(p);
  if (rows <= 16) return fp16 ? launch<true, 16>(p, workspace, stream) : launch<false, 16>(p, workspace, stream);
  if (rows <= 32) return fp16 ? launch<true, 32>(p, workspace, stream) : launch<false, 32>(p, workspace, stream);
  return launch_latent_decode_pair(p, fp16, workspace, stream);
}

}  // namespace cascade
