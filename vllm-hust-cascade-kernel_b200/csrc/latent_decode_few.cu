// Latent attention, absorbed form (cascade_latent_decode), for requests of up to
// 32 query rows (a few heads per GPU): bound by reading the cache, 1,152 bytes
// per token. The 128 rows that a tensor-core tile has go to the cache:
//   S^T [128 tokens x kN rows]  = C [128 x 576] X^T
//   O^T [4 x 128 values x kN rows] += V^T [512 x 128] P
// with kN = 16 or 32 query rows as the MMA's N, so a CTA holds a whole output
// (4 kN TMEM columns) and needs no other. Both products read the cache tile from
// shared memory as it was loaded (K-major, then M-major): 36 + 32 steps of 43
// cycles for 128 tokens, 2,900 cycles against the 6,500 that an SM's share of
// HBM takes for their 147 KB.
//
// Softmax: a thread per token. The rows' running maxima are the same in every
// thread; they move only when some score exceeds its row's by more than 2^8 (a
// vote per tile), so the columns' maxima over 128 lanes are rarely needed. The
// sums stay per thread and row until the piece ends, in fp32, of the unrounded
// exponentials. P is rounded to the inputs' type, which the second product needs.
//
// Shared memory: a ring of five 32 KB slots for pairs of 64-value groups
// (128 tokens x 128 values: one M block of the second product), freed block by block as
// P V goes, and kRope slots of 16 KB for the rotary group, freed by the scores.
//
// Warps: 0-3 softmax and output, 4 cache loads, 5 MMA issue, 6 query loads.
#include <algorithm>

#include "latent_decode.cuh"

namespace cascade {
namespace {

constexpr int kTok = 128;
constexpr int kThreads = 7 * 32;
constexpr int kPairs = 5;
constexpr int kGroup = kTok * 128;  // 128 tokens x 64 values

template <int kN>
struct Few {
  static constexpr int kRope = kN == 16 ? 2 : 1;
  static constexpr int kQGroup = kN * 128;
  static constexpr int kRowBytes = kN * 2;  // of P: a token's weights
  static constexpr int kOffQ = 0;
  static constexpr int kOffP = kOffQ + 9 * kQGroup;
  static constexpr int kOffV = kOffP + kTok * kRowBytes;
  static constexpr int kOffR = kOffV + kPairs * 2 * kGroup;
  static constexpr int kTiles = kOffR + kRope * kGroup;
  static constexpr int kColS = 0, kColO = kN;  // TMEM columns
  static constexpr int kTmem = kN == 16 ? 128 : 256;
  static_assert(kColO + 4 * kN <= kTmem && kOffP % 1024 == 0 && kOffV % 1024 == 0, "layout");

  struct __align__(16) Aux {
    union {
      float top[4][kN];  // columns' maxima per warp
      int64_t scan[2][kThreads / 32];  // find_run only
    };
    float sum[4][kN];
    int lim[kN];  // tokens that a row sees
    uint64_t v_full[kPairs], v_free[kPairs], r_full[kRope], r_free[kRope];
    uint64_t q_full, q_free, s_full, p_full, o_full, stall, drain;
    uint32_t tmem_base;
    Sched sched;
  };
  static constexpr int kStatic = 32;  // the wait state comes first
  static constexpr int kSmem = (kStatic + static_cast<int>(sizeof(Aux)) + 1023) / 1024 * 1024 + kTiles - kStatic;
  static_assert(kSmem + kStatic <= 227 * 1024, "shared memory per CTA");
};

struct Params {
  LatentDecodeLaunch L;
  CUtensorMap map;    // 64 values x box_rows cache rows
  CUtensorMap map_q;  // 64 values x kN query rows x 9 groups
  int box_rows;
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
    for (int s = 0; s < kPairs; ++s) mbar_init(&aux->v_full[s], 1), mbar_init(&aux->v_free[s], 1);
    for (int s = 0; s < F::kRope; ++s) mbar_init(&aux->r_full[s], 1), mbar_init(&aux->r_free[s], 1);
    mbar_init(&aux->q_full, 1);
    mbar_init(&aux->q_free, 1);
    mbar_init(&aux->s_full, 1);
    mbar_init(&aux->p_full, 4);
    mbar_init(&aux->o_full, 1);
    mbar_init(&aux->stall, 1);
    mbar_init(&aux->drain, 1);
    fence_mbar_init();
  }
  if (tid == 32) tma_prefetch_desc(&P.map);
  if (tid == 64) tma_prefetch_desc(&P.map_q);
  if (warp == 5) {
    tmem_alloc(&aux->tmem_base, F::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  find_run<kN, kTok, kThreads>(p, run, runs, aux->scan, &aux->sched);  // (with CTA barriers)
  tc_fence_after();
  const uint32_t tbase = aux->tmem_base;
  Walk<kN, kTok> w(p, aux->sched);

  if (warp == 4) {
    // ---------------------------------------------------------- cache loads
    const int boxes = kTok / P.box_rows, oob = max(1, p.num_blocks * p.block_size);
    int it = 0;
    bool live = true;
    while (live && w.next()) {
      const int32_t* bt = p.block_table + static_cast<int64_t>(w.b) * p.block_cols;
      const int pages = (min(w.kv, w.u.cap) + p.block_size - 1) / p.block_size;
      // lane i holds the pool row of box i of the next tile
      auto row_of = [&](int t) {
        const int tok = t * kTok + lane * P.box_rows, page = tok / p.block_size;
        return lane < boxes && page < pages ? paged_row(bt[page], tok, p.block_size, p.num_blocks, oob) : oob;
      };
      int y = row_of(w.t0);
      for (int t = w.t0; t < w.t0 + w.n; ++t, ++it) {
        const int y_next = t + 1 < w.t0 + w.n ? row_of(t + 1) : 0;
        for (int j = 0; j < 5; ++j) {  // four pairs of latent groups, then the rotary one
          const int i = j < 4 ? 4 * it + j : it, slots = j < 4 ? kPairs : F::kRope, s = i % slots;
          uint64_t* full = j < 4 ? &aux->v_full[s] : &aux->r_full[s];
          live = i < slots || mbar_wait_warp(j < 4 ? &aux->v_free[s] : &aux->r_free[s], (i / slots - 1) & 1);
          if (!live) break;
          uint8_t* dst = smem + (j < 4 ? F::kOffV + s * 2 * kGroup : F::kOffR + s * kGroup) + lane * P.box_rows * 128;
          if (lane == 0) mbar_arrive_expect_tx(full, j < 4 ? 2 * kGroup : kGroup);
          __syncwarp();
          if (lane < boxes) {
            tma_load_3d(dst, &P.map, full, 0, y, 2 * j);
            if (j < 4) tma_load_3d(dst + kGroup, &P.map, full, 0, y, 2 * j + 1);
          }
          __syncwarp();
        }
        if (!live) break;
        y = y_next;
      }
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issue
    const uint32_t idesc_s = make_idesc_f16(kTok, kN, kFp16 ? 0u : 1u, 0, 0);
    const uint32_t idesc_o = make_idesc_f16(kTok, kN, kFp16 ? 0u : 1u, 1, 1);
    const uint32_t tm = uniform(tbase), s0 = uniform(smem_u32(smem));
    const uint64_t dq = make_smem_desc(s0 + F::kOffQ, 16, 1024, 2);
    // P: a token's kN weights in a row of 32 (64) bytes, swizzled in as many
    const uint64_t dp = make_smem_desc(s0 + F::kOffP, 16, 8 * F::kRowBytes, kN == 16 ? 6 : 4);
    int it = 0, piece = 0;
    bool live = true;
    while (live && w.next()) {
      live = mbar_wait_warp(&aux->q_full, piece & 1);
      for (int t = 0; live && t < w.n; ++t, ++it) {
        for (int j = 0; live && j < 5; ++j) {
          const uint32_t i = uniform(j < 4 ? 4 * it + j : it), slots = j < 4 ? kPairs : F::kRope, s = i % slots;
          live = mbar_wait_warp(j < 4 ? &aux->v_full[s] : &aux->r_full[s], (i / slots) & 1);
          if (!live) break;
          tc_fence_after();
          const uint64_t da = make_smem_desc(s0 + (j < 4 ? F::kOffV + s * 2 * kGroup : F::kOffR + s * kGroup), 16, 1024, 2);
          const uint64_t db = dq + j * 2 * F::kQGroup / 16;
          __syncwarp();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f16_ss(tm + F::kColS, da + k * 2, db + k * 2, idesc_s, j + k > 0);
            if (j < 4) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16_ss(tm + F::kColS, da + kGroup / 16 + k * 2, db + F::kQGroup / 16 + k * 2, idesc_s, 1u);
            } else {
              umma_commit(&aux->s_full);
              umma_commit(&aux->r_free[s]);
              if (t + 1 == w.n) umma_commit(&aux->q_free);
            }
          }
          __syncwarp();
        }
        live = live && mbar_wait_warp(&aux->p_full, it & 1);
        if (!live) break;
        tc_fence_after();
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          const uint32_t s = uniform(static_cast<uint32_t>(4 * it + j) % kPairs);
          const uint64_t dv = make_smem_desc(s0 + F::kOffV + s * 2 * kGroup, kGroup, 1024, 2);
          __syncwarp();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              umma_f16_ss(tm + F::kColO + j * kN, dv + k * 2048 / 16, dp + k * 16 * F::kRowBytes / 16, idesc_o, t + k > 0);
            umma_commit(&aux->v_free[s]);
            if (j == 3 && t + 1 == w.n) umma_commit(&aux->o_full);
          }
          __syncwarp();
        }
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
      if (piece > 0 && !mbar_wait_warp(&aux->q_free, (piece - 1) & 1)) break;
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
    if (p.debug_stall) mbar_wait_warp(&aux->stall, 0);  // test hook: runs into the wait limit
    int it = 0, piece = 0;
    while (w.next()) {
      const int row0 = w.mt * kN, valid = min(w.kv, w.u.cap);
      const int clean = w.u.limit(w.q, w.kv, row0 / p.num_heads) / kTok;  // tiles below are seen in full by every row
      if (tid < kN) aux->lim[tid] = w.u.limit(w.q, w.kv, min((row0 + tid) / p.num_heads, w.q - 1));
      meet();
      float m[kN], l[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j) m[j] = -INFINITY, l[j] = 0.f;
      for (int t = w.t0; t < w.t0 + w.n; ++t, ++it) {
        mbar_wait_warp(&aux->s_full, it & 1);
        tc_fence_after();
        uint32_t x[kN];
        tmem_ld_row<kN>(tl + F::kColS, x);
        tmem_wait_ld();
        const int tok = t * kTok + tid;
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
          float dm[kN];
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            const float mx = sl2 * fmaxf(fmaxf(aux->top[0][j], aux->top[1][j]), fmaxf(aux->top[2][j], aux->top[3][j]));
            const bool up = mx > m[j] + 8.f;
            dm[j] = up ? ex2(m[j] - mx) : 1.f;  // 0 while nothing has been seen
            if (up) m[j] = mx;
            l[j] *= dm[j];
          }
          if (t > w.t0) {  // the scores came after the last tile's P V: the output is at rest
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {
              uint32_t o[kN];
              tmem_ld_row<kN>(tl + F::kColO + b * kN, o);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < kN; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * dm[j]);
              tmem_st_row<kN>(tl + F::kColO + b * kN, o);
            }
            tmem_wait_st();
          }
        }
        // P over the last tile's, which its product has read by now
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
        uint8_t* dst = smem + F::kOffP + tid * F::kRowBytes;
        const int swap = kN == 16 ? (tid >> 2) & 1 : (tid >> 1) & 3;
#pragma unroll
        for (int q = 0; q < kN / 8; ++q)
          *reinterpret_cast<uint4*>(dst + ((q ^ swap) << 4)) =
              make_uint4(pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
        if (tok >= valid) {
          // rows past the request's length may hold NaN: weight 0 does not hide
          // them from the product, so they are cleared (the scores have read them)
          for (int j = 0; j < 4; ++j) {
            uint8_t* slot = smem + F::kOffV + (4 * it + j) % kPairs * 2 * kGroup + tid * 128;
#pragma unroll
            for (int q = 0; q < 16; ++q)
              *reinterpret_cast<uint4*>(slot + (q >> 3) * kGroup + (q & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux->p_full);
      }
      // the rows' sums, added in one order by all
      int col;
      const float sum = reduce_columns<kN>(l, lane, col, [](float a, float b) { return a + b; });
      aux->sum[warp][col] = sum;
      meet();
      const int64_t grow0 = w.tok * p.num_heads + row0;
      const int rows = static_cast<int>(min(static_cast<int64_t>(kN), min(static_cast<int64_t>(w.q) * p.num_heads - row0,
                                                                        p.num_tokens * p.num_heads - grow0)));
      const bool whole = w.starts && w.ends;
      const int64_t slot = (2 * run + (w.starts ? 1 : 0)) * kN;
      float inv[kN];
      int32_t info = 0;
      if (w.starts && !w.ends) {
        // the run that holds the unit's last tile
        const Sched& sc = aux->sched;
        const int64_t n_runs = min(static_cast<int64_t>(runs), sc.tiles);
        const int64_t last = sc.begin + (it - w.n) + w.unit_tiles - 1;
        const int64_t hi = ((last + 1) * n_runs + sc.tiles - 1) / sc.tiles - 1;
        info = pack_info(run, static_cast<int>(hi) - run + 1, tid & (kN - 1));
      }
      const bool write = !cta_aborted();
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const float s = (aux->sum[0][j] + aux->sum[1][j]) + (aux->sum[2][j] + aux->sum[3][j]);
        inv[j] = s == 0.f ? 0.f : 1.f / s;  // a NaN among the scores stays one
        if (tid == j && j < rows && write) {
          const float lse = s == 0.f ? -INFINITY : (m[j] + __log2f(s)) * 0.6931471805599453f;
          if (whole)
            p.lse[grow0 + j] = lse;
          else
            P.parts.lse[slot + j] = lse;
          if (w.starts) P.parts.row_info[grow0 + j] = info;
        }
      }
      mbar_wait_warp(&aux->o_full, piece & 1);
      tc_fence_after();
#pragma unroll 1
      for (int b = 0; b < 4; ++b) {
        uint32_t o[kN];
        tmem_ld_row<kN>(tl + F::kColO + b * kN, o);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          const float v = inv[j] == 0.f ? 0.f : __uint_as_float(o[j]) * inv[j];
          if (j < rows && write) {
            if (whole)
              static_cast<uint16_t*>(p.out)[(grow0 + j) * kLatentDim + b * kTok + tid] =
                  static_cast<uint16_t>(pack2<kFp16>(v, 0.f));
            else
              P.parts.o[(slot + j) * kLatentDim + b * kTok + tid] = v;
          }
        }
      }
      tc_fence_before();  // the next piece's first product comes after its P
      ++piece;
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
  const int bound = run_bound<kN, kTok>(p, kNumSMs);
  Params P;
  P.L = p;
  P.parts = partials<kN>(p, bound, workspace);
  P.box_rows = std::min(p.block_size, kTok);
  // cache rows as 9 groups of 64 values; a load is one group of one page (at most 128 rows). A cache without pages: a
  // map over one row that nothing in bounds reads.
  const uint64_t pool_rows = std::max<uint64_t>(1, static_cast<uint64_t>(p.num_blocks) * p.block_size);
  const void* base = p.num_blocks > 0 ? p.cache : p.query;
  const uint64_t extent[3] = {64, pool_rows, 9}, stride[2] = {kLatentRow * 2, 128};
  const uint64_t extent_q[3] = {64, static_cast<uint64_t>(p.num_tokens) * p.num_heads, 9};
  const uint32_t box[3] = {64, static_cast<uint32_t>(P.box_rows), 1}, box_q[3] = {64, kN, 9};
  if (!encode_tmap_nd(&P.map, base, 3, extent, stride, box) || !encode_tmap_nd(&P.map_q, p.query, 3, extent_q, stride, box_q))
    return cudaErrorInvalidValue;
  auto kern = latent_decode_few_kernel<kFp16, kN>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), Few<kN>::kSmem);
  if (e != cudaSuccess) return e;
  kern<<<bound, kThreads, Few<kN>::kSmem, stream>>>(P);
  e = cudaGetLastError();
  if (e != cudaSuccess || bound == 1) return e;
  return launch_combine<kFp16, kN>(p, P.parts, bound, stream);
}

// Query rows per request, on average (the lengths may be on the device).
int64_t mean_rows(const LatentDecodeLaunch& p) { return (p.num_tokens + p.batch - 1) / p.batch * p.num_heads; }

}  // namespace

size_t latent_decode_workspace(const LatentDecodeLaunch& p) {
  const int64_t rows = mean_rows(p);
  return rows <= 16   ? partial_bytes<16>(p, run_bound<16, kTok>(p, kNumSMs))
         : rows <= 32 ? partial_bytes<32>(p, run_bound<32, kTok>(p, kNumSMs))
                      : latent_decode_pair_workspace(p);
}

cudaError_t launch_latent_decode(const LatentDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream) {
  const int64_t rows = mean_rows(p);
  if (rows <= 16) return fp16 ? launch<true, 16>(p, workspace, stream) : launch<false, 16>(p, workspace, stream);
  if (rows <= 32) return fp16 ? launch<true, 32>(p, workspace, stream) : launch<false, 32>(p, workspace, stream);
  return launch_latent_decode_pair(p, fp16, workspace, stream);
}

}  // namespace cascade
