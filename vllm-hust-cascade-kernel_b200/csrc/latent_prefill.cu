// Latent attention, expanded form (cascade_latent_prefill), on the tensor cores.
//
// For a query row of head h: s_t = scale (<q[0:128], k_th> + <q[128:192], r_t>)
// over the sequence's keys it may see, out = sum_t softmax(s)_t v_th. 640 flops
// per (query, key, head): bound by the tensor cores, with the exponentials (16
// per clock and SM: 2,048 cycles for the 256 x 128 scores whose products take
// 2,700) close behind.
//
// One CTA computes 256 query tokens of one (sequence, head) as two tiles of 128
// that share the key and value tiles of 128 tokens; their softmax warpgroups
// alternate, so the tensor pipe has one tile's products while the other's
// softmax runs. Per key tile j the issue order is PV_A(j), S_A(j+1), PV_B(j),
// S_B(j+1). Scores S (fp32) and P (16-bit, over S's columns)
// of both tiles and both outputs fill the tensor memory (4 x 128 columns).
// Shared memory: the query tiles (96 KB) and a ring of eight 16 KB chunks for
// keys (three of 128 tokens x 64 dims, the third the shared rotary part) and
// values (two of 64 tokens x 128 dims).
//
// Softmax: two threads per row, 64 of a tile's 128 keys each (one thread took
// 2,180 cycles from scores to P, in which its tile's products stood still); the
// running maximum moves only when a score exceeds it by more than 2^8, so the
// output is rescaled rarely; sums of the exponentials in fp32.
//
// Causal: key tiles past a tile's last row are not computed, only tiles that
// cross the diagonal or the sequence's end are masked. CTAs go to the longest
// rows first, the pairs of one head next to one another (its keys and values
// stay in L2).
//
// Measured (two prompts of 6,350 and 7,150 tokens x 16 heads, 468 GFLOP, floor
// 282 us): 489 us per call in a loop, 956 TFLOP/s; 435 to 470 replayed in a graph,
// with the power cap. A step (256 x 128 scores) takes about
// 3,870 cycles, its products 2,700: a tile's scores wait for its P V, which waits
// for its softmax (1,900 cycles, 1,450 of them exponentials at 11 per clock) and
// two barrier hops, and tensor memory has no room for a third tile's scores.
//
// Warps: 0-7 softmax and output of tile A, 8-15 of tile B, 16 TMA, 17 MMA issue.
#include <algorithm>
#include <cstddef>

#include "kernels.h"
#include "ptx.cuh"

namespace cascade {
namespace {

constexpr int kRows = 128, kTok = 128;
constexpr int kThreads = 18 * 32;
constexpr int kChunk = 16384;
constexpr int kSlots = 8;
constexpr int kPolyOf8 = 2;  // of eight groups of four exponentials, those with two on the FMA pipe (0: 438, 2: 427, 4: 426, 8: 449 us
                             // on the two long prompts)
constexpr int kOffQ = 0;                        // [tile][3 chunks]
constexpr int kOffRing = kOffQ + 6 * kChunk;
constexpr int kBytes = kOffRing + kSlots * kChunk;

struct __align__(16) Aux {
  float shared[2][2][kRows];  // [tile][half of the keys]: the row's maximum, at the end its sum
  uint64_t q_full, k_full[2], v_full[2], v_empty[2], s_full[2][2], p_full[2], o_final[2], stall, drain;
  uint32_t tmem_base;
};
constexpr int kStaticBytes = 32;  // the wait state comes first
constexpr int kSmemBytes = (kStaticBytes + static_cast<int>(sizeof(Aux)) + 1023) / 1024 * 1024 + kBytes - kStaticBytes;
static_assert(kSmemBytes + kStaticBytes <= 227 * 1024, "shared memory per CTA");

struct Params {
  LatentPrefillLaunch L;
  CUtensorMap q, k, rope, v;
  int32_t k_head, v_head;  // 0: one head's keys (values) serve all
};

template <bool kFp16>
__global__ void __launch_bounds__(kThreads, 1) latent_prefill_kernel(const __grid_constant__ Params P) {
  const LatentPrefillLaunch& p = P.L;
  const int b = blockIdx.z, h = blockIdx.y;
  const int row0 = static_cast<int>(gridDim.x - 1 - blockIdx.x) * 2 * kRows;
  const int64_t q0 = p.cu_q[b], k0 = p.cu_kv[b];
  const int64_t nq = p.cu_q[b + 1] - q0, nk = p.cu_kv[b + 1] - k0;
  if (row0 >= nq || q0 < 0 || q0 + nq > p.num_tokens || k0 < 0 || nk < 0 || k0 + nk > p.num_kv) return;
  const int n = static_cast<int>(nq), m = static_cast<int>(nk);
  // keys that query token i sees
  auto limit = [&](int i) { return p.causal ? max(0, min(m, m - n + i + 1)) : m; };
  // key tiles of query tile t (0 if it has no rows): B's are at least A's, or none
  auto tiles = [&](int t) {
    const int first = row0 + t * kRows;
    return first < n ? (limit(min(n, first + kRows) - 1) + kTok - 1) / kTok : 0;
  };
  const int nt[2] = {tiles(0), tiles(1)};
  const int steps = max(nt[0], nt[1]);
  const int tl = nt[1] > 0 ? 1 : 0;  // the tile whose products come last in a step

  extern __shared__ uint8_t smem_raw[];
  Aux* aux = reinterpret_cast<Aux*>(smem_raw);
  uint8_t* smem = smem_raw + sizeof(Aux) + ((0u - (smem_u32(smem_raw) + static_cast<uint32_t>(sizeof(Aux)))) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    cta_wait_init(static_cast<uint64_t>(p.wait_limit_us) * 1000);
    mbar_init(&aux->q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&aux->k_full[i], 1);
      mbar_init(&aux->v_full[i], 1);
      mbar_init(&aux->v_empty[i], 1);
      mbar_init(&aux->s_full[i][0], 1);
      mbar_init(&aux->s_full[i][1], 1);
      mbar_init(&aux->p_full[i], 8);
      mbar_init(&aux->o_final[i], 1);
    }
    mbar_init(&aux->stall, 1);
    mbar_init(&aux->drain, 1);
    fence_mbar_init();
  }
  if (warp == 17) {
    tmem_alloc(&aux->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = aux->tmem_base;
  auto slot_of = [&](int q) { return smem + kOffRing + (q % kSlots) * kChunk; };  // chunk q of the load order

  if (warp == 16) {
    // ------------------------------------------------------------- producer
    // load order K(0), V(0), K(1), V(1), ...: chunks 5j + 0..2 and 5j + 3..4.
    // A chunk's slot was chunk q - 8's: K(j) replaces the end of K(j-2) and
    // V(j-2), V(j) the start of K(j-1). s_full of a tile also says that what
    // was issued before it is done.
    bool live = true;
    if (steps > 0 && elect_one()) {
      // (a tile without products stages its rows of zeros in its part at once: nothing may land there)
      const int first = nt[0] > 0 ? 0 : 1;
      mbar_arrive_expect_tx(&aux->q_full, (tl + 1 - first) * 3 * kChunk);
      for (int t = first; t <= tl; ++t)
        for (int c = 0; c < 3; ++c)
          tma_load_3d(smem + kOffQ + (t * 3 + c) * kChunk, &P.q, &aux->q_full, 0,
                      static_cast<int>(q0) + row0 + t * kRows, h * 3 + c);
    }
    __syncwarp();
    for (int j = 0; live && j < steps; ++j) {
      const int tok = static_cast<int>(k0) + j * kTok;
      live = j < 2 || mbar_wait_warp(&aux->v_empty[j & 1], ((j >> 1) - 1) & 1);
      if (!live) break;
      if (elect_one()) {
        uint64_t* bar = &aux->k_full[j & 1];
        mbar_arrive_expect_tx(bar, 3 * kChunk);
        for (int c = 0; c < 2; ++c) tma_load_4d(slot_of(5 * j + c), &P.k, bar, 0, tok, c, h * P.k_head);
        tma_load_3d(slot_of(5 * j + 2), &P.rope, bar, 0, tok, 0);
      }
      __syncwarp();
      live = j < 1 || mbar_wait_warp(&aux->s_full[tl][(j - 1) & 1], ((j - 1) >> 1) & 1);
      if (!live) break;
      if (elect_one()) {
        uint64_t* bar = &aux->v_full[j & 1];
        mbar_arrive_expect_tx(bar, 2 * kChunk);
        for (int c = 0; c < 2; ++c) tma_load_4d(slot_of(5 * j + 3 + c), &P.v, bar, 0, tok + c * 64, 0, h * P.v_head);
      }
      __syncwarp();
    }
  } else if (warp == 17) {
    // ----------------------------------------------------------- MMA issuer
    constexpr uint32_t fmt = kFp16 ? 0u : 1u;
    const uint32_t idesc_s = make_idesc_f16(kRows, kTok, fmt, 0, 0);
    const uint32_t idesc_pv = make_idesc_f16(kRows, kPrefillDv, fmt, 0, 1);
    const uint32_t tm = uniform(tbase), s0 = uniform(smem_u32(smem));
    auto scores = [&](int t, int j) {
      const uint32_t u = uniform(static_cast<uint32_t>(j));
      const uint64_t dq = make_smem_desc(s0 + kOffQ + t * 3 * kChunk, 16, 1024, 2);
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < 3; ++c) {
          const uint64_t dk = make_smem_desc(s0 + kOffRing + (5 * u + c) % kSlots * kChunk, 16, 1024, 2);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ss(tm + t * 128, dq + (c * kChunk + k * 32) / 16, dk + k * 2, idesc_s, c + k > 0);
        }
        umma_commit(&aux->s_full[t][j & 1]);
      }
      __syncwarp();
    };
    auto values = [&](int t, int j, bool last) {
      const uint32_t u = uniform(static_cast<uint32_t>(j));
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          // 64 tokens x two groups of 64 dims, 8 KB apart
          const uint64_t dv = make_smem_desc(s0 + kOffRing + (5 * u + 3 + c) % kSlots * kChunk, kChunk / 2, 1024, 2);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ts(tm + 256 + t * 128, tm + t * 128 + c * 64 + k * 8, dv + k * 128, idesc_pv,
                        j > 0 || c + k > 0);
        }
        if (t == tl) umma_commit(&aux->v_empty[j & 1]);
        if (last) umma_commit(&aux->o_final[t]);
      }
      __syncwarp();
    };
    bool live = steps > 0 && mbar_wait_warp(&aux->q_full, 0) && mbar_wait_warp(&aux->k_full[0], 0);
    if (live) {
      if (nt[0] > 0) scores(0, 0);
      if (nt[1] > 0) scores(1, 0);
    }
    for (int j = 0; live && j < steps; ++j) {
      live = mbar_wait_warp(&aux->v_full[j & 1], (j >> 1) & 1);
      bool have_k = false;
      for (int t = 0; live && t < 2; ++t) {
        if (j >= nt[t]) continue;
        live = mbar_wait_warp(&aux->p_full[t], j & 1);
        if (!live) break;
        values(t, j, j + 1 == nt[t]);
        if (j + 1 < nt[t]) {
          live = have_k || mbar_wait_warp(&aux->k_full[(j + 1) & 1], ((j + 1) >> 1) & 1);
          have_k = true;
          if (live) scores(t, j + 1);
        }
      }
    }
    if (steps > 0 && !live && lane == 0) {
      umma_commit(&aux->drain);
      mbar_wait_drain(&aux->drain, 0);
    }
  } else {
    // ------------------------------------------------- softmax, output of tile t
    const int t = warp >> 3, hh = (warp >> 2) & 1, r = tid & 127, row = row0 + t * kRows + r;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t scol = tbase + lane_off + t * 128, ocol = tbase + lane_off + 256 + t * 128 + hh * 64;
    const float sl2 = p.scale * 1.4426950408889634f;
    const int mine = t ? nt[1] : nt[0];
    const int lim = limit(min(row, n - 1));
    const int clean = limit(min(row0 + t * kRows, n - 1)) / kTok;  // tiles below are seen in full by every row
    // the two warps of 32 rows meet here; neither leaves the loop early (an aborted CTA's waits return at once), so
    // neither is waited for in vain
    auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + t * 4 + (warp & 3)) : "memory"); };
    float mx = -INFINITY, l = 0.f;
    if (p.debug_stall) mbar_wait_warp(&aux->stall, 0);  // test hook: runs into the wait limit
    for (int j = 0; j < mine; ++j) {
      mbar_wait_warp(&aux->s_full[t][j & 1], (j >> 1) & 1);
      tc_fence_after();
      const int seen = j >= clean ? lim - j * kTok - hh * 64 : 64;
      auto load = [&](int g, uint32_t (&x)[32]) {
        tmem_ld_32x32b_x32(scol + hh * 64 + g * 32, x);
        tmem_wait_ld();
        if (j >= clean) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = g * 32 + e < seen ? x[e] : 0xff800000u;
        }
      };
      float a0 = -INFINITY, a1 = -INFINITY, a2 = -INFINITY, a3 = -INFINITY;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t x[32];
        load(g, x);
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          a0 = fmax3f_nan(a0, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
          a1 = fmax3f_nan(a1, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
          a2 = fmax3f_nan(a2, __uint_as_float(x[e + 4]), __uint_as_float(x[e + 5]));
          a3 = fmax3f_nan(a3, __uint_as_float(x[e + 6]), __uint_as_float(x[e + 7]));
        }
      }
      a0 = fmax3f_nan(fmax3f_nan(a0, a1, a2), a3, a3);
      aux->shared[t][hh][r] = a0;
      meet();
      const float top = fmax3f_nan(a0, aux->shared[t][hh ^ 1][r], a0) * sl2;
      const bool move = top > mx + 8.f;
      const float dm = move ? ex2(mx - top) : 1.f;  // 0 while nothing has been seen
      if (move) mx = top;
      const float neg = mx == -INFINITY ? 0.f : -mx;
      if (j > 0 && __any_sync(0xffffffffu, move)) {
        // the scores of tile j come after P V of tile j - 1: the output is at rest
#pragma unroll 1
        for (int g = 0; g < 2; ++g) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(ocol + g * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * dm);
          tmem_st_32x32b_x32(ocol + g * 32, o);
        }
      }
      // P goes over the first 32 columns of this half's own scores, read by then
      float r0 = 0.f, r1 = 0.f, r2 = 0.f, r3 = 0.f;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t x[32], pk[16];
        load(g, x);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float y0, y1, y2, y3;
          ffma2_bcast(y0, y1, __uint_as_float(x[e]), __uint_as_float(x[e + 1]), sl2, neg);
          ffma2_bcast(y2, y3, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]), sl2, neg);
          y0 = ex2(y0), y1 = ex2(y1);
          if (e / 4 < kPolyOf8) {
            ex2_poly2(y2, y3);
          } else {
            y2 = ex2(y2), y3 = ex2(y3);
          }
          fadd2(r0, r1, y0, y1);
          fadd2(r2, r3, y2, y3);
          pk[e >> 1] = pack2<kFp16>(y0, y1);
          pk[(e >> 1) + 1] = pack2<kFp16>(y2, y3);
        }
        tmem_st_32x32b_x16(scol + hh * 64 + g * 16, pk);
      }
      l = l * dm + ((r0 + r1) + (r2 + r3));
      // the exponentials on the FMA pipe lose a NaN: a score's own, or inf - inf of a score of +inf
      if (!(top < INFINITY)) l = __int_as_float(0x7fffffff);
      if ((j + 1) * kTok > m && (t == 0 || j >= nt[0]) && hh == 0) {
        // rows past the sequence may hold NaN, which weight 0 does not hide from
        // the product: the tile whose product comes first clears them
        mbar_wait_warp(&aux->v_full[j & 1], (j >> 1) & 1);
        if (j * kTok + r >= m) {
          uint8_t* chunk = slot_of(5 * j + 3 + (r >> 6)) + (r & 63) * 128;
#pragma unroll
          for (int q = 0; q < 16; ++q)
            *reinterpret_cast<uint4*>(chunk + (q >> 3) * (kChunk / 2) + (((q ^ r) & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&aux->p_full[t]);
    }
    float inv = 0.f, lse = -INFINITY;
    if (mine > 0) {
      mbar_wait_warp(&aux->o_final[t], 0);  // both warps have read the maxima: the slots take the sums
      tc_fence_after();
      aux->shared[t][hh][r] = l;
      meet();
      l = aux->shared[t][0][r] + aux->shared[t][1][r];
      if (mx > -INFINITY || l != l) {  // (a NaN is no maximum)
        inv = 1.f / l;
        lse = (mx + __log2f(l)) * 0.6931471805599453f;
      }
    }
    // output: 128 bytes per row and warp through the query tile's shared memory (done with; 16-byte chunk q of
    // row r at q ^ (r % 8)), so that a store instruction writes whole lines of four rows
    const int rows = min(32, n - (row0 + t * kRows + (r & ~31)));  // this warp's
    uint8_t* stage = smem + kOffQ + t * 3 * kChunk + (warp & 7) * 4096;
    if (rows > 0 && !__any_sync(0xffffffffu, cta_aborted())) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t o[32] = {};
        if (mine > 0) {
          tmem_ld_32x32b_x32(ocol + g * 32, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = q * 8 + i * 2;
            w[i] = inv == 0.f ? 0u : pack2<kFp16>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
          }
          *reinterpret_cast<uint4*>(stage + lane * 128 + (((g * 4 + q) ^ (lane & 7)) << 4)) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
      const int64_t first = (q0 + row0 + t * kRows + (r & ~31)) * p.num_heads + h;
      if (hh == 0 && lane < rows) p.lse[first + static_cast<int64_t>(lane) * p.num_heads] = lse;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int rr = i * 4 + (lane >> 3), q = lane & 7;
        const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((q ^ (rr & 7)) << 4));
        if (rr < rows)
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + (first + static_cast<int64_t>(rr) * p.num_heads) * kPrefillDv +
                                    hh * 64 + q * 8) = v;
      }
    }
  }
  if (cta_aborted()) {
    // loads may be in flight (at most 224 KB): they get a millisecond before the CTA leaves
    for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 1000 * 1000;) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

}  // namespace

cudaError_t launch_latent_prefill(const LatentPrefillLaunch& p, bool fp16, cudaStream_t stream) {
  Params P;
  P.L = p;
  P.k_head = p.key_hs != 0;
  P.v_head = p.value_hs != 0;
  // no keys at all: maps over the query stand in, nothing is loaded through them
  const bool any = p.num_kv > 0;
  const uint64_t T = static_cast<uint64_t>(p.num_tokens), S = any ? static_cast<uint64_t>(p.num_kv) : 1;
  const uint64_t H = static_cast<uint64_t>(p.num_heads);
  auto bytes = [](int64_t stride) { return static_cast<uint64_t>(stride) * 2; };
  const uint64_t q_extent[3] = {64, T, 3 * H}, q_stride[2] = {H * kPrefillDk * 2, 128};
  const uint32_t q_box[3] = {64, kRows, 1}, k_box[4] = {64, kTok, 1, 1}, v_box[4] = {64, 64, 2, 1}, r_box[3] = {64, kTok, 1};
  const uint64_t k_extent[4] = {64, S, 2, P.k_head ? H : 1}, v_extent[4] = {64, S, 2, P.v_head ? H : 1};
  const uint64_t k_stride[3] = {bytes(p.key_ts), 128, P.k_head ? bytes(p.key_hs) : 256};
  const uint64_t v_stride[3] = {bytes(p.value_ts), 128, P.v_head ? bytes(p.value_hs) : 256};
  const uint64_t r_extent[3] = {64, S, 1}, r_stride[2] = {bytes(p.rope_ts), 128};
  if (!encode_tmap_nd(&P.q, p.query, 3, q_extent, q_stride, q_box) ||
      !encode_tmap_nd(&P.k, any ? p.key : p.query, 4, k_extent, k_stride, k_box) ||
      !encode_tmap_nd(&P.v, any ? p.value : p.query, 4, v_extent, v_stride, v_box) ||
      !encode_tmap_nd(&P.rope, any ? p.key_rope : p.query, 3, r_extent, r_stride, r_box))
    return cudaErrorInvalidValue;
  auto kern = fp16 ? latent_prefill_kernel<true> : latent_prefill_kernel<false>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), kSmemBytes);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>((p.max_q + 2 * kRows - 1) / (2 * kRows)), p.num_heads, p.batch);
  kern<<<grid, kThreads, kSmemBytes, stream>>>(P);
  return cudaGetLastError();
}

}  // namespace cascade
