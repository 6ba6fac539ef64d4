// Attention over a 4-bit key-value cache (cascade_quant_decode) for many query rows
// per request and kv head (chunks of prompts, prefixes that a batch shares), on the
// tensor cores: bound by them, with the exponentials (16 per clock and SM) close
// behind.
//
// A block of 256 query rows (token and head of the group, in that order) of one
// request and kv head are two tiles of 128 that share the unpacked tokens, 64 at a
// time. Keys stay exact: with a group's centre c and scale s a value is
// (code - 8) s + s / 2 + c, and s is split in two, s = s1 + s2, of 7 and 4 significant
// bits, so that the whole numbers code - 8 times s1 and s2 are fp16 numbers for every s
// ((code - 7.5) s has a bit more than the smallest of them); the centres and scales
// meet the groups' sums of the query in a product of 16 more columns. 272 columns for
// 128 (a key rounded to fp16 would be 2^-11 off in each of its 128 products, the
// scores' sums in fp32 are not). Queries are fp16 too, each row times a power of two. Values are
// rounded to fp16 once.
//
// Warps: 0-3 softmax and output of tile A, a thread per row, 4-7 of tile B, 8 MMA
// issue, 9-15 unpack (9 loads, too). Per step j of 64 tokens the issue order is PV_A(j),
// S_A(j+1), PV_B(j), S_B(j+1), so one tile's products run beside the other's softmax;
// unpacked keys and values have two buffers. Tensor memory holds both tiles' queries
// (64 columns each; from shared memory a product with 64 tokens would wait for its
// 128 query rows, 49 cycles for 32), scores (64, P over them) and outputs (128).
//
// A CTA takes an equal run of steps over the units (request, block) of one kv head;
// what run boundaries cut is merged by quant_combine_kernel.
//
// Measured: 2,048 query tokens x 32 heads over 16,384 tokens 740 us, 697 TFLOP/s of the
// formula's products (17 columns of 16 are issued for its 8 in the scores); some 790 us
// at the power limit. The issuing warp is busy throughout: a step's products alone take
// some 650 cycles of a tile's 725. In place of this: two issuing warps 836 us (for 746),
// two threads per row 800, a quarter of the exponentials as polynomials 775.
#include <algorithm>
#include <cstddef>

#include "quant_decode.cuh"

namespace cascade {
namespace {

constexpr int kBlock = 256, kRows = 128, kTok = 64;
// What a new unit costs, in steps (queries, first tokens, output): 8 requests of 300 query tokens over 300 to 5,000 tokens,
// 8 x 4 heads, 219 us with 6, 232 with 2, 226 with 10; 16 of 32 over up to 8,000 115, 116, 120.
constexpr int kSetup = 6;
constexpr int kThreads = 16 * 32;
constexpr int kUnpackWarps = 7;
constexpr int kStages = 4;                       // steps loaded ahead, less one
constexpr int kRaw = kTok * kQuantRow;           // keys or values of a step as they lie
constexpr int kStageOut = 4 * 4096;              // a tile's output on its way: 128 bytes of each row of a warp's
constexpr int kPart = 8192;                      // of keys or values: 64 tokens x 64 values
constexpr int kOffOut = 0;                       // [tile]
constexpr int kOffK = kOffOut + 2 * kStageOut;   // [buffer][part of the scale][64 values' group][token]
constexpr int kOffV = kOffK + 8 * kPart;         // [buffer][64 values' group][token]
constexpr int kOffZq = kOffV + 4 * kPart;        // [tile][2 x 8 columns][128 rows][16 bytes]
constexpr int kOffZk = kOffZq + 2 * 4096;        // [buffer][2 x 8 columns][64 tokens][16 bytes]
constexpr int kOffRaw = kOffZk + 2 * 2048;       // [stage][keys, values]
constexpr int kBytes = kOffRaw + kStages * 2 * kRaw;

struct __align__(16) Aux {
  uint64_t raw_full[kStages], raw_empty[kStages], k_full[2], k_empty[2], v_full[2], v_empty[2];  // per buffer
  uint64_t q_full[2], s_full[2], p_full[2], o_final[2], stall, drain;                                      // per tile
  uint32_t odd;  // some group of a request's values was NaN
  uint32_t tmem_base;
  QuantRun run;
};
constexpr int kStaticBytes = 32;  // the wait state comes first
constexpr int kSmemBytes = (kStaticBytes + static_cast<int>(sizeof(Aux)) + 1023) / 1024 * 1024 + kBytes - kStaticBytes;
static_assert(kSmemBytes + kStaticBytes <= 227 * 1024, "shared memory per CTA");

struct Params {
  QuantDecodeLaunch L;
  CUtensorMap key, value;  // box: 80 bytes x box_rows cache rows of one head
  QuantPartials parts;
  int32_t box_rows;        // 16, 32 or 64
};

using Unit = QuantUnit<kBlock, kTok>;
using Walk = QuantWalk<kBlock, kTok, kSetup>;

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}
// the codes of a word, less 7.5 or (keys) 8: pairs of values (n, n + 4), n = 0..3
template <bool kKeys>
__device__ __forceinline__ void codes(uint32_t w, __half2 (&c)[4]) {
  const uint32_t lo = w << 1, hi = w >> 7, magic = 0x64006400u;
  const float less = kKeys ? 8.f : 7.5f;
  const __half2 a = __float2half2_rn(0.5f), b = __float2half2_rn(-512.f - less), d = __float2half2_rn(0.03125f), e = __float2half2_rn(-32.f - less);
  c[0] = __hfma2(as_half2(and_or(lo, 0x001E001Eu, magic)), a, b);
  c[1] = __hfma2(as_half2(and_or(lo, 0x01E001E0u, magic)), d, e);
  c[2] = __hfma2(as_half2(and_or(hi, 0x001E001Eu, magic)), a, b);
  c[3] = __hfma2(as_half2(and_or(hi, 0x01E001E0u, magic)), d, e);
}

// steps of tile t (128 rows) of a block, of the piece's `n` from step t0 on
__device__ __forceinline__ int tile_steps(const Unit& u, const Walk& w, int t) {
  const int first = w.block * kBlock + t * kRows, all = w.q * u.p.group;
  if (first >= all) return 0;
  const int last = (min(all, first + kRows) - 1) / u.p.group;
  return max(0, min(w.n, (u.limit(w.q, w.kv, last) + kTok - 1) / kTok - w.t0));
}

template <bool kFp16>
__global__ void __launch_bounds__(kThreads, 1) quant_tiles_kernel(const __grid_constant__ Params P) {
  const QuantDecodeLaunch& p = P.L;
  const Unit unit(p);
  const int h = static_cast<int>(blockIdx.x) % p.kv_heads, c = static_cast<int>(blockIdx.x) / p.kv_heads;
  extern __shared__ uint8_t smem_raw[];
  Aux* aux = reinterpret_cast<Aux*>(smem_raw);
  uint8_t* smem = smem_raw + sizeof(Aux) + ((0u - (smem_u32(smem_raw) + static_cast<uint32_t>(sizeof(Aux)))) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&aux->raw_full[i], 1);
      mbar_init(&aux->raw_empty[i], kUnpackWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&aux->k_full[i], kUnpackWarps);
      mbar_init(&aux->v_full[i], kUnpackWarps);
      mbar_init(&aux->k_empty[i], 1);
      mbar_init(&aux->v_empty[i], 1);
      mbar_init(&aux->q_full[i], 4);
      mbar_init(&aux->s_full[i], 1);
      mbar_init(&aux->p_full[i], 4);
      mbar_init(&aux->o_final[i], 1);
    }
    aux->odd = 0;
    mbar_init(&aux->stall, 1);
    mbar_init(&aux->drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&P.key);
    tma_prefetch_desc(&P.value);
  }
  if (warp == 8) {
    tmem_alloc(&aux->tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == 9) {
    const QuantRun r = find_run<kBlock, kTok, kSetup>(unit, c, P.parts.runs);
    if (lane == 0) {
      aux->run = r;
      // The second tile waits while units without rows for it are worked on, all of the run perhaps: 1.6 us a step
      // (measured), and as long again or twice if NaN values are looked for; requests without query tokens are passed by one after
      // the other.
      const uint64_t us = p.wait_limit_us ? p.wait_limit_us : kWaitLimitNs / 1000 + 8 * (r.end - r.begin) + 2ull * p.batch;
      cta_wait_init(us * 1000);
    }
  }
  if (warp == 10 && p.q_len == 0) {  // rows of tokens that are no request's: nothing to merge
    int64_t own = 0;
    for (int b = lane; b < p.batch; b += 32) own += min(max(p.q_lens[b], static_cast<int64_t>(0)), p.num_tokens);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) own += __shfl_xor_sync(0xffffffffu, own, d);
    for (int64_t i = min(own, p.num_tokens) * p.num_heads + blockIdx.x * 32 + lane; i < p.num_tokens * p.num_heads;
         i += static_cast<int64_t>(gridDim.x) * 32)
      P.parts.row_info[i] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = aux->tmem_base;
  const QuantRun run = aux->run;
  const bool any = c < run.runs;
  Walk walk(p, run);

  if (warp >= 9) {
    // ------------------------------------------------------------- unpack
    const int w = warp - 9;
    Walk load(p, run);
    const int shift = __ffs(p.block_size) - 1, oob = p.num_blocks ? p.num_blocks * p.block_size : 1, boxes = kTok / P.box_rows;
    int left = 0, step = 0, issued = 0;
    int32_t id = 0;
    bool more = any && w == 0;
    // (warp 9) page id of this lane's box of the next step, as loaded: not used, and so not waited for, until then
    auto next_ids = [&] {
      if (left == 0) {
        more = more && load.next();
        if (!more) return;
        left = load.n, step = load.t0;
      }
      const int at = step * kTok + lane * P.box_rows;
      id = lane < boxes && at < load.kv ? p.block_table[static_cast<int64_t>(load.b) * p.block_cols + (at >> shift)] : INT32_MIN;
    };
    auto issue = [&] {
      const int at = step * kTok + lane * P.box_rows, stage = issued % kStages;
      const bool good = static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks);
      if (!good && id != INT32_MIN) atomicOr(&g_cascade_device_error, kErrBadBlockId);
      const int row = good ? id * p.block_size + (at & (p.block_size - 1)) : oob;
      uint8_t* dst = smem + kOffRaw + stage * 2 * kRaw + lane * P.box_rows * kQuantRow;
      if (lane == 0) mbar_arrive_expect_tx(&aux->raw_full[stage], 2 * kRaw);
      __syncwarp();
      if (lane < boxes) {
        tma_load_3d(dst, &P.key, &aux->raw_full[stage], 0, row, h);
        tma_load_3d(dst + kRaw, &P.value, &aux->raw_full[stage], 0, row, h);
      }
      __syncwarp();
      ++issued, ++step, --left;
      next_ids();
    };
    if (more) {
      next_ids();
      for (int i = 0; i < kStages - 1 && more; ++i) issue();
    }
    const int t = lane & 3, g8 = (lane >> 3) + 4 * ((lane >> 2) & 1);  // rows 4 apart are 16 banks apart
    int n = 0;
    bool live = any;
    while (live && walk.next()) {
      for (int j = 0; live && j < walk.n; ++j, ++n) {
        const int stage = n % kStages, buf = n & 1, before = ((n >> 1) - 1) & 1;
        const uint8_t* raw = smem + kOffRaw + stage * 2 * kRaw;
        const int tok = (walk.t0 + j) * kTok, turn = (w + n) % kUnpackWarps;  // 8 tokens of keys, or values, at a time
        if (w == 0 && more && n > 0) {  // the stage of the step before is free, or nearly
          live = mbar_wait_warp(&aux->raw_empty[(n - 1) % kStages], ((n - 1) / kStages) & 1);
          if (live) issue();
        } else if (w == 0 && more) {
          issue();
        }
        live = live && mbar_wait_warp(&aux->raw_full[stage], (n / kStages) & 1) &&
               (n < 2 || mbar_wait_warp(&aux->k_empty[buf], before));
        if (!live) break;
        for (int i = turn; i < kTok / 8; i += kUnpackWarps) {
          const int r = i * 8 + g8;
          const uint4 word = *reinterpret_cast<const uint4*>(raw + r * kQuantRow + 16 * t);
          const uint4 par = *reinterpret_cast<const uint4*>(raw + r * kQuantRow + kQuantCodes);
          const uint32_t ws[4] = {word.x, word.y, word.z, word.w}, ps[4] = {par.x, par.y, par.z, par.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            __half2 cd[4];
            codes<true>(ws[k], cd);
            const __half2 s = __high2half2(as_half2(ps[k]));
            const __half2 s1 = as_half2(as_u32(s) & 0xFFF0FFF0u), s2 = __hsub2(s, s1);
            uint32_t x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = as_u32(__hmul2(cd[e], s1)), y[e] = as_u32(__hmul2(cd[e], s2));
            const int q = 4 * k + t;  // eight values
            uint8_t* dst = smem + kOffK + (buf * 4 + (q >> 3)) * kPart + r * 128 + (((q ^ r) & 7) << 4);
            *reinterpret_cast<uint4*>(dst) = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4*>(dst + 2 * kPart) = make_uint4(y[0], y[1], y[2], y[3]);
          }
          if (t < 2) {
            // the columns of centres and scales
            *reinterpret_cast<uint4*>(smem + kOffZk + buf * 2048 + t * 1024 + r * 16) = par;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux->k_full[buf]);
        live = n < 2 || mbar_wait_warp(&aux->v_empty[buf], before);
        if (!live) break;
        for (int i = kUnpackWarps - 1 - turn; i < kTok / 8; i += kUnpackWarps) {
          const int r = i * 8 + g8;
          const uint4 word = *reinterpret_cast<const uint4*>(raw + kRaw + r * kQuantRow + 16 * t);
          const uint4 par = *reinterpret_cast<const uint4*>(raw + kRaw + r * kQuantRow + kQuantCodes);
          const uint32_t ws[4] = {word.x, word.y, word.z, word.w}, ps[4] = {par.x, par.y, par.z, par.w};
          // (a group of values that is NaN is 0 here, so that rows that do not see it keep their sums)
          if (tok + r < walk.kv && (odd_par(ps[0]) || odd_par(ps[1]) || odd_par(ps[2]) || odd_par(ps[3]))) aux->odd = 1;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            __half2 cd[4];
            codes<false>(ws[k], cd);
            const uint32_t pk = tok + r >= walk.kv || odd_par(ps[k]) ? 0u : ps[k];
            const __half2 s = __high2half2(as_half2(pk)), off = __low2half2(as_half2(pk));
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = as_u32(__hfma2(cd[e], s, off));
            const int q = 4 * k + t;
            *reinterpret_cast<uint4*>(smem + kOffV + (buf * 2 + (q >> 3)) * kPart + r * 128 + (((q ^ r) & 7) << 4)) =
                make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&aux->v_full[buf]);
          mbar_arrive(&aux->raw_empty[stage]);
        }
      }
    }
    // an aborted call: the loads in flight (at most kStages steps') land before their warp leaves
    if (w == 0) {
      for (; n < issued; ++n) mbar_wait_drain(&aux->raw_full[n % kStages], (n / kStages) & 1);
    }
  } else if (warp == 8) {
    // ----------------------------------------------------------- MMA issuer
    const uint32_t idesc_s = make_idesc_f16(kRows, kTok, 0u, 0, 0);
    const uint32_t idesc_pv = make_idesc_f16(kRows, kHeadDim, 0u, 0, 1);
    const uint32_t tm = uniform(tbase), s0 = uniform(smem_u32(smem));
    auto scores = [&](int t, int buf, bool last) {
      const uint64_t dk = make_smem_desc(s0 + kOffK + buf * 4 * kPart, 16, 1024, 2);
      const uint64_t zq = make_smem_desc(s0 + kOffZq + t * 4096, 2048, 128, 0);
      const uint64_t zk = make_smem_desc(s0 + kOffZk + buf * 2048, 1024, 128, 0);
      tc_fence_after();
      if (elect_one()) {
        umma_f16_ss(tm + t * 64, zq, zk, idesc_s, 0);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ts(tm + t * 64, tm + 128 + t * 64 + k * 8, dk + ((part * 2 + k / 4) * kPart + k % 4 * 32) / 16, idesc_s, 1);
        }
        umma_commit(&aux->s_full[t]);
        if (last) umma_commit(&aux->k_empty[buf]);
      }
      __syncwarp();
    };
    auto values = [&](int t, int buf, bool fresh, bool last, bool final) {
      tc_fence_after();
      if (elect_one()) {
        // 64 tokens x two groups of 64 values, 8 KB apart
        const uint64_t dv = make_smem_desc(s0 + kOffV + buf * 2 * kPart, kPart, 1024, 2);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f16_ts(tm + 256 + t * 128, tm + t * 64 + k * 8, dv + k * 128, idesc_pv, !fresh || k > 0);
        if (last) umma_commit(&aux->v_empty[buf]);
        if (final) umma_commit(&aux->o_final[t]);
      }
      __syncwarp();
    };
    int n = 0, sc[2] = {0, 0}, pieces[2] = {0, 0};  // steps, and a tile's steps and pieces, so far
    bool live = any, used = false;
    while (live && walk.next()) {
      const int nt[2] = {tile_steps(unit, walk, 0), tile_steps(unit, walk, 1)};
      // (the last tile with rows has all the piece's steps, but for a unit whose rows see nothing: it has a step all the
      // same, without products)
      const int tl = nt[1] > 0 ? 1 : 0;
      used = true;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (live && nt[t] > 0) live = mbar_wait_warp(&aux->q_full[t], pieces[t]++ & 1);
      live = live && mbar_wait_warp(&aux->k_full[n & 1], (n >> 1) & 1);
      if (!live) break;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (nt[t] > 0) scores(t, uniform(n & 1), t == tl);
      if (nt[tl] == 0) {
        live = mbar_wait_warp(&aux->v_full[n & 1], (n >> 1) & 1);
        if (live && elect_one()) {
          umma_commit(&aux->k_empty[n & 1]);
          umma_commit(&aux->v_empty[n & 1]);
        }
        __syncwarp();
        ++n;
        continue;
      }
      for (int j = 0; live && j < walk.n; ++j, ++n) {
        const int buf = uniform(n & 1);
        live = mbar_wait_warp(&aux->v_full[buf], (n >> 1) & 1);
        bool have_k = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!live || j >= nt[t]) continue;
          live = mbar_wait_warp(&aux->p_full[t], sc[t]++ & 1);
          if (live) values(t, buf, j == 0, t == tl, j + 1 == nt[t]);
          if (live && j + 1 < nt[t]) {
            live = have_k || mbar_wait_warp(&aux->k_full[buf ^ 1], ((n + 1) >> 1) & 1);
            have_k = true;
            if (live) scores(t, buf ^ 1, t == tl);
          }
        }
      }
    }
    // Products may be in flight when another warp gives up, also after the last one was issued: they end before this warp
    // frees the tensor memory.
    if (used) {
      if (elect_one()) umma_commit(&aux->drain);
      __syncwarp();
      if (lane == 0) mbar_wait_drain(&aux->drain, 0);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------- softmax, output of tile t
    const int t = warp >> 2, r = tid & 127;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t scol = tbase + lane_off + t * 64, qcol = tbase + lane_off + 128 + t * 64, ocol = tbase + lane_off + 256 + t * 128;
    if (p.debug_stall && any) mbar_wait_warp(&aux->stall, 0);  // test hook: runs into the wait limit
    int sc = 0, pieces = 0;  // steps and pieces of this tile so far
    while (any && walk.next()) {
      const int rows = min(kBlock, walk.q * p.group - walk.block * kBlock);  // of the block
      const int row = t * kRows + r, at = walk.block * kBlock + row, i = at / p.group;
      const bool real = row < rows;
      const int64_t out_row = real ? (walk.tok + i) * p.num_heads + h * p.group + (at - i * p.group) : 0;
      const int mine = tile_steps(unit, walk, t);
      float mult = 0.f, ref = -INFINITY, bar_at = -INFINITY, gap = 0.f, l = 0.f;  // ref: the score whose weight is 2^6
      if (mine > 0) {
        // ------------------------------------------------------------ query
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.query) + out_row * kHeadDim);
        uint4 v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = real ? __ldg(src + k) : make_uint4(0u, 0u, 0u, 0u);
        auto value = [&](int k, int e) {
          const uint32_t w = e < 2 ? v[k].x : e < 4 ? v[k].y : e < 6 ? v[k].z : v[k].w;
          if constexpr (kFp16) return e & 1 ? __high2float(as_half2(w)) : __low2float(as_half2(w));
          return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
        };
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) top = fmax3f_nan(top, fabsf(value(k, e)), fabsf(value(k, e + 1)));
        }
        // times 2^up: [2^8, 2^9), or less for rows below 2^-119. A row with a NaN or an infinity is NaN.
        const int ex = max((__float_as_int(top) >> 23) & 255, 8), up = 135 - ex;
        const float f = ex == 255 ? __int_as_float(0x7fffffff) : __int_as_float((127 + up) << 23);
        uint8_t* z = smem + kOffZq + t * 4096 + r * 16;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float sums[2] = {0.f, 0.f};
          uint32_t qw[32];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = value(half * 8 + k, e) * f;
            sums[k >> 2] += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
#pragma unroll
            for (int e = 0; e < 4; ++e) qw[k * 4 + e] = pack2<true>(y[e], y[e + 4]);
          }
          tmem_st_32x32b_x32(qcol + half * 32, qw);
          // a centre meets the sum, a scale half of it, each as two fp16 numbers
          uint32_t z0[2], z1[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            z0[k] = pack2<true>(sums[k], 0.5f * sums[k]);
            const float2 hi = __half22float2(as_half2(z0[k]));
            z1[k] = pack2<true>(sums[k] - hi.x, 0.5f * sums[k] - hi.y);
          }
          *reinterpret_cast<uint2*>(z + half * 8) = make_uint2(z0[0], z0[1]);
          *reinterpret_cast<uint2*>(z + 2048 + half * 8) = make_uint2(z1[0], z1[1]);
        }
        // (not 0, nor NaN: a masked score, -inf, stays -inf)
        mult = fmaxf(__int_as_float((127 - up) << 23) * (p.scale * 1.4426950408889634f), 1e-37f);
        gap = 8.f / mult;
        fence_proxy_async_smem();
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux->q_full[t]);
      }
      // ---------------------------------------------------------- softmax
      const int lim = unit.limit(walk.q, walk.kv, min(at, walk.q * p.group - 1) / p.group) - walk.t0 * kTok;
      // steps below are seen in full by every row of the tile
      const int clean = min(walk.kv, unit.limit(walk.q, walk.kv, (walk.block * kBlock + t * kRows) / p.group)) / kTok - walk.t0;
      for (int j = 0; j < mine; ++j, ++sc) {
        mbar_wait_warp(&aux->s_full[t], sc & 1);
        tc_fence_after();
        uint32_t x[2][32];
        tmem_ld_32x32b_x32(scol, x[0]);
        tmem_ld_32x32b_x32(scol + 32, x[1]);
        tmem_wait_ld();
        if (j >= clean) {
          const int seen = lim - j * kTok;
#pragma unroll
          for (int e = 0; e < 64; ++e) x[e >> 5][e & 31] = e < seen ? x[e >> 5][e & 31] : 0xff800000u;
        }
        float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 64; e += 2)
          a[(e >> 1) & 3] = fmax3f_nan(a[(e >> 1) & 3], __uint_as_float(x[e >> 5][e & 31]), __uint_as_float(x[e >> 5][(e & 31) + 1]));
        const float top = fmax3f_nan(fmax3f_nan(a[0], a[1], a[2]), a[3], a[3]);
        // weights up to 2^6 after a move, to 2^14 before the next: fp16 holds 2^-24 of them
        const bool move = top > bar_at;
        const float dm = move ? ex2((ref - top) * mult) : 1.f;  // 0 while nothing has been seen
        if (move) ref = top, bar_at = __fadd_rd(top, gap);
        const float less = ref == -INFINITY ? 0.f : -ref;
        if (j > 0 && __any_sync(0xffffffffu, move)) {
          // the scores of step j come after P V of step j - 1: the output is at rest
#pragma unroll 1
          for (int g = 0; g < 8; ++g) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(ocol + g * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * dm);
            tmem_st_32x32b_x16(ocol + g * 16, o);
          }
        }
        float r0 = 0.f, r1 = 0.f, r2 = 0.f, r3 = 0.f;
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          const uint32_t* s = &x[e >> 5][e & 31];
          // (the difference first: beside a large product the rounding of a reference would be the weight)
          float y0 = __uint_as_float(s[0]), y1 = __uint_as_float(s[1]), y2 = __uint_as_float(s[2]), y3 = __uint_as_float(s[3]);
          fadd2(y0, y1, less, less);
          fadd2(y2, y3, less, less);
          ffma2_bcast(y0, y1, y0, y1, mult, 6.f);
          ffma2_bcast(y2, y3, y2, y3, mult, 6.f);
          y0 = ex2(y0), y1 = ex2(y1), y2 = ex2(y2), y3 = ex2(y3);
          fadd2(r0, r1, y0, y1);
          fadd2(r2, r3, y2, y3);
          pk[e >> 1] = pack2<true>(y0, y1);
          pk[(e >> 1) + 1] = pack2<true>(y2, y3);
        }
        tmem_st_32x32b_x32(scol, pk);  // over the scores' first half
        l = l * dm + ((r0 + r1) + (r2 + r3));
        if (!(top < INFINITY)) l = __int_as_float(0x7fffffff);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux->p_full[t]);
      }
      // ----------------------------------------------------------- output
      float inv = 0.f, lse = -INFINITY;
      uint32_t bad = 0;  // bit i: this row sees a NaN in the values' group i
      if (mine > 0) {
        mbar_wait_warp(&aux->o_final[t], pieces++ & 1);
        tc_fence_after();
        if (ref > -INFINITY || l != l) {  // (a NaN is no maximum)
          inv = 1.f / l;
          lse = fmaf(ref, mult * 0.6931471805599453f, (log2f(l) - 6.f) * 0.6931471805599453f);
          if (lse == INFINITY) inv = lse = __int_as_float(0x7fffffff);  // a score beyond fp32
        }
        if (*reinterpret_cast<volatile uint32_t*>(&aux->odd)) {  // (rarely) which rows see which: the piece's values are looked at again
          const int shift = __ffs(p.block_size) - 1, end = min(walk.kv, (walk.t0 + mine) * kTok);
          for (int tok = walk.t0 * kTok; tok < end; tok += 32) {
            uint32_t odd = 0;
            if (tok + lane < end) odd = odd_groups(p, walk.b, tok + lane, shift, h);
            for (uint32_t who = __ballot_sync(0xffffffffu, odd != 0); who; who &= who - 1) {
              const int l = __ffs(who) - 1;
              const uint32_t its = __shfl_sync(0xffffffffu, odd, l);
              if (tok + l - walk.t0 * kTok < lim) bad |= its;
            }
          }
        }
      }
      const bool whole = walk.starts && walk.ends, aborted = __any_sync(0xffffffffu, cta_aborted());
      const int64_t slot = ((static_cast<int64_t>(walk.starts ? 2 * c + 1 : 2 * c) * p.kv_heads + h) * kBlock) + t * kRows;
      if (real && !aborted) {
        if (walk.starts)
          P.parts.row_info[out_row] =
              walk.ends ? 0 : cut_info(run, c, walk.base + unit.tiles(walk.q, walk.kv, walk.block) - 1) + row;
        if (whole)
          p.lse[out_row] = lse;
        else
          P.parts.lse[slot + r] = lse;
      }
      // Through shared memory, 128 bytes of a row at a time (16-byte part q of row r at q ^ (r % 8)), so that a store
      // instruction writes whole lines of four rows. Values lie as their codes' pairs do: n, n + 4 of each eight.
      const int first_row = (r & ~31), here = min(32, rows - (t * kRows + first_row));
      uint8_t* stage = smem + kOffOut + warp * 4096;
      if (here > 0 && !aborted) {
#pragma unroll 1
        for (int g = 0; g < 4; ++g) {  // 32 values
          uint32_t o[32] = {};
          const float by = bad >> g & 1 ? __int_as_float(0x7fffffff) : inv;
          if (mine > 0) {
            tmem_ld_32x32b_x32(ocol + g * 32, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = inv == 0.f ? 0u : __float_as_uint(__uint_as_float(o[e]) * by);
          auto y = [&](int q, int n) { return __uint_as_float(o[q * 8 + n]); };
          if (whole) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((((g & 1) * 4 + q) ^ (lane & 7)) << 4)) =
                  make_uint4(pack2<kFp16>(y(q, 0), y(q, 2)), pack2<kFp16>(y(q, 4), y(q, 6)), pack2<kFp16>(y(q, 1), y(q, 3)),
                             pack2<kFp16>(y(q, 5), y(q, 7)));
            if (!(g & 1)) continue;
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((2 * q) ^ (lane & 7)) << 4)) =
                  make_uint4(o[q * 8], o[q * 8 + 2], o[q * 8 + 4], o[q * 8 + 6]);
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((2 * q + 1) ^ (lane & 7)) << 4)) =
                  make_uint4(o[q * 8 + 1], o[q * 8 + 3], o[q * 8 + 5], o[q * 8 + 7]);
            }
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int rr = k * 4 + (lane >> 3), q = lane & 7;
            const int64_t to = __shfl_sync(0xffffffffu, out_row, rr);
            const uint4 w = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((q ^ (rr & 7)) << 4));
            if (rr >= here) continue;
            if (whole)
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + to * kHeadDim + (g >> 1) * 64 + q * 8) = w;
            else
              *reinterpret_cast<uint4*>(P.parts.o + (slot + first_row + rr) * kHeadDim + g * 32 + q * 4) = w;
          }
          __syncwarp();
        }
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// Runs per kv head: a CTA per SM, no more than there are steps.
int run_count(const QuantDecodeLaunch& p) {
  const int64_t rows = p.num_tokens * p.group, units = p.batch + rows / kBlock;
  const int64_t steps = std::max<int64_t>(1, (static_cast<int64_t>(p.block_cols) * p.block_size + kTok - 1) / kTok);
  const int64_t most = std::min<int64_t>(units, 1 << 20) * (kSetup + steps);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({most, kNumSMs / p.kv_heads, kMaxRuns})));
}

template <bool kFp16>
cudaError_t launch(const QuantDecodeLaunch& p, void* workspace, cudaStream_t stream) {
  Params P;
  P.L = p;
  const int runs = run_count(p);
  P.parts = quant_partials(p, runs, kBlock, workspace);
  P.box_rows = std::min(kTok, p.block_size);
  // no pages at all: maps over a row of the query's stand in, nothing is loaded through them
  const bool any = p.num_blocks > 0;
  const uint64_t extent[3] = {kQuantRow, any ? static_cast<uint64_t>(p.num_blocks) * p.block_size : 1,
                              any ? static_cast<uint64_t>(p.kv_heads) : 1};
  const uint64_t stride[2] = {static_cast<uint64_t>(p.kv_heads) * kQuantRow, kQuantRow};
  const uint32_t box[3] = {kQuantRow, static_cast<uint32_t>(P.box_rows), 1};
  if (!encode_tmap_bytes(&P.key, any ? p.key : p.query, extent, stride, box) ||
      !encode_tmap_bytes(&P.value, any ? p.value : p.query, extent, stride, box))
    return cudaErrorInvalidValue;
  auto kern = quant_tiles_kernel<kFp16>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), kSmemBytes);
  if (e != cudaSuccess) return e;
  kern<<<static_cast<unsigned>(runs * p.kv_heads), kThreads, kSmemBytes, stream>>>(P);
  e = cudaGetLastError();
  if (e != cudaSuccess || runs == 1) return e;
  return launch_quant_combine<kFp16, kBlock>(p, P.parts, stream);
}

}  // namespace

size_t quant_tiles_workspace(const QuantDecodeLaunch& p) { return quant_partial_bytes(p, run_count(p), kBlock); }

cudaError_t launch_quant_tiles(const QuantDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream) {
  return fp16 ? launch<true>(p, workspace, stream) : launch<false>(p, workspace, stream);
}

}  // namespace cascade
