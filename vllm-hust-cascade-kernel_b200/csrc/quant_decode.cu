// Attention over a 4-bit key-value cache (cascade_quant_decode) for few query
// rows per request and kv head: bound by reading the cache, 160 bytes per token
// and kv head, with the unpacking of its 256 codes close behind.
//
// The codes go to the tensor cores as they are. With a group's centre c and scale
// s, a key's score is sum over its groups of
//   s <q, code> + (c - 7.5 s) sum q,
// so a nibble, masked in place, is an operand: in fp16 the bits 0..3 hold code *
// 2^-24 and the bits 4..7 code * 2^-20 (subnormals, exact), and q takes the factors
// 2^24 and 2^20 (a row is first scaled by a power of two to [2^13, 2^14), so 16-bit
// queries stay exact down to 2^-27 of their row's largest value). One AND per two
// codes, and a shift per eight. The term of centres and scales is one more product
// of 16 columns: (c, s) of four groups against sum q and -7.5 sum q, each as two
// fp16 numbers. fp32 holds every sum. (mma.sync aligns products as if a subnormal
// operand were 2^-14. So the codes' sums keep some 2^-22 of sum |q k| with fp16 queries: a
// log-sum-exp is 1.4e-7 to 1.1e-6 of its size off, 3e-8 to 2e-7 as fp32 products; with bf16
// queries 6e-8 to 3e-7. And where all of a key's centres and scales are that small, at
// 2^-24 a score is 2^-18 of it off. As tf32 products those would not be: 128 x 64 heads 169
// us for 166, 96 x 16 rows over 4,000 tokens 180 for 172.)
// Values are converted, (code - 7.5) s + c in one fused multiply-add, rounded to
// fp16, as P is: fp16 holds 2^-11 of both where bf16 would hold 2^-8.
//
// mma.sync m16n8k16 has the tokens as its M (scores) and the head's values as its
// M (output), the query rows as its N, so eight rows cost eight columns, and the
// probabilities' fragments turn by one movmatrix. (tcgen05 would need M = 128 of
// tokens, converted through shared memory; here 16 of 128 lanes' worth of rows
// exist. With 32 rows the tcgen05 kernel is the slower one, as row_blocks says.)
//
// A warp has one kv head's rows, their softmax and output, over a run of 32-token
// tiles; the warps of up to eight heads share the tiles' ring, which the first of
// them keeps filled by TMA. The place of a token in the MMA's rows (Places)
// keeps every shared-memory load of 80-byte rows free of bank conflicts.
// The running maxima move only when a score exceeds its row's by more than 2^8.
//
// 8 kv heads x 8 query heads: 128 requests of 1,500 to 8,200 tokens (798 MB) 166 us,
// 4.8 TB/s; 149 without the arithmetic, of which 8 for the start (lengths, run, page
// ids, first tile) and 4 for the merge. One request of 900 tokens 14.3 us.
#include <algorithm>
#include <type_traits>

#include "quant_decode.cuh"

namespace cascade {
namespace {

constexpr int kTok = 32;     // tokens per tile
// What a new unit costs, in tiles: its page ids, query rows and output. 24 to 48 requests of 1 to 6,000 tokens and 4 to 8
// heads' rows: 52.4, 57.3, 54.1 us with 6, 63.1, 63.7, 59.4 with 2, 51.4, 58.2, 54.9 with 10, 53.3, 59.6, 56.6 with 16; 96
// requests of up to 700 tokens would have it less: 25.9 with 6, 25.0 with 2.
constexpr int kSetup = 6;
constexpr int kTileBytes = kTok * kQuantRow;  // of keys or of values
constexpr int32_t kNoPage = INT32_MIN;
constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u;

template <int kN>  // query rows / 8
struct Shape {
  static constexpr int kRows = 8 * kN;
  static constexpr int kWarps = kN == 1 ? 16 : kN == 2 ? 12 : 8;  // (128, 168, 255 registers)
  static constexpr int kStages = kN < 3 ? 2 : 3;                  // tiles per group
  static constexpr int kHeads = kN == 2 ? 4 : 8;                  // most kv heads per group
  static constexpr int kRing = kWarps * kStages * 2 * kTileBytes;
  // the queries' fragments: in registers, or in shared memory ([warp][8 rows][group of 32 values][lane])
  static constexpr int kQuery = kN == 1 ? 0 : kWarps * kN * 4 * 32 * 16;
  static constexpr int kSmem = kRing + kQuery + 128;  // (to align the ring: the TMA writes to 128-byte boundaries)
  static_assert(kSmem + 1024 <= 227 * 1024, "shared memory per CTA");
};

struct Params {
  QuantDecodeLaunch L;
  CUtensorMap key, value;  // box: `box_rows` cache rows of the group's heads, [heads or pairs][rows][kStride bytes]
  QuantPartials parts;
  int32_t box_rows;     // 16 or 32
  int32_t row_shift;    // map rows are 2^row_shift cache rows (one kv head: 8 rows, 640 bytes)
  int32_t heads;        // kv heads per group
  int32_t head_groups;  // of the kv heads
  int32_t groups;       // per CTA
};

__device__ __forceinline__ uint32_t trans8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ float high_half(uint32_t x) { return __high2float(as_half2(x)); }
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}
// One nibble of two tokens' half words as code - 7.5, exactly: over fp16's 1024 the bits 1..4 are 1024 + 2 code, the bits 5..8
// 1024 + 32 code. (At bit 0 the 7.5 would be half a step.)
__device__ __forceinline__ __half2 low_code(uint32_t x, uint32_t magic) {
  return __hfma2(as_half2(and_or(x, 0x001E001Eu, magic)), __float2half2_rn(0.5f), __float2half2_rn(-519.5f));
}
__device__ __forceinline__ __half2 high_code(uint32_t x, uint32_t magic) {
  return __hfma2(as_half2(and_or(x, 0x01E001E0u, magic)), __float2half2_rn(0.03125f), __float2half2_rn(-39.5f));
}

// d = a b, nothing added
__device__ __forceinline__ void mma_fresh(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// The places of 16 tokens: row m = g of the scores' product is token_of(g), row g + 8 the one kNext after it, so the
// probabilities' columns 2 t, 2 t + 8 are token_of(2 t) and kNext after, 2 t + 1 and 2 t + 9 token_of(2 t + 1) and kNext after.
// Shared memory holds rows kStride bytes apart (two heads side by side, or one): rows g, g + 1 are 16 banks apart for the keys'
// loads, four even (or odd) rows 8 banks apart each for the values'.
template <int kStride>
struct Places;
template <>
struct Places<80> {
  static constexpr int kNext = 1;
  static __device__ __forceinline__ int token_of(int g) { return g & 1 ? 8 + ((g + 3) & 7) : g; }
};
template <>
struct Places<160> {
  static constexpr int kNext = 8;
  static __device__ __forceinline__ int token_of(int g) { return g & 1 ? 4 + (((g >> 1) + 2) & 3) : g >> 1; }
};

template <bool kFp16, int kN, int kStride>
__global__ void __launch_bounds__(32 * Shape<kN>::kWarps, 1) quant_decode_kernel(const __grid_constant__ Params P) {
  using S = Shape<kN>;
  constexpr int kRows = S::kRows, kStages = S::kStages, kWarps = S::kWarps;
  extern __shared__ uint8_t smem_raw[];
  using Pl = Places<kStride>;
  constexpr int kNext = Pl::kNext * kStride;
  __shared__ uint64_t full[kWarps][kStages], empty[kWarps][kStages];  // per group
  __shared__ uint64_t stall;
  __shared__ QuantRun found[kWarps];
  __shared__ uint32_t odd[kWarps];  // a tile whose rows see different tokens held a NaN among its values
  const QuantDecodeLaunch& p = P.L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem_raw + ((0u - smem_u32(smem_raw)) & 127u);
  pdl_launch_dependents();
  const int group = warp / P.heads, member = warp - group * P.heads;
  const int id = blockIdx.x * P.groups + group, head0 = id % P.head_groups * P.heads, h = head0 + member, c = id / P.head_groups;
  if (lane == 0) odd[warp] = 0;
  if (lane < kStages && member == 0) {
    mbar_init(&full[group][lane], 1);
    mbar_init(&empty[group][lane], min(P.heads, p.kv_heads - head0));
    fence_mbar_init();
  }
  if (threadIdx.x == 32 * (kWarps - 1)) {
    cta_wait_init(static_cast<uint64_t>(p.wait_limit_us) * 1000);
    mbar_init(&stall, 1);
    fence_mbar_init();
    tma_prefetch_desc(&P.key);
    tma_prefetch_desc(&P.value);
  }
  const QuantUnit<kRows, kTok> unit(p);
  if (member == 0) {
    const QuantRun r = find_run<kRows, kTok, kSetup>(unit, c, P.parts.runs);
    if (lane == 0) found[group] = r;
  }
  __syncthreads();
  const QuantRun run = found[group];
  if (p.q_len == 0) {  // rows of tokens that are no request's: nothing to merge
    int64_t own = 0;
    for (int b = lane; b < p.batch; b += 32) own += min(max(p.q_lens[b], static_cast<int64_t>(0)), p.num_tokens);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) own += __shfl_xor_sync(0xffffffffu, own, d);
    for (int64_t i = min(own, p.num_tokens) * p.num_heads + blockIdx.x * blockDim.x + threadIdx.x;
         i < p.num_tokens * p.num_heads; i += static_cast<int64_t>(gridDim.x) * blockDim.x)
      P.parts.row_info[i] = 0;
  }
  if (group >= P.groups || h >= p.kv_heads || c >= run.runs) return;

  const int nz = P.heads * kQuantRow / kStride;                    // heads, or pairs of heads, of a box
  const int stage_bytes = P.heads * 2 * kTileBytes;                // keys, then values
  uint8_t* mine = ring + group * kStages * stage_bytes;
  const uint32_t head_off = (kStride == 160 ? member >> 1 : member) * P.box_rows * kStride + (kStride == 160 ? (member & 1) * kQuantRow : 0);
  const uint32_t base = smem_u32(mine) + head_off;
  const uint32_t value_off = P.heads * kTileBytes, half_off = P.box_rows == 16 ? nz * 16 * kStride : 16 * kStride;  // (16 tokens on)
  uint8_t* query = ring + S::kRing + warp * (S::kQuery / kWarps);  // this warp's
  const uint32_t query_at = smem_u32(query);
  int issued = 0, done = 0;
  bool live = true;
  if (p.debug_stall) live = mbar_wait_warp(&stall, 0);  // test hook: runs into the wait limit

  uint32_t magic;  // (kept in a register: an immediate in the AND and one in the OR would take two instructions)
  asm volatile("mov.u32 %0, 0x64006400;" : "=r"(magic));

  // this lane's places in 16 tokens: keys' codes, their centres and scales; values' (of two of four tokens)
  const int tok_k = Pl::token_of(g), tok_v0 = Pl::token_of(2 * t), tok_v1 = Pl::token_of(2 * t + 1);
  const uint32_t off_k = tok_k * kStride + 16 * t, off_kp = tok_k * kStride + kQuantCodes;
  const uint32_t off_v0 = tok_v0 * kStride + 8 * g, off_v1 = tok_v1 * kStride + 8 * g;
  const uint32_t off_p0 = tok_v0 * kStride + kQuantCodes + 8 * (g & 1), off_p1 = tok_v1 * kStride + kQuantCodes + 8 * (g & 1);

  QuantWalk<kRows, kTok, kSetup> walk(p, run);
  const int shift = __ffs(p.block_size) - 1, oob = p.num_blocks ? p.num_blocks * p.block_size : 8;
  while (live && walk.next()) {
    // ---------------------------------------------------------------- loads
    // The group's first warp loads its tiles: page ids of the boxes (one or two per tile) of this lane's of 32 tiles, as
    // the maps' rows, and of the 32 tiles after them
    const bool two = P.box_rows < kTok;
    int rows_now[2], next_tile = walk.t0, rows_at = walk.t0;
    int32_t ids[2];
    auto load_ids = [&](int tile) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = tile * kTok + i * 16;
        // (a unit without tokens has a tile all the same: nothing of it is used)
        ids[i] = at < walk.kv && tile < walk.t0 + walk.n && (i == 0 || two)
                     ? p.block_table[static_cast<int64_t>(walk.b) * p.block_cols + (at >> shift)]
                     : kNoPage;
      }
    };
    auto to_rows = [&](int tile) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = tile * kTok + i * 16;
        const bool good = static_cast<uint32_t>(ids[i]) < static_cast<uint32_t>(p.num_blocks);
        rows_now[i] = (good ? ids[i] * p.block_size + (at & (p.block_size - 1)) : oob) >> P.row_shift;
        if (!good && ids[i] != kNoPage) atomicOr(&g_cascade_device_error, kErrBadBlockId);
      }
    };
    auto issue = [&] {
      if (next_tile - rows_at == 32) {
        rows_at = next_tile;
        to_rows(next_tile + lane);
        load_ids(next_tile + 32 + lane);
      }
      const int row0 = __shfl_sync(0xffffffffu, rows_now[0], next_tile - rows_at);
      const int row1 = two ? __shfl_sync(0xffffffffu, rows_now[1], next_tile - rows_at) : 0;
      const int stage = issued % kStages;
      if (issued >= kStages) live = live && mbar_wait_warp(&empty[group][stage], (issued / kStages - 1) & 1);
      if (live && elect_one()) {
        uint64_t* bar = &full[group][stage];
        uint8_t* dst = mine + stage * stage_bytes;
        const int z = head0 * kQuantRow / kStride;
        mbar_arrive_expect_tx(bar, stage_bytes);
        tma_load_3d(dst, &P.key, bar, 0, row0, z);
        tma_load_3d(dst + value_off, &P.value, bar, 0, row0, z);
        if (two) {
          tma_load_3d(dst + half_off, &P.key, bar, 0, row1, z);
          tma_load_3d(dst + value_off + half_off, &P.value, bar, 0, row1, z);
        }
      }
      __syncwarp();
      if (live) ++issued, ++next_tile;
    };
    if (member == 0) load_ids(walk.t0 + lane);

    // ---------------------------------------------------------------- query
    // row n of this block as the products' columns: lane (g, t) has d = 32 i + 8 t + 0..7 of row 8 n + g
    const int rows = min(kRows, walk.q * p.group - walk.block * kRows);  // of this unit
    auto row_of = [&](int r, int& i) {  // output row of row r of the unit, and its query token
      const int at = walk.block * kRows + r;
      i = at < p.group ? 0 : at / p.group;
      return (walk.tok + i) * p.num_heads + h * p.group + (at - i * p.group);
    };
    uint4 raw[kN][4];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      int i;
      const bool real = n * 8 + g < rows;
      const uint16_t* src = static_cast<const uint16_t*>(p.query) + row_of(real ? n * 8 + g : 0, i) * kHeadDim + 8 * t;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        raw[n][k] = real ? __ldg(reinterpret_cast<const uint4*>(src + 32 * k)) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (member == 0) {
      to_rows(walk.t0 + lane);
      load_ids(walk.t0 + 32 + lane);
      for (int i = 0; i < min(kStages, walk.n); ++i) issue();
    }

    uint32_t qf[1][16], zf[kN][2];  // qf: one block of rows' (others read theirs back)
    float mult[kN][2];   // of columns 2 t, 2 t + 1: score * scale * log2(e) per unit of the products
    int lim[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      float x[32], top = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t w[4] = {raw[n][k].x, raw[n][k].y, raw[n][k].z, raw[n][k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = kFp16 ? __half22float2(as_half2(w[e]))
                                 : make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
          x[8 * k + 2 * e] = f.x, x[8 * k + 2 * e + 1] = f.y;
          top = fmax3f_nan(top, fabsf(f.x), fabsf(f.y));
        }
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) top = fmax3f_nan(top, __shfl_xor_sync(0xffffffffu, top, d), top);
      // times 2^up: [2^13, 2^14), or less for rows below 2^-114. A row with a NaN or an infinity is NaN.
      const int ex = max((__float_as_int(top) >> 23) & 255, 13), up = 140 - ex;
      const float f = ex == 255 ? __int_as_float(0x7fffffff) : __int_as_float((127 + up) << 23);
      float sums[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float* y = x + 8 * k;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= f;
        float s = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        sums[k] = s + __shfl_xor_sync(0xffffffffu, s, 2);
        const uint32_t f[4] = {pack2<true>(y[0], y[4]), pack2<true>(y[1] * 0.0625f, y[5] * 0.0625f), pack2<true>(y[2], y[6]),
                               pack2<true>(y[3] * 0.0625f, y[7] * 0.0625f)};
        if constexpr (kN == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[0][4 * k + e] = f[e];
        } else {
          *reinterpret_cast<uint4*>(query + ((n * 4 + k) * 32 + lane) * 16) = make_uint4(f[0], f[1], f[2], f[3]);
        }
      }
      const float z = (t == 0 ? sums[0] : t == 1 ? sums[1] : t == 2 ? sums[2] : sums[3]) * 0x1p-14f, y = -7.5f * z;
      zf[n][0] = pack2<true>(z, y);
      const float2 hi = __half22float2(as_half2(zf[n][0]));
      zf[n][1] = pack2<true>(z - hi.x, y - hi.y);
      // (not 0, nor NaN: a masked score, -inf, stays -inf)
      const float m = fmaxf(__int_as_float((127 - up) << 23) * (p.scale * 1.4426950408889634f) * 0x1p14f, 1e-37f);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        int i;
        mult[n][k] = __shfl_sync(0xffffffffu, m, (2 * t + k) * 4);
        row_of(min(n * 8 + 2 * t + k, rows - 1), i);
        lim[n][k] = unit.limit(walk.q, walk.kv, i);
      }
    }
    if constexpr (kN > 1) __syncwarp();  // (a lane reads back what it wrote alone; this orders the asm loads behind it)
    int token;
    row_of(0, token);
    const int clean = min(walk.kv, unit.limit(walk.q, walk.kv, token));  // tokens below are seen by every row
    row_of(rows - 1, token);
    const int most = unit.limit(walk.q, walk.kv, token);  // tokens from here on by none

    float o[kN][8][4], sum[kN][2], less[kN][2], bar_at[kN][2];  // less: the negative of the score whose weight is 2^6
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int k = 0; k < 8; ++k) o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) sum[n][k] = less[n][k] = 0.f, bar_at[n][k] = -INFINITY;
    }

    // a tile: 32 tokens from `tok` on, their keys at shared address `ka`
    auto step = [&](uint32_t ka, int tok, auto masked) {
      float s[2][kN][4];
      uint32_t wa[2][4], wb[2][4], pa[2][4], pb[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t a = ka + (u ? half_off : 0);
        const uint4 wa4 = lds128(a + off_k), wb4 = lds128(a + off_k + kNext);
        const uint4 pa4 = lds128(a + off_kp), pb4 = lds128(a + off_kp + kNext);
        wa[u][0] = wa4.x, wa[u][1] = wa4.y, wa[u][2] = wa4.z, wa[u][3] = wa4.w;
        wb[u][0] = wb4.x, wb[u][1] = wb4.y, wb[u][2] = wb4.z, wb[u][3] = wb4.w;
        pa[u][0] = pa4.x, pa[u][1] = pa4.y, pa[u][2] = pa4.z, pa[u][3] = pa4.w;
        pb[u][0] = pb4.x, pb[u][1] = pb4.y, pb[u][2] = pb4.z, pb[u][3] = pb4.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a0[2][4], a1[2][4];
        float fa[2], fb[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t xa = wa[u][i] >> 8, xb = wb[u][i] >> 8;
          a0[u][0] = wa[u][i] & kLow, a0[u][1] = wb[u][i] & kLow, a0[u][2] = wa[u][i] & kHigh, a0[u][3] = wb[u][i] & kHigh;
          a1[u][0] = xa & kLow, a1[u][1] = xb & kLow, a1[u][2] = xa & kHigh, a1[u][3] = xb & kHigh;
          fa[u] = high_half(pa[u][i]), fb[u] = high_half(pb[u][i]);
        }
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          uint32_t q[4];
          if constexpr (kN == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = qf[0][4 * i + e];
          } else {
            const uint4 v = lds128(query_at + ((n * 4 + i) * 32 + lane) * 16);
            q[0] = v.x, q[1] = v.y, q[2] = v.z, q[3] = v.w;
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float x[4];
            mma_fresh(x, a0[u], q[0], q[1]);
            mma_16816<true>(x, a1[u], q[2], q[3]);
            if (i == 0) {
              s[u][n][0] = fa[u] * x[0], s[u][n][1] = fa[u] * x[1], s[u][n][2] = fb[u] * x[2], s[u][n][3] = fb[u] * x[3];
            } else {
              s[u][n][0] = fmaf(fa[u], x[0], s[u][n][0]), s[u][n][1] = fmaf(fa[u], x[1], s[u][n][1]);
              s[u][n][2] = fmaf(fb[u], x[2], s[u][n][2]), s[u][n][3] = fmaf(fb[u], x[3], s[u][n][3]);
            }
          }
        }
      }
      // centres: products of 2^-14 where the codes' are of 2^-24; in the larger unit `mult` holds for queries of any size
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t a = ka + (u ? half_off : 0) + off_kp + 4 * t;
        const uint32_t za = lds32(a), zb = lds32(a + kNext), z[4] = {za, zb, za, zb};
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          float x[4];
          mma_fresh(x, z, zf[n][0], zf[n][1]);
#pragma unroll
          for (int k = 0; k < 4; ++k) s[u][n][k] = fmaf(s[u][n][k], 0x1p10f, x[k]);
        }
      }
      const uint32_t va = ka + value_off;
      if constexpr (masked.value) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int mine = tok + u * 16 + tok_k;
#pragma unroll
          for (int n = 0; n < kN; ++n) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              s[u][n][k] = mine < lim[n][k] ? s[u][n][k] : -INFINITY;
              s[u][n][2 + k] = mine + Pl::kNext < lim[n][k] ? s[u][n][2 + k] : -INFINITY;
            }
          }
        }
      }
      bool move = false;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          move = move || fmaxf(fmax3f(s[0][n][k], s[0][n][2 + k], s[1][n][k]), s[1][n][2 + k]) > bar_at[n][k];
      }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float top = fmaxf(fmax3f(s[0][n][k], s[0][n][2 + k], s[1][n][k]), s[1][n][2 + k]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            if (top > bar_at[n][k]) {
              // weights up to 2^6 from here on, to 2^14 before the next move: fp16 holds 2^-24 of them
              const float f = bar_at[n][k] == -INFINITY ? 0.f : ex2((-less[n][k] - top) * mult[n][k]);
              less[n][k] = -top, bar_at[n][k] = __fadd_rd(top, 8.f / mult[n][k]);
              sum[n][k] *= f;
#pragma unroll
              for (int j = 0; j < 8; ++j) o[n][j][k] *= f, o[n][j][2 + k] *= f;
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t pf[kN][2];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          float e[4];
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            // (the difference first: beside a large product the rounding of a reference would be the weight)
            fadd2(s[u][n][k], s[u][n][k + 1], less[n][0], less[n][1]);
            e[k] = ex2(fmaf(s[u][n][k], mult[n][0], 6.f)), e[k + 1] = ex2(fmaf(s[u][n][k + 1], mult[n][1], 6.f));
          }
          sum[n][0] += e[0] + e[2], sum[n][1] += e[1] + e[3];
          pf[n][0] = trans8x8(pack2<true>(e[0], e[1]));
          pf[n][1] = trans8x8(pack2<true>(e[2], e[3]));
        }
        // values: lane (g, t) has d = words 2 g, 2 g + 1 of four tokens, whose groups are 2 (g % 2) and the next
        const uint32_t a = va + (u ? half_off : 0);
        const uint2 w[4] = {lds64(a + off_v0), lds64(a + off_v1), lds64(a + off_v0 + kNext), lds64(a + off_v1 + kNext)};
        uint2 par[4] = {lds64(a + off_p0), lds64(a + off_p1), lds64(a + off_p0 + kNext), lds64(a + off_p1 + kNext)};
        if constexpr (masked.value) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int mine = tok + u * 16 + (j & 1 ? tok_v1 : tok_v0) + (j >> 1) * Pl::kNext;
            // (a group of values that is NaN is 0 here, so that rows that do not see it keep their sums)
            if (mine >= most) par[j].x = par[j].y = 0;
            const bool bad_x = odd_par(par[j].x), bad_y = odd_par(par[j].y);
            if (bad_x) par[j].x = 0;
            if (bad_y) par[j].y = 0;
            if (bad_x || bad_y) odd[warp] = 1;
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          auto word = [&](int j) { return i ? w[j].y : w[j].x; };
          auto pr = [&](int j) { return i ? par[j].y : par[j].x; };
          __half2 sc[2], off[2];
          uint32_t x[2][2];  // [token pair][half of the word]
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            sc[j] = as_half2(__byte_perm(pr(2 * j), pr(2 * j + 1), 0x7632));
            off[j] = as_half2(__byte_perm(pr(2 * j), pr(2 * j + 1), 0x5410));
            x[j][0] = __byte_perm(word(2 * j), word(2 * j + 1), 0x5410);
            x[j][1] = __byte_perm(word(2 * j), word(2 * j + 1), 0x7632);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t y = k < 2 ? x[j >> 1][j & 1] << 1 : x[j >> 1][j & 1] >> 7;
              f[j] = as_u32(__hfma2(k & 1 ? high_code(y, magic) : low_code(y, magic), sc[j >> 1], off[j >> 1]));
            }
#pragma unroll
            for (int n = 0; n < kN; ++n) mma_16816<true>(o[n][4 * i + k], f, pf[n][0], pf[n][1]);
          }
        }
      }
    };

    for (int j = 0; j < walk.n; ++j) {
      const int stage = done % kStages;
      live = live && mbar_wait_warp(&full[group][stage], (done / kStages) & 1);
      if (!live) break;
      const uint32_t at = base + stage * stage_bytes;
      const int tok = (walk.t0 + j) * kTok;
      if (tok + kTok <= clean)
        step(at, tok, std::false_type());
      else if (tok < most)
        step(at, tok, std::true_type());
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[group][stage]);
      ++done;
      if (member == 0 && next_tile < walk.t0 + walk.n) issue();
    }
    if (!live) break;

    // --------------------------------------------------------------- output
    const bool whole = walk.starts && walk.ends;
    const int32_t info =
        walk.starts && !walk.ends ? cut_info(run, c, walk.base + unit.tiles(walk.q, walk.kv, walk.block) - 1) : 0;
    const int64_t slot = (static_cast<int64_t>(walk.starts ? 2 * c + 1 : 2 * c) * p.kv_heads + h) * kRows;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float l = sum[n][k];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        const int r = n * 8 + 2 * t + k;
        float inv = l == 0.f ? 0.f : 1.f / l;
        float lse = l == 0.f ? -INFINITY : fmaf(-less[n][k], mult[n][k] * 0.6931471805599453f, (log2f(l) - 6.f) * 0.6931471805599453f);
        if (lse == INFINITY) inv = lse = __int_as_float(0x7fffffff);  // a score beyond fp32
        if (r >= rows) continue;
        int i;
        const int64_t row = row_of(r, i);
        if (g == 0) {
          if (walk.starts) P.parts.row_info[row] = info ? info + r : 0;
          if (whole)
            p.lse[row] = lse;
          else
            P.parts.lse[slot + r] = lse;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = 32 * ((2 * g + j) & 3) + 8 * ((2 * g + j) >> 2);
          float y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = o[n][4 * j + e][k] * inv, y[4 + e] = o[n][4 * j + e][2 + k] * inv;
          if (whole) {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * kHeadDim + d) =
                make_uint4(pack2<kFp16>(y[0], y[1]), pack2<kFp16>(y[2], y[3]), pack2<kFp16>(y[4], y[5]), pack2<kFp16>(y[6], y[7]));
          } else {
            float4* dst = reinterpret_cast<float4*>(P.parts.o + (slot + r) * kHeadDim + d);
            dst[0] = make_float4(y[0], y[1], y[2], y[3]);
            dst[1] = make_float4(y[4], y[5], y[6], y[7]);
          }
        }
      }
    }
    if (*const_cast<volatile uint32_t*>(&odd[warp])) {  // (rarely) which rows see which NaN: those tiles' values are looked at again
      __syncwarp();
      int i;
      const int64_t row = row_of(min(lane, rows - 1), i);
      const int seen = lane < rows ? unit.limit(walk.q, walk.kv, i) : 0, end = min(most, (walk.t0 + walk.n) * kTok);
      uint32_t bad = 0;  // bit i: row `lane` sees a NaN in its values' group i
      for (int tok = max(clean / kTok, walk.t0) * kTok; tok < end; tok += 32) {
        const uint32_t its = tok + lane < end ? odd_groups(p, walk.b, tok + lane, shift, h) : 0;
        for (uint32_t who = __ballot_sync(0xffffffffu, its != 0); who; who &= who - 1) {
          const int l = __ffs(who) - 1;
          const uint32_t groups = __shfl_sync(0xffffffffu, its, l);
          if (tok + l < seen) bad |= groups;
        }
      }
      for (int r = 0; r < rows; ++r) {
        const int64_t to = __shfl_sync(0xffffffffu, row, r);
        for (uint32_t its = __shfl_sync(0xffffffffu, bad, r); its; its &= its - 1) {
          const int d = 32 * (__ffs(its) - 1) + lane;
          if (whole)
            static_cast<uint16_t*>(p.out)[to * kHeadDim + d] = 0x7fff;  // (of either type)
          else
            P.parts.o[(slot + r) * kHeadDim + d] = __int_as_float(0x7fffffff);
        }
      }
    }
  }
  if (!live) {  // an aborted call: the loads in flight land before their warp leaves
    for (; done < issued; ++done) mbar_wait_drain(&full[group][done % kStages], (done / kStages) & 1);
  }
}

// How the kv heads share tiles: groups of up to kHeads, as equal as may be, and of whole pairs where there are pairs.
struct Groups {
  int heads, head_groups, groups;  // kv heads per group, groups that have all of them, groups per CTA
};
template <int kN>
Groups group_heads(int kv_heads) {
  using S = Shape<kN>;
  const int of = kv_heads % 2 ? 1 : 2, units = kv_heads / of;
  Groups g;
  g.head_groups = (kv_heads + S::kHeads - 1) / S::kHeads;
  g.heads = (units + g.head_groups - 1) / g.head_groups * of;
  g.head_groups = (kv_heads + g.heads - 1) / g.heads;
  g.groups = S::kWarps / g.heads;
  return g;
}

// Runs per kv head: as many groups as are resident, no more than there are tiles.
template <int kN>
int run_count(const QuantDecodeLaunch& p) {
  const Groups g = group_heads<kN>(p.kv_heads);
  const int64_t rows = p.num_tokens * p.group, units = p.batch + rows / Shape<kN>::kRows;
  const int64_t tiles = std::max<int64_t>(1, (static_cast<int64_t>(p.block_cols) * p.block_size + kTok - 1) / kTok);
  const int64_t most = std::min<int64_t>(units, 1 << 20) * (kSetup + tiles);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({most, kNumSMs * g.groups / g.head_groups, kMaxRuns})));
}

template <bool kFp16, int kN>
cudaError_t launch(const QuantDecodeLaunch& p, void* workspace, cudaStream_t stream) {
  using S = Shape<kN>;
  Params P;
  P.L = p;
  const int runs = run_count<kN>(p);
  const Groups g = group_heads<kN>(p.kv_heads);
  P.parts = quant_partials(p, runs, S::kRows, workspace);
  P.box_rows = std::min(kTok, p.block_size);
  P.heads = g.heads, P.head_groups = g.head_groups, P.groups = g.groups;
  // Boxes of two heads' rows, 160 bytes, reach 6.8 to 6.9 TB/s, of one head's 5.9; one kv head's rows lie next to one
  // another, eight of them are a row of the map. (Loads of single heads by warps of their own: 5.8, and 3.4 once they are
  // four tiles apart.)
  const bool pairs = p.kv_heads % 2 == 0, one = p.kv_heads == 1;
  P.row_shift = one ? 3 : 0;
  // no pages at all: maps over rows of the query's stand in, nothing is loaded through them
  const bool any = p.num_blocks > 0;
  const uint64_t inner = one ? 8 * kQuantRow : pairs ? 2 * kQuantRow : kQuantRow;
  const uint64_t extent[3] = {inner, any ? (static_cast<uint64_t>(p.num_blocks) * p.block_size) >> P.row_shift : 1,
                              any ? p.kv_heads * kQuantRow / std::min<uint64_t>(inner, p.kv_heads * kQuantRow) : 1};
  const uint64_t stride[2] = {one ? inner : static_cast<uint64_t>(p.kv_heads) * kQuantRow, inner};
  const uint32_t box[3] = {static_cast<uint32_t>(inner), static_cast<uint32_t>(P.box_rows) >> P.row_shift,
                           static_cast<uint32_t>(one ? 1 : pairs ? g.heads / 2 : g.heads)};
  if (!encode_tmap_bytes(&P.key, any ? p.key : p.query, extent, stride, box) ||
      !encode_tmap_bytes(&P.value, any ? p.value : p.query, extent, stride, box))
    return cudaErrorInvalidValue;
  auto kern = pairs ? quant_decode_kernel<kFp16, kN, 160> : quant_decode_kernel<kFp16, kN, 80>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), S::kSmem);
  if (e != cudaSuccess) return e;
  kern<<<static_cast<unsigned>((static_cast<int64_t>(runs) * g.head_groups + g.groups - 1) / g.groups), 32 * S::kWarps, S::kSmem,
         stream>>>(P);
  e = cudaGetLastError();
  if (e != cudaSuccess || runs == 1) return e;
  return launch_quant_combine<kFp16, S::kRows>(p, P.parts, stream);
}

// Blocks of 8 query rows per warp: as a request has rows (known from the shapes: the mean, with lengths on the device).
// Unpacking, most of a block's some 330 instructions per 16 tokens, is shared by a warp's blocks. More than four would
// take a second walk over the tokens, and go to the 256-row blocks of quant_tiles.cu (0). Both ways, 8 kv heads: 96 requests
// over 4,000 tokens with 32 rows 306 us here against 519, with 36 rows 537 (in two walks) against 519, with 64 rows 559
// against 527, with 128 rows 1,035 against 544; one request over 32,768 tokens with 32 rows 54 against 58, with 36 67
// against 56, with 128 112 against 62.
int row_blocks(const QuantDecodeLaunch& p) {
  const int64_t rows = (p.num_tokens * p.group + p.batch - 1) / p.batch;
  return rows <= 32 ? static_cast<int>((rows + 7) / 8) : 0;
}

template <int kN>
size_t workspace_of(const QuantDecodeLaunch& p) {
  return quant_partial_bytes(p, run_count<kN>(p), Shape<kN>::kRows);
}

}  // namespace

size_t quant_decode_workspace(const QuantDecodeLaunch& p) {
  const int n = row_blocks(p);
  if (n == 0) return quant_tiles_workspace(p);
  return n == 1 ? workspace_of<1>(p) : n == 2 ? workspace_of<2>(p) : n == 3 ? workspace_of<3>(p) : workspace_of<4>(p);
}

cudaError_t launch_quant_decode(const QuantDecodeLaunch& p, bool fp16, void* workspace, cudaStream_t stream) {
  auto go = [&](auto n) { return fp16 ? launch<true, n.value>(p, workspace, stream) : launch<false, n.value>(p, workspace, stream); };
  switch (row_blocks(p)) {
    case 0: return launch_quant_tiles(p, fp16, workspace, stream);
    case 1: return go(std::integral_constant<int, 1>());
    case 2: return go(std::integral_constant<int, 2>());
    case 3: return go(std::integral_constant<int, 3>());
    default: return go(std::integral_constant<int, 4>());
  }
}

}  // namespace cascade
