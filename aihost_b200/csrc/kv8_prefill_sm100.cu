// kv8_prefill_sm100.cu — attention of many query rows over the 8-bit or the 4-bit paged cache on the
// 5th-generation tensor cores (prompts and long continuations, fp16 tensors).
//
// One block takes 256 query rows of one KV head (tokens x the heads of its group, so a cache row is
// converted once for the whole group), as two tiles of 128, and walks a range of the cache in
// 128-row tiles (flash attention, online softmax):
//   warp 1       copies the int8 rows of each tile, page by page, into a ring (bulk copies).
//   warpgroup 3  makes them fp16 exactly and stores them in the 128-byte swizzled layout the MMAs
//                read; K and V rings of their own.
//   warp 2       the pages' scales, which stay out of the products: one factor per 16 rows of K
//                (times scale and log2 e) and of V (over the range's largest), in a small ring.
//   warp 0       issues tcgen05.mma: S = Q K^T into tensor memory, O += P V with P read from there;
//                the two tiles take turns, so one's softmax runs under the other's products. The
//                whole warp runs this code on warp-uniform values and one elected lane issues:
//                descriptors then stay in uniform registers.
//   warpgroups 1, 2  one thread per query row: S from tensor memory, K's factors, cap and bias, masks
//                on tiles that cross the row's range, running maximum (O is rescaled only when it
//                grows by more than 2^8), exp2, row sum, P times V's factors as fp16.
// Ranges are cut into chunks where there are few tiles; the last block of a tile to arrive merges.
//
// Precision: an unrotated fp16 q is exact. A rotated one is rounded to fp16, and the fp16 of what that leaves
// enters as a second operand. At head_dim 128 that costs 64 KB, which come from the rings (one K and one V
// tile instead of two), and a third more products; a caller may do without (AIHOST_KV8_ROUND_Q): results are
// then off by 3.6e-4 instead of 2.9e-4 (relative root mean square; an fp16 result alone is by 2.1e-4). Either is
// of one half of the rotated q, since turning (x, y) may pass fp16's range; K's factors take it back. P is
// rounded to fp16 once, as the output is; maxima, sums and accumulators are fp32, int8 values exact. (P as
// a pair too: 690 us in place of 505 for the first case below; the rest of 128 weights a row costs the softmax what
// the products do not.)
//
// Measured: 2048 new rows over 14336 cached, 32/8 heads x 128, q rotated, 560 us (515 GFLOP: 920 TFLOP/s, 56 % of
// the measured 1634; 650 us where calls follow one another for long, under the power cap), with q rounded 495-506
// (544-550). The MMAs of a tile pair take ~3070 cycles (2048 with q rounded), the loop ~4200 (3760): a tile's turn
// is its S and P V and its softmax (~2740 beside the other tile's), one after another; and the last 0.73 of a wave
// are chunks, each with a block's fixed work. Two prompts of 4 K rows with documents, 181 us (163): of a block's
// ~40 K cycles about half are fixed (lookup and ranges 5 K, Q 5 K, its rotation 4.6 K, first S 1.6 K, results
// 5 K). Six uneven prompts, 14/2 heads x 64, scores capped: 63.5 us.
// Not better on the first of these with q rounded: S in two halves of 64 keys (620 us), the next
// S read into registers ahead (spills, 1330), two threads per query row (569), softmax as a loop over 32
// columns that reads S twice (564), a quarter of the exponentials by a polynomial on the FMA pipe (595),
// non-uniform descriptors (790), set-up before the tile is known (553).
//
// Over the 4-bit cache (FOUR) the converters make c - 8 of K's codes and c - 7.5 of V's, exact in fp16 (V's ranges come with its
// rows, for steps below zero); warp 2 brings five fp32 factors for every row, and the softmax applies them: K's step and mid to S, the
// logarithm of V's step too, so that P is the weight times the step; two more bring P back to the weight, for the row sum, and
// to its share of V's mids, for a sum of its own beside O.
// Measured: the 2048 rows over 14336 1027 us, the documents 240, the six prompts 82. The softmax bounds it: a factor per column
// is a turn of shared memory for each warp and one more packed operation. With V's step in the operand and P, four factors, 992,
// 228 and 80, but a weight below 2^-17 of the row's largest loses bits however large its row's step is. Not better: K's
// factors and V's as fp16 (1067, 240, 84), two rows' factors in 16 bytes (1025, 238, 82), the logarithms only read in tiles
// whose steps differ by more than 2^4 (1079, 243, 83: spills). Without V's factors, V as fp16(low + step c), 817, 200 and 73, but
// results off by 3.5e-4 instead of 2.8e-4. V's codes enter less their mean: less 8, O drifts by half a step times the sum of P, and
// what the tensor core cuts off it made the error 4.4e-4 after 250 tiles in one block (2.8e-4 at any length so).
#include <algorithm>

#include "common.cuh"
#include "kv8.h"
#include "kv8_tile.cuh"

namespace aihost {
namespace {

constexpr int kTileRows = 128;
constexpr int kRows = 2 * kTileRows;  // query rows of a block
constexpr int kKeys = 128;            // cache rows of a tile
constexpr int kThreads = 512;
// setmaxnreg split of the 128 x 512 registers at launch: warps 0-3, softmax warpgroups, converters. Measured
// against 64 / 176 / 96: the long prompt below 489 us and 499-534, prompts with documents 162-165 either way.
constexpr uint32_t kRegsMma = 56, kRegsSoftmax = 184, kRegsConvert = 88;
static_assert(128 * (kRegsMma + 2 * kRegsSoftmax + kRegsConvert) <= 128 * kThreads, "setmaxnreg split exceeds the launch");
constexpr float kSlack = 8.0f;    // the maximum may lag by 2^8 before O is rescaled
constexpr float kQUnit = 0.5f;    // a rotated q enters times this
constexpr float kVUnit = 128.0f;  // P * (v scale / largest) * 128 <= 2^15 stays in fp16's range
constexpr int kFactors = kKeys / 16;
constexpr int kFactorRing = 4;

// 4 bits: a tile's ranges as the softmax takes them. score = k_step (q.(c - 8)) + k_mid sum(q), times scale and log2 e, and v_log =
// log2 of V's step more: the weight times the step, P, relative to the row's largest such product, so that it keeps its bits
// whatever steps the rows of larger scores have. v_rcp brings it back to the weight, v_mid to that times V's low + 7.5 step. A
// step below 0 counts as its amount, with the codes from the row's other end.
struct RowFactors {
  float k_step[kKeys], k_mid[kKeys], v_log[kKeys], v_rcp[kKeys], v_mid[kKeys];
};
constexpr float kStepUnit = 128.0f, kStepLog = 7.0f;  // P enters times that: at most 2^(kSlack + 7) = 2^15

// REST: what a rotated q leaves when it is rounded to fp16 enters as a second operand (head_dim 64: always).
// FOUR: over the 4-bit cache.
template <int D, bool REST, bool FOUR>
struct Cfg {
  static constexpr int KB = D / 64;                   // 64-element (128-byte) column blocks
  static constexpr int TILE = KB * kKeys * 128;       // one [128 x D] fp16 tile
  static constexpr int NS = D == 64 ? 3 : REST ? 1 : 2;  // K and V ring depth
  static constexpr int K_OFF = 2 * TILE;              // after the two Q tiles
  static constexpr int V_OFF = K_OFF + NS * TILE;
  static constexpr int CODES = kKeys * D / (FOUR ? 2 : 1);  // one tile's rows as stored,
  static constexpr int RAW = CODES + (FOUR ? kKeys * 4 : 0);  // and the rows' ranges (V's)
  static constexpr int NR = D == 64 ? 4 : 2;          // ring of them, K and V in turn
  static constexpr int RAW_OFF = V_OFF + NS * TILE;
  static constexpr bool Q_REST = D == 64 || REST;
  static constexpr int Q_REST_OFF = RAW_OFF + NR * RAW;
  static constexpr int BAR_OFF = Q_REST_OFF + (Q_REST ? 2 * TILE : 0);
  static constexpr int RANGE_OFF = BAR_OFF + 1024;
  static constexpr int SMEM = RANGE_OFF + (FOUR ? kFactorRing * static_cast<int>(sizeof(RowFactors)) : 0) + 1024;  // and alignment slack
  static __device__ __forceinline__ uint32_t s_col(int t) { return t ? 128u : 0u; }
  static __device__ __forceinline__ uint32_t o_col(int t) { return 256u + static_cast<uint32_t>(t * D); }
};

struct Shared {
  uint64_t q_ready[2], s_full[2], p_full[2][2], o_full[2];
  uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3];
  uint64_t raw_full[4], raw_empty[4];
  float k_factor[kFactorRing][kFactors];
  float v_factor[kFactorRing][kFactors];
  float v_exp[kFactorRing][kFactors];
  float v_max[4];
  float freq[64];  // the rotation's frequencies: a parameter indexed by lane costs a turn per distinct index
  uint32_t tmem_base;
  int32_t last;
  int32_t place[7];  // what the end of the block needs of its start, kept out of the loop's registers
};
static_assert(sizeof(Shared) <= 1024, "the layout reserves 1024 bytes");

// Byte offset of 16-byte chunk c of row `row` in a [128 x D] fp16 tile: 128-byte swizzled rows of
// 64 elements, blocks of 64 columns one after another.
__device__ __forceinline__ uint32_t chunk_off(int row, int c) {
  return static_cast<uint32_t>((c >> 3) * (kKeys * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 16 int8 as two 16-byte chunks of fp16, exactly.
__device__ __forceinline__ void convert16(const uint4& v, uint4& lo, uint4& hi) {
  const uint32_t w0 = v.x ^ 0x80808080u, w1 = v.y ^ 0x80808080u, w2 = v.z ^ 0x80808080u, w3 = v.w ^ 0x80808080u;
  lo = make_uint4(half2_of(w0, 0x4140), half2_of(w0, 0x4342), half2_of(w1, 0x4140), half2_of(w1, 0x4342));
  hi = make_uint4(half2_of(w2, 0x4140), half2_of(w2, 0x4342), half2_of(w3, 0x4140), half2_of(w3, 0x4342));
}

// x * P(x^2) * cap2 for the thread's scores, P of degree N.
template <int N>
__device__ __forceinline__ void odd_of(uint32_t (&sr)[4][32], const float (&coef)[N + 1], float cap2) {
  float2 k2[N + 1];
#pragma unroll
  for (int k = 0; k <= N; ++k) k2[k] = make_float2(coef[k] * cap2, coef[k] * cap2);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      const float2 x = make_float2(__uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1]));
      const float2 y = fmul2(x, x);
      float2 p = k2[N];
#pragma unroll
      for (int k = N - 1; k >= 0; --k) p = ffma2(p, y, k2[k]);
      p = fmul2(x, p);
      sr[c][e] = __float_as_uint(p.x);
      sr[c][e + 1] = __float_as_uint(p.y);
    }
}

// score = cap * tanh(x), x in units of the cap, times log2 e (cap2 = cap * log2 e). Where the whole
// warp has |x| <= 1, tanh x = x * P(x^2) on the FMA pipe (the exponentials already fill the SFU): P of
// degree 6, our weighted least-squares fit on [0, 1], 5e-8 off; where it has |x| <= 0.35, as with caps
// well above the scores, the one of degree 3. Else tanh_far for all, 1e-7 of the cap off, which is below P's
// rounding for caps up to 5000 (tanh_of, whose error goes by the score: 328 us in place of 263 for three
// prompts of 1500 to 2000 rows with scores beyond a cap of 4). Measured with and without the shorter
// polynomial: 6 prompts with cap 50 63.5 and 70 us, 3 with cap 30 195 and 221; with scores beyond a cap of 4
// the one comparison more costs 282 against 277.
__device__ __forceinline__ void cap_scores(uint32_t (&sr)[4][32], float cap2) {
  float tops[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < 32; e += 2)
      tops[c] = fmax3(tops[c], fabsf(__uint_as_float(sr[c][e])), fabsf(__uint_as_float(sr[c][e + 1])));
  const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  if (!__any_sync(0xffffffffu, top > kTanhSmall)) {
    constexpr float kP[4] = {kTanh0, kTanh1, kTanh2, kTanh3};
    odd_of<3>(sr, kP, cap2);
  } else if (!__any_sync(0xffffffffu, top > 1.0f)) {
    constexpr float kP[7] = {0.9999999403953552f,  -0.33332839608192444f, 0.13325203955173492f, -0.05345702916383743f,
                             0.020289979875087738f, -0.006203378085047007f, 0.001041022245772183f};
    odd_of<6>(sr, kP, cap2);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 32; ++e) sr[c][e] = __float_as_uint(cap2 * tanh_far(__uint_as_float(sr[c][e])));
  }
}

// D[tmem] (+)= A * B with A's descriptor or tensor memory address, issued by one lane of the warp, which
// runs this together on warp-uniform operands.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t at, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(at), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit_elected(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void arrive_elected(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n @e mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];\n}\n" ::"r"(
          smem_u32(bar))
      : "memory");
}
// `bytes` (a multiple of 16) from global to shared memory, both 16-byte aligned, counted on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Whether a range (low, step) is two numbers, and whether the step is below 0.
__device__ __forceinline__ bool range_fine(uint32_t range) { return (range & 0x7c00u) != 0x7c00u && (range & 0x7c000000u) != 0x7c000000u; }
__device__ __forceinline__ bool v_turned(uint32_t range) { return range >> 31; }

// 32 lanes x 8 consecutive 32-bit columns of tensor memory.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// A wait that the whole warp leaves together, with one answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int32_t* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status));
}

template <int D, bool MOD, bool REST, bool FOUR>
__global__ void __launch_bounds__(kThreads, 1) kv8_prefill_kernel(const __grid_constant__ Kv8AttnArgs a) {
  using C = Cfg<D, REST, FOUR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared& sh = *reinterpret_cast<Shared*>(smem + C::BAR_OFF);
  RowFactors* const factors = reinterpret_cast<RowFactors*>(smem + C::RANGE_OFF);  // FOUR
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int32_t H = a.g.n_kv_heads, G = a.g.n_q_heads / H, ps = a.g.page_shift;
  // longest ranges first: a sequence's last tiles see the most
  // units (tile, head): the first a.whole in one block each, then the others' chunks
  const bool whole = blockIdx.x < static_cast<uint32_t>(a.whole);
  uint32_t unit = blockIdx.x, split = 0;
  if (a.max_splits > 1 && !whole) {
    const uint32_t rest = static_cast<uint32_t>(a.tiles * H - a.whole);
    split = (unit - a.whole) / rest;
    unit -= split * rest;
  }
  const int32_t h = static_cast<int32_t>(unit % H), tile = a.tiles - 1 - static_cast<int32_t>(unit / H);
  griddep_launch_dependents();
  const Tile tl = find_tile(a, tile, G, kRows, lane);
  if (!tl.ok) return;
  const int32_t n_rows = min(static_cast<int64_t>(kRows), static_cast<int64_t>(tl.n_new) * G - tl.row0);

  // ---- cache tiles [j0, j1) of either query tile, and this block's chunk of them
  int32_t j0[2], j1[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    int32_t lo = INT32_MAX, hi = 0;
    if (t * kTileRows < n_rows) {
      const int32_t i0 = (tl.row0 + t * kTileRows) / G, i1 = (tl.row0 + min((t + 1) * kTileRows, n_rows) - 1) / G;
      const int32_t prefix = a.prefix_len ? min(a.prefix_len[tl.b], tl.kv_len) : 0;
      if (!a.row_first) {
        lo = 0;
        hi = max(tl.pos0 + i1 + 1, prefix);
      } else {
        for (int32_t i = i0 + lane; i <= i1; i += 32) {
          const int32_t first = max(a.row_first[tl.start + i], 0), end = max(tl.pos0 + i + 1, prefix);
          if (first < end) {
            lo = min(lo, first);
            hi = max(hi, end);
          }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
      }
    }
    j0[t] = hi > 0 ? lo / kKeys : 0;
    j1[t] = hi > 0 ? (hi + kKeys - 1) / kKeys : 0;
  }
  const bool any0 = j1[0] > 0, any1 = j1[1] > 0;
  const int32_t all0 = any0 ? (any1 ? min(j0[0], j0[1]) : j0[0]) : j0[1], all1 = max(j1[0], j1[1]);
  const int32_t chunk = whole ? max(all1 - all0, 1) : a.chunk / kKeys;
  const int32_t n_splits = max(1, (all1 - all0 + chunk - 1) / chunk);
  if (static_cast<int32_t>(split) >= n_splits) return;
  const int32_t jb = all0 + static_cast<int32_t>(split) * chunk, je = min(all1, jb + chunk);
  const int32_t n_load = max(je - jb, 0);  // 0: no row of the block sees anything
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    j0[t] = max(j0[t], jb);
    j1[t] = min(j1[t], je);
  }
  int32_t* const status = a.status;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh.q_ready[t], kTileRows);
      mbar_init(&sh.s_full[t], 2);  // the products' commit, and the issuing thread's own arrival
      mbar_init(&sh.p_full[t][0], kTileRows);  // P comes in two halves of 64 keys
      mbar_init(&sh.p_full[t][1], kTileRows);
      mbar_init(&sh.o_full[t], 1);
    }
    for (int i = 0; i < C::NS; ++i) {
      mbar_init(&sh.k_full[i], 128 + 1);  // the converters, and warp 2 with the tile's factors
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 128);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < C::NR; ++i) {
      mbar_init(&sh.raw_full[i], 1);
      mbar_init(&sh.raw_empty[i], 4);
    }
    fence_mbar_init();
  }
  if (threadIdx.x >= 64 && threadIdx.x < 64 + D / 2)
    sh.freq[threadIdx.x - 64] = a.freqs.f[threadIdx.x - 64];
  if (threadIdx.x == 32 * 12) {
    const int32_t place[7] = {tl.start, tl.row0, n_rows, h, static_cast<int32_t>(split), static_cast<int32_t>(unit) - a.whole, n_splits};
    for (int k = 0; k < 7; ++k) sh.place[k] = place[k];
  }
  if (warp == 1) tmem_alloc(&sh.tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;

  const int32_t row_end = min(je * kKeys, tl.kv_len);  // rows from here on are not read
  const int32_t* const table = a.block_table + static_cast<int64_t>(tl.b) * a.g.max_pages;
  bool stray = false;
  if (warp < 4) {
    regs_dealloc<kRegsMma>();
    if (warp == 0) {
      // ---------------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc_qk = make_idesc_f16(kTileRows, kKeys, 0, 0);
      constexpr uint32_t idesc_pv = make_idesc_f16(kTileRows, D, 0, 1);
      auto uni = [](int32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
      const int32_t n = uni(n_load);
      const int32_t lo0 = uni(j0[0] - jb), hi0 = uni(j1[0] - jb), lo1 = uni(j0[1] - jb), hi1 = uni(j1[1] - jb);
      const uint32_t tm = static_cast<uint32_t>(uni(static_cast<int32_t>(tmem)));
      const uint32_t base = static_cast<uint32_t>(uni(static_cast<int32_t>(smem_u32(smem))));
      // descriptors count in 16-byte units: an operand `off` bytes on is + off / 16
      const uint64_t q_desc = make_sw128_desc(base, 16, 1024), k_desc = make_sw128_desc(base + C::K_OFF, 16, 1024);
      const uint64_t v_desc = make_sw128_desc(base + C::V_OFF, kKeys * 128, 1024);
      auto issue_qk = [&](int t, int s) {
        const uint64_t qd = q_desc + t * (C::TILE / 16), kd = k_desc + s * (C::TILE / 16);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr int kBlock = kKeys * 128;
          const uint32_t off = ((kk >> 2) * kBlock + (kk & 3) * 32) / 16;
          mma_ss(tm + C::s_col(t), qd + off, kd + off, idesc_qk, kk > 0);
        }
        if (C::Q_REST && a.rope_mode != AIHOST_ROPE_NONE) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            constexpr int kBlock = kKeys * 128;
            const uint32_t off = ((kk >> 2) * kBlock + (kk & 3) * 32) / 16;
            mma_ss(tm + C::s_col(t), qd + C::Q_REST_OFF / 16 + off, kd + off, idesc_qk, 1);
          }
        }
        commit_elected(&sh.s_full[t]);
        arrive_elected(&sh.s_full[t]);  // passes on what was written besides (the factors)
      };
      auto issue_pv = [&](int t, int half, int s, bool first) {
        const uint64_t vd = v_desc + s * (C::TILE / 16);
#pragma unroll
        for (int kk = half * (kKeys / 32); kk < (half + 1) * (kKeys / 32); ++kk)
          mma_ts(tm + C::o_col(t), tm + C::s_col(t) + kk * 8, vd + kk * (2048 / 16), idesc_pv, !first || kk > 0);
      };
      bool ok = n > 0 && warp_wait(&sh.q_ready[0], 0, status) && warp_wait(&sh.q_ready[1], 0, status) &&
                warp_wait(&sh.k_full[0], 0, status);
      tc_fence_after();
      if (ok) {
        if (lo0 <= 0 && hi0 > 0) issue_qk(0, 0);
        if (lo1 <= 0 && hi1 > 0) issue_qk(1, 0);
        commit_elected(&sh.k_empty[0]);
      }
      int s = 0;
      uint32_t par = 0;
      for (int32_t i = 0; ok && i < n; ++i) {
        const int s1 = s + 1 == C::NS ? 0 : s + 1;
        const uint32_t par1 = s1 ? par : par ^ 1;
        bool go = warp_wait(&sh.v_full[s], par, status);
        // with one K tile at a time, the next one is made while the first P V runs
        if (C::NS > 1) go = go && (i + 1 >= n || warp_wait(&sh.k_full[s1], par1, status));
        if (!go) break;
        tc_fence_after();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int32_t t_lo = t ? lo1 : lo0, t_hi = t ? hi1 : hi0;
          if (i >= t_lo && i < t_hi) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              go = go && warp_wait(&sh.p_full[t][half], (i - t_lo) & 1, status);
              tc_fence_after();
              if (go) issue_pv(t, half, s, i == t_lo);
            }
            if (!go) break;
            if (i + 1 == t_hi) commit_elected(&sh.o_full[t]);
          }
          if (C::NS == 1 && t == 1) commit_elected(&sh.v_empty[s]);
          if (C::NS == 1 && t == 0 && i + 1 < n) {
            go = warp_wait(&sh.k_full[s1], par1, status);
            if (!go) break;
            tc_fence_after();
          }
          if (i + 1 >= t_lo && i + 1 < t_hi) issue_qk(t, s1);
        }
        if (!go) break;
        if (C::NS > 1) commit_elected(&sh.v_empty[s]);
        if (i + 1 < n) commit_elected(&sh.k_empty[s1]);
        s = s1;
        par = par1;
      }
      // the last commit arrives in the block's shared memory, and nobody else waits for it
      if (ok) warp_wait(&sh.v_empty[(n - 1) % C::NS], ((n - 1) / C::NS) & 1, status);
    } else if (warp == 1) {
      // ---------------------------------------------------------------- int8 rows, page by page
      // lane f copies the tile's f-th page (a page holds 16 to 128 of its 128 rows); its table entry is
      // read two tiles ahead
      const int32_t per_page = min(a.g.page_rows, kKeys), n_seg = kKeys / per_page;
      auto entry_of = [&](int32_t i) -> int32_t {
        const int32_t row = (jb + i) * kKeys + lane * per_page;
        return lane < n_seg && row < row_end ? table[row >> ps] : INT32_MIN;
      };
      int32_t e0 = n_load > 0 ? entry_of(0) : INT32_MIN, e1 = n_load > 1 ? entry_of(1) : INT32_MIN;
      int32_t issued = 0;
      for (int32_t i = 0; i < n_load; ++i) {
        const int32_t e = e0;
        e0 = e1;
        if (i + 2 < n_load) e1 = entry_of(i + 2);
        const bool mine = e != INT32_MIN;
        const int64_t page = mine ? page_or_first(e, a.g.n_pages, stray) : 0;
        constexpr int kRowBytes = FOUR ? D / 2 : D;
        const int64_t at = ((page * H + h) << ps) * kRowBytes;  // a tile starts at a page's first row: pages divide it
        const uint32_t bytes = static_cast<uint32_t>(per_page * kRowBytes);
        const uint32_t n_mine = __popc(__ballot_sync(0xffffffffu, mine));
        bool ok = true;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int32_t g = 2 * i + v, slot = g % C::NR;
          ok = ok && warp_wait(&sh.raw_empty[slot], ((g / C::NR) & 1) ^ 1, status);
          if (!ok) break;
          const uint32_t range_bytes = FOUR && v ? static_cast<uint32_t>(per_page * 4) : 0;
          if (lane == 0) mbar_arrive_expect_tx(&sh.raw_full[slot], n_mine * (bytes + range_bytes));
          __syncwarp();
          if (mine) bulk_load(smem + C::RAW_OFF + slot * C::RAW + lane * bytes, (v ? a.v_pool : a.k_pool) + at, bytes,
                              &sh.raw_full[slot]);
          if (FOUR && v && mine)
            bulk_load(smem + C::RAW_OFF + slot * C::RAW + C::CODES + lane * range_bytes, a.v_range + at / kRowBytes, range_bytes,
                      &sh.raw_full[slot]);
          issued = g + 1;
        }
        if (!ok) break;
      }
      // the last copies have landed before the block may end, however its other warps fared
      for (int32_t g = max(issued - C::NR, 0); g < issued; ++g)
        warp_wait(&sh.raw_full[g % C::NR], (g / C::NR) & 1, status);
    } else if (FOUR && warp == 2) {
      // ---------------------------------------------------------------- ranges, four rows a lane
      const float q_scale = a.rope_mode != AIHOST_ROPE_NONE ? a.scale * (1.0f / kQUnit) : a.scale;
      const float k_unit = MOD && a.score_cap > 0.0f ? q_scale / a.score_cap : q_scale * kLog2e;
      auto entry_of = [&](int32_t i) -> int32_t {
        const int32_t row = (jb + i) * kKeys + lane * 4;
        return i < n_load && row < row_end ? table[row >> ps] : INT32_MIN;
      };
      auto fetch = [&](int32_t i, int32_t e, uint4 (&r)[2]) {
        r[0] = r[1] = make_uint4(0, 0, 0, 0);
        if (e != INT32_MIN) {
          const int32_t row = (jb + i) * kKeys + lane * 4;
          const int64_t at = ((page_or_first(e, a.g.n_pages, stray) * H + h) << ps) + (row & (a.g.page_rows - 1));
          r[0] = __ldg(reinterpret_cast<const uint4*>(a.k_range + at));
          r[1] = __ldg(reinterpret_cast<const uint4*>(a.v_range + at));
        }
      };
      uint4 now[2], next[2];
      fetch(0, entry_of(0), now);
      int32_t e_next = entry_of(1);
      for (int32_t i = 0; i < n_load; ++i) {
        fetch(i + 1, e_next, next);
        e_next = entry_of(i + 2);
        const int s = i % C::NS;
        // as with the scales below: the ring's slot is free, and k_full's phase is this tile's
        if (!warp_wait(C::NS > 1 ? &sh.v_empty[s] : &sh.k_empty[s], ((i / C::NS) & 1) ^ 1, status)) break;
        const uint32_t kr[4] = {now[0].x, now[0].y, now[0].z, now[0].w}, vr[4] = {now[1].x, now[1].y, now[1].z, now[1].w};
        float f[5][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 k = __half22float2(*reinterpret_cast<const __half2*>(&kr[e]));
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&vr[e]));
          // a row of V that is no number marks itself through K, as one of K does: of a hidden row, whose weight is 0, nothing
          // may come, and an infinite score of a row seen could be -infinity.
          // A step of zero counts as 2^-60: such a P is 0 as fp16, and comes back whole in the sums.
          const bool fine = range_fine(vr[e]);
          const float step = v.y != 0.0f ? fabsf(v.y) : 8.6736173798840355e-19f;
          f[0][e] = fine && range_fine(kr[e]) ? k.y * k_unit : __uint_as_float(0x7fffffffu);
          f[1][e] = fmaf(8.0f, k.y, k.x) * k_unit;
          f[2][e] = fine ? log2f(step) : 0.0f;
          f[3][e] = fine ? 1.0f / (step * kStepUnit) : 0.0f;
          f[4][e] = fine ? fmaf(7.5f, v.y, v.x) * f[3][e] : 0.0f;
        }
        RowFactors& to = factors[i % kFactorRing];
        float* const rows[5] = {to.k_step, to.k_mid, to.v_log, to.v_rcp, to.v_mid};
#pragma unroll
        for (int n = 0; n < 5; ++n) *reinterpret_cast<float4*>(rows[n] + lane * 4) = make_float4(f[n][0], f[n][1], f[n][2], f[n][3]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.k_full[s]);
        now[0] = next[0], now[1] = next[1];
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- factors
      float ks[2] = {0.0f, 0.0f}, vs[2] = {0.0f, 0.0f};
      bool on[2] = {false, false};
      int32_t e_next = 0;
      auto entry_of = [&](int32_t i) -> int32_t {
        const int32_t row = (jb + i) * kKeys + lane * 16;
        return i < n_load && lane < kFactors && row < row_end ? table[row >> ps] : INT32_MIN;
      };
      auto fetch = [&](int32_t e, int k) {
        on[k] = e != INT32_MIN;
        if (on[k]) {
          const int64_t at = page_or_first(e, a.g.n_pages, stray) * H + h;
          ks[k] = __ldg(a.k_scale + at);
          vs[k] = __ldg(a.v_scale + at);
        }
      };
      fetch(entry_of(0), 0);
      e_next = entry_of(1);
      asm volatile("bar.sync 2, 160;" ::: "memory");
      const float vmax = fmaxf(fmaxf(sh.v_max[0], sh.v_max[1]), fmaxf(sh.v_max[2], sh.v_max[3]));
      const float v_rcp = v_reciprocal(vmax);
      const float q_scale = a.rope_mode != AIHOST_ROPE_NONE ? a.scale * (1.0f / kQUnit) : a.scale;
      const float k_unit = MOD && a.score_cap > 0.0f ? q_scale / a.score_cap : q_scale * kLog2e;
      for (int32_t i = 0; i < n_load; ++i) {
        fetch(e_next, 1);
        e_next = entry_of(i + 2);
        const int s = i % C::NS;
        // the tile NS before is done with: so is the ring's slot, and k_full's phase is this tile's
        // (of one K tile at a time, the products: the next one's wait for these factors before the V tile is done with)
        if (!warp_wait(C::NS > 1 ? &sh.v_empty[s] : &sh.k_empty[s], ((i / C::NS) & 1) ^ 1, status)) break;
        if (lane < kFactors) {
          // A scale that is no number marks the page through K's factor: a hidden row's weight is then 0
          // and its V factor must not turn it into NaN again.
          const bool fine = vs[0] < INFINITY;
          sh.k_factor[i % kFactorRing][lane] = !on[0] ? 0.0f : fine ? ks[0] * k_unit : __uint_as_float(0x7fffffffu);
          const float v_rel = !on[0] || !fine ? 0.0f : vs[0] * v_rcp;
          sh.v_factor[i % kFactorRing][lane] = v_rel * kVUnit;
          sh.v_exp[i % kFactorRing][lane] = v_exp_of(v_rel);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.k_full[s]);
        ks[0] = ks[1], vs[0] = vs[1], on[0] = on[1];
      }
    }
    if (stray) atomicOr(status, kStatusBadIndex);
  } else if (warp >= 12) {
    // ------------------------------------------------------------------ converters
    regs_dealloc<kRegsConvert>();
    const int w = warp - 12;
    if constexpr (!FOUR) {
      float vmax = 0.0f;  // the chunk's largest V scale
      for (int32_t k = ((jb * kKeys) >> ps) + w * 32 + lane; k < (row_end + a.g.page_rows - 1) >> ps; k += 128)
        vmax = fmaxf(vmax, __ldg(a.v_scale + page_or_first(table[k], a.g.n_pages, stray) * H + h));
#pragma unroll
      for (int o = 16; o; o >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
      if (lane == 0) sh.v_max[w] = vmax;
      asm volatile("bar.sync 2, 160;" ::: "memory");
    }
    // 16 bytes a lane. Eight lanes that load or store together: 8 bits, two rows, the even row's chunks of
    // one half and the odd row's of the other (D = 128; D = 64: two whole rows); 4 bits, chunk c of rows 2 (c + n) and
    // 2 (c + n) + 1 of eight for D = 128, both chunks of four rows for D = 64: different banks both ways.
    constexpr int kRowBytes = FOUR ? D / 2 : D;
    constexpr int RPL = 512 / kRowBytes;   // rows per warp and load
    constexpr int NL = kKeys / (4 * RPL);  // loads per tile and lane
    const int r_in = FOUR ? (D == 128 ? 2 * ((lane + (lane >> 3)) & 3) + ((lane >> 2) & 1) : lane >> 1)
                          : (D == 128 ? ((lane >> 2) & 1) + ((lane >> 4) << 1) : lane >> 2);
    const int c = FOUR ? (D == 128 ? lane & 3 : lane & 1)
                       : (D == 128 ? (lane & 3) + ((((lane >> 3) ^ (lane >> 2)) & 1) << 2) : lane & 3);
    uint4 v[NL];
    uint32_t range[NL] = {};
    auto take = [&](int slot, bool of_v) {  // a raw tile into registers, while the products still use the tile that it replaces
      const uint8_t* const src = smem + C::RAW_OFF + slot * C::RAW;
#pragma unroll
      for (int k = 0; k < NL; ++k) {
        const int row = (k * 4 + w) * RPL + r_in;
        v[k] = *reinterpret_cast<const uint4*>(src + row * kRowBytes + c * 16);
        if (FOUR && of_v) range[k] = *reinterpret_cast<const uint32_t*>(src + C::CODES + row * 4);
      }
      // The next rows come by the async proxy: without the fence some were found here in the place of these, whose
      // values are used after other waits only (cold caches, up to 2 % of the calls).
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.raw_empty[slot]);
    };
    auto give = [&](uint8_t* dst, uint64_t* full_bar, bool of_v) {
#pragma unroll
      for (int k = 0; k < NL; ++k) {
        const int row = (k * 4 + w) * RPL + r_in;
        if constexpr (FOUR) {
          const uint32_t turn = of_v && v_turned(range[k]) ? 0xffffffffu : 0u;  // 15 - c
          const uint32_t word[4] = {v[k].x ^ turn, v[k].y ^ turn, v[k].z ^ turn, v[k].w ^ turn};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t x[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) x[n] = of_v ? codes_less_mean(word[j], n) : codes_less_8(word[j], n);
            *reinterpret_cast<uint4*>(dst + chunk_off(row, 4 * c + j)) = make_uint4(x[0], x[1], x[2], x[3]);
          }
        } else {
          uint4 lo, hi;
          convert16(v[k], lo, hi);
          *reinterpret_cast<uint4*>(dst + chunk_off(row, 2 * c)) = lo;
          *reinterpret_cast<uint4*>(dst + chunk_off(row, 2 * c + 1)) = hi;
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(full_bar);
    };
    for (int32_t i = 0; i < n_load; ++i) {
      const int s = i % C::NS;
      const uint32_t par = ((i / C::NS) & 1) ^ 1;
      const int gk = 2 * i, gv = 2 * i + 1;
      if (!warp_wait(&sh.raw_full[gk % C::NR], (gk / C::NR) & 1, status)) break;
      take(gk % C::NR, false);
      if (!warp_wait(&sh.k_empty[s], par, status)) break;
      give(smem + C::K_OFF + s * C::TILE, &sh.k_full[s], false);
      if (!warp_wait(&sh.raw_full[gv % C::NR], (gv / C::NR) & 1, status)) break;
      take(gv % C::NR, true);
      if (!warp_wait(&sh.v_empty[s], par, status)) break;
      give(smem + C::V_OFF + s * C::TILE, &sh.v_full[s], true);
    }
    if (stray) atomicOr(status, kStatusBadIndex);
  } else {
    // ------------------------------------------------------------------ softmax: a thread per query row
    regs_alloc<kRegsSoftmax>();
    const int t = warp >= 8 ? 1 : 0;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row within the tile == tensor memory lane
    const int rr = t * kTileRows + r;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const bool valid = rr < n_rows;
    int32_t first, end, pos;
    row_range(a, tl, G, n_rows, rr, first, end, pos);
    if (!valid) first = 0, end = INT32_MAX;  // such a row works for nobody and never asks for masks
    const int32_t row = tl.row0 + min(rr, n_rows - 1), tok = row / G, head = h * G + row % G;
    // ---- the warp's 32 rows of Q, rotated in fp32, as fp16 (and its rest): LPR lanes to a row, each with 16-byte
    // chunks c and c + LPR (a half apart), and LPR rows to a lane, one after another, so that the heads of
    // one token share its sines and cosines
    uint8_t* const q_tile = smem + t * C::TILE;
    {
      constexpr int LPR = D / 16;
      const int c = lane % LPR, row_a = quarter * 32 + lane / LPR * LPR;
      auto row_of_q = [&](int k, int32_t& i) -> const uint4* {
        const int32_t q_row = tl.row0 + min(t * kTileRows + row_a + k, n_rows - 1);
        i = q_row / G;
        return reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.q) +
                                              (tl.start + static_cast<int64_t>(i)) * a.q_token_stride +
                                              static_cast<int64_t>(h * G + q_row % G) * D * 2);
      };
      uint4 x[LPR][2];
#pragma unroll
      for (int k = 0; k < LPR; ++k) {
        int32_t i;
        const uint4* const src = row_of_q(k, i);
        x[k][0] = __ldg(src + c);
        x[k][1] = __ldg(src + c + LPR);
      }
#pragma unroll
      for (int k = 0; k < LPR; ++k) {
        *reinterpret_cast<uint4*>(q_tile + chunk_off(row_a + k, c)) = x[k][0];
        *reinterpret_cast<uint4*>(q_tile + chunk_off(row_a + k, c + LPR)) = x[k][1];
      }
      // rotated in place, by a loop that is not unrolled: it runs once per block, from a cold instruction cache
      if (a.rope_mode != AIHOST_ROPE_NONE) {
        const bool halves = a.rope_mode == AIHOST_ROPE_NEOX;
        // 2^-21 off at head_dim 128 (with sincos_near 193 us for the documents, so 183)
        auto rotation = [](float angle, float* s, float* c) {
          if constexpr (D == 64) sincos_near(angle, s, c);
          else sincos_reduced(angle, s, c);
        };
        float sn[8], cs[8];  // by halves: of pairs 8 c + e; else of pairs 4 c + e and 4 (c + LPR) + e - 4
        int32_t last = -1;
#pragma unroll 1
        for (int k = 0; k < LPR; ++k) {
          const int32_t i = (tl.row0 + min(t * kTileRows + row_a + k, n_rows - 1)) / G;
          if (i != last) {
            last = i;
            const float fpos = static_cast<float>(tl.pos0 + i);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              rotation(fpos * sh.freq[halves ? 8 * c + e : 4 * (e < 4 ? c : c + LPR - 1) + e], &sn[e], &cs[e]);
#pragma unroll
            for (int e = 0; e < 8; ++e) sn[e] *= kQUnit, cs[e] *= kQUnit;
          }
          uint4* const p0 = reinterpret_cast<uint4*>(q_tile + chunk_off(row_a + k, c));
          uint4* const p1 = reinterpret_cast<uint4*>(q_tile + chunk_off(row_a + k, c + LPR));
          const uint4 v0 = *p0, v1 = *p1;
          uint32_t u0[4] = {v0.x, v0.y, v0.z, v0.w}, u1[4] = {v1.x, v1.y, v1.z, v1.w}, r0[4], r1[4];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&u0[m]));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&u1[m]));
            float2 g0, g1;
            if (halves) {  // (f0.x, f1.x) and (f0.y, f1.y)
              g0 = make_float2(f0.x * cs[2 * m] - f1.x * sn[2 * m], f0.y * cs[2 * m + 1] - f1.y * sn[2 * m + 1]);
              g1 = make_float2(f0.x * sn[2 * m] + f1.x * cs[2 * m], f0.y * sn[2 * m + 1] + f1.y * cs[2 * m + 1]);
            } else {  // (f0.x, f0.y) and (f1.x, f1.y)
              g0 = make_float2(f0.x * cs[m] - f0.y * sn[m], f0.x * sn[m] + f0.y * cs[m]);
              g1 = make_float2(f1.x * cs[4 + m] - f1.y * sn[4 + m], f1.x * sn[4 + m] + f1.y * cs[4 + m]);
            }
            u0[m] = pack2(g0.x, g0.y);
            u1[m] = pack2(g1.x, g1.y);
            r0[m] = pack2_rest(g0.x, g0.y, u0[m]);
            r1[m] = pack2_rest(g1.x, g1.y, u1[m]);
          }
          *p0 = make_uint4(u0[0], u0[1], u0[2], u0[3]);
          *p1 = make_uint4(u1[0], u1[1], u1[2], u1[3]);
          if constexpr (C::Q_REST) {
            p0[C::Q_REST_OFF / 16] = make_uint4(r0[0], r0[1], r0[2], r0[3]);
            p1[C::Q_REST_OFF / 16] = make_uint4(r1[0], r1[1], r1[2], r1[3]);
          }
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&sh.q_ready[t]);
    }
    float q_sum = 0.0f;  // of the thread's row of q, as it enters
    if constexpr (FOUR) {
      __syncwarp();
      const bool rest = C::Q_REST && a.rope_mode != AIHOST_ROPE_NONE;
#pragma unroll 1
      for (int n = rest ? 1 : 0; n >= 0; --n)
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          const uint4 x = *reinterpret_cast<const uint4*>(q_tile + n * C::Q_REST_OFF + chunk_off(r, c));
          const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
            q_sum += f.x + f.y;
          }
        }
    }

    const float slope = MOD && a.alibi_slopes ? a.alibi_slopes[head] * kLog2e : 0.0f;
    const bool capped = MOD && a.score_cap > 0.0f;
    const float cap2 = a.score_cap * kLog2e, fpos = static_cast<float>(pos);
    float m = kNoMax, l = 0.0f, z = 0.0f;  // z: the sum of the weights times V's mids (FOUR)
    const uint32_t s_tmem = tmem + lane_base + C::s_col(t), o_tmem = tmem + lane_base + C::o_col(t);
    const int32_t lo_j = t ? j0[1] : j0[0], hi_j = t ? j1[1] : j1[0], n_own = hi_j - lo_j;
    bool ok = true;
    for (int32_t i = 0; i < n_own; ++i) {
      if (!warp_wait(&sh.s_full[t], i & 1, status)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sr[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + c * 32, sr[c]);
      const int slot = (lo_j + i - jb) % kFactorRing;
      const int32_t kv0 = (lo_j + i) * kKeys;
      const bool need_mask = __any_sync(0xffffffffu, kv0 < first || kv0 + kKeys > end);
      const RowFactors& rows = factors[slot];
      auto two = [](const float (&x)[kKeys], int e) { return *reinterpret_cast<const float2*>(&x[e]); };
      float kf[kFactors];
      if constexpr (!FOUR) {
#pragma unroll
        for (int f = 0; f < kFactors; ++f) kf[f] = sh.k_factor[slot][f];
      }
      tmem_wait_ld();
      if constexpr (FOUR) {
        const float2 q2 = make_float2(q_sum, q_sum);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 mid = two(rows.k_mid, c * 32 + e);
            const float2 x = ffma2(make_float2(__uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1])), two(rows.k_step, c * 32 + e),
                                   MOD ? fmul2(q2, mid) : ffma2(q2, mid, two(rows.v_log, c * 32 + e)));
            sr[c][e] = __float_as_uint(x.x);
            sr[c][e + 1] = __float_as_uint(x.y);
          }
      }
      if (!FOUR && (MOD || need_mask)) {  // the factors are spent here: scores in log2 units, hidden ones -inf
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float f = kf[c * 2 + e / 16];
            const float2 x = fmul2(make_float2(__uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1])), make_float2(f, f));
            sr[c][e] = __float_as_uint(x.x);
            sr[c][e + 1] = __float_as_uint(x.y);
          }
#pragma unroll
        for (int f = 0; f < kFactors; ++f) kf[f] = 1.0f;
      }
      if (MOD || need_mask) {
        if constexpr (MOD) {
          if (capped) cap_scores(sr, cap2);
          if (a.alibi_slopes) {
            const float d0 = fpos - static_cast<float>(kv0);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                sr[c][e] = __float_as_uint(
                    fmaf(-slope, fabsf(d0 - static_cast<float>(c * 32 + e)), __uint_as_float(sr[c][e])));
          }
          if constexpr (FOUR) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 x = fadd2(make_float2(__uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1])), two(rows.v_log, c * 32 + e));
                sr[c][e] = __float_as_uint(x.x);
                sr[c][e + 1] = __float_as_uint(x.y);
              }
          }
        }
        if (need_mask) {
          const int32_t lo_e = first - kv0, hi_e = end - kv0;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e < lo_e || c * 32 + e >= hi_e) sr[c][e] = __float_as_uint(-INFINITY);
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int f = 0; f < kFactors; ++f) {
        const uint32_t* const g = &sr[f / 2][(f & 1) * 16];
        float p0 = fmax3(__uint_as_float(g[0]), __uint_as_float(g[1]), __uint_as_float(g[2]));
        float p1 = fmax3(__uint_as_float(g[3]), __uint_as_float(g[4]), __uint_as_float(g[5]));
        float p2 = fmax3(__uint_as_float(g[6]), __uint_as_float(g[7]), __uint_as_float(g[8]));
        float p3 = fmax3(__uint_as_float(g[9]), __uint_as_float(g[10]), __uint_as_float(g[11]));
        p0 = fmax3(p0, __uint_as_float(g[12]), __uint_as_float(g[13]));
        p1 = fmax3(p1, __uint_as_float(g[14]), __uint_as_float(g[15]));
        if constexpr (FOUR) mx = fmaxf(mx, fmax3(fmaxf(p0, p1), p2, p3));
        else mx = fmaxf(mx, fmaf(fmax3(fmaxf(p0, p1), p2, p3), kf[f], sh.v_exp[slot][f]));
      }
      const bool grow = mx > m + kSlack;
      float f_o = 1.0f;
      if (grow) {
        f_o = ex2_approx(m - mx);
        l *= f_o;
        z *= f_o;
        m = mx;
      }
      // the P V before was committed ahead of this S: O is at rest
      if (i > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {  // 8 columns at a time: S is in registers
          uint32_t o[8];
          tmem_ld8(o_tmem + c * 8, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f_o);
          tmem_st8(o_tmem + c * 8, o);
        }
      }
      float2 z_sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
      const float neg = FOUR ? kStepLog - m : -m;
      const float2 neg_m = make_float2(neg, neg);
      float2 sum[4] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if constexpr (FOUR) {
            const int j = c * 32 + 2 * e;
            const float2 x = fadd2(make_float2(__uint_as_float(sr[c][2 * e]), __uint_as_float(sr[c][2 * e + 1])), neg_m);
            const float2 p = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            sum[e & 3] = ffma2(p, two(rows.v_rcp, j), sum[e & 3]);
            z_sum[e & 1] = ffma2(p, two(rows.v_mid, j), z_sum[e & 1]);
            pk[e] = pack2(p.x, p.y);
            continue;
          }
          const int f = c * 2 + e / 8;
          const float2 x = ffma2(make_float2(__uint_as_float(sr[c][2 * e]), __uint_as_float(sr[c][2 * e + 1])),
                                 make_float2(kf[f], kf[f]), neg_m);
          const float2 p = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          sum[e & 3] = fadd2(sum[e & 3], p);
          const float vf = sh.v_factor[slot][f];
          const float2 pv = fmul2(p, make_float2(vf, vf));
          pk[e] = pack2(pv.x, pv.y);
        }
        tmem_st16(s_tmem + c * 16, pk);
        if (c & 1) {  // the half's products can start (the O rescale has completed with it)
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&sh.p_full[t][c >> 1]);
        }
      }
      if constexpr (FOUR) z += (z_sum[0].x + z_sum[0].y) + (z_sum[1].x + z_sum[1].y);
      l += ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) + ((sum[2].x + sum[2].y) + (sum[3].x + sum[3].y));
    }
    // ---- O / l, or this chunk's share of it
    if (ok && n_own > 0) ok = warp_wait(&sh.o_full[t], 0, status);
    tc_fence_after();
    // written by the converters before the first S; with no tile there is nothing to scale
    const float vmax = FOUR ? 1.0f :
        n_own > 0 ? fmaxf(fmaxf(sh.v_max[0], sh.v_max[1]), fmaxf(sh.v_max[2], sh.v_max[3])) : 0.0f;
    auto kept = [&](int k) {  // read here, or the compiler would carry the values through the loop
      int32_t v;
      asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(smem_u32(&sh.place[k])));
      return v;
    };
    const int32_t r256 = t * kTileRows + r, n_rows = kept(2), q_row = kept(1) + min(r256, n_rows - 1);
    const bool stored = r256 < n_rows;
    const int64_t out_row = ((kept(0) + static_cast<int64_t>(q_row / G)) * a.g.n_q_heads + kept(3) * G + q_row % G) * D;
    const int32_t split = kept(4), n_splits = kept(6);
    // fp16: into the query tile's space (its last product is done), then out by whole rows
    const bool by_rows = a.out_dtype == AIHOST_F16;
    auto store32 = [&](int c, const float (&o)[32]) {
      if (by_rows) {
#pragma unroll
        for (int v = 0; v < 4; ++v)
          *reinterpret_cast<uint4*>(q_tile + chunk_off(r, 4 * c + v)) =
              make_uint4(pack2(o[8 * v], o[8 * v + 1]), pack2(o[8 * v + 2], o[8 * v + 3]),
                              pack2(o[8 * v + 4], o[8 * v + 5]), pack2(o[8 * v + 6], o[8 * v + 7]));
      } else if (stored) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.out) + out_row + c * 32);
#pragma unroll
        for (int v = 0; v < 8; ++v) dst[v] = make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
      }
    };
    auto flush_rows = [&] {
      if (!by_rows) return;
      __syncwarp();
      constexpr int LR = D / 8;  // lanes to a row
#pragma unroll 4
      for (int k = 0; k < LR; ++k) {
        const int src = k * (32 / LR) + lane / LR;  // row of the warp
        const int64_t row_at = __shfl_sync(0xffffffffu, out_row, src);
        const bool on = __shfl_sync(0xffffffffu, static_cast<int>(stored), src);
        if (on)
          *reinterpret_cast<uint4*>(static_cast<__half*>(a.out) + row_at + lane % LR * 8) =
              *reinterpret_cast<const uint4*>(q_tile + chunk_off(quarter * 32 + src, lane % LR));
      }
    };
    const int64_t part_unit = kept(5);
    // partials: [unit after the whole ones][split][D / 4][256 rows] of 4 floats, so that a warp's rows lie together
    float4* const part = reinterpret_cast<float4*>(a.part_o) + (part_unit * a.max_splits) * (D / 4) * kRows + r256;
    float2* const part_ml = reinterpret_cast<float2*>(a.part_ml) + part_unit * a.max_splits * kRows + r256;
    if (ok) {
      const float inv_l = n_splits > 1 ? 1.0f : l != 0.0f ? 1.0f / l : 0.0f;
      const float unit_o = n_splits > 1 ? 1.0f / kVUnit : l != 0.0f ? 1.0f / kVUnit / l : 0.0f;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (n_own > 0) {
          uint32_t u[32];
          tmem_ld32(o_tmem + c * 32, u);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if constexpr (FOUR) o[e] = fmaf(__uint_as_float(u[e]), 1.0f / kStepUnit, z) * inv_l;
            else o[e] = __uint_as_float(u[e]) * unit_o * vmax;  // in this order: unit_o * vmax may be too small a number
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.0f;
        }
        if (n_splits == 1) {
          store32(c, o);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            part[(static_cast<int64_t>(split) * (D / 4) + c * 8 + e) * kRows] =
                make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
      if (n_splits > 1) part_ml[static_cast<int64_t>(split) * kRows] = make_float2(m, l);
      else flush_rows();
    }
    if (n_splits > 1) {  // the last block of this tile and head to arrive merges the chunks
      __threadfence();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (threadIdx.x == 128) sh.last = last_to_arrive(a.counters + part_unit, n_splits);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (sh.last) {
        __threadfence();
        float mm = kNoMax;
        for (int sp = 0; sp < n_splits; ++sp) mm = fmaxf(mm, __ldcg(part_ml + static_cast<int64_t>(sp) * kRows).x);
        float ll = 0.0f;
        for (int sp = 0; sp < n_splits; ++sp) {
          const float2 v = __ldcg(part_ml + static_cast<int64_t>(sp) * kRows);
          ll += v.y * ex2_approx(v.x - mm);
        }
        const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.0f;
          for (int sp = 0; sp < n_splits; ++sp) {
            const float f = ex2_approx(__ldcg(part_ml + static_cast<int64_t>(sp) * kRows).x - mm) * inv;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 v = __ldcg(part + (static_cast<int64_t>(sp) * (D / 4) + c * 8 + e) * kRows);
              o[4 * e] += v.x * f, o[4 * e + 1] += v.y * f, o[4 * e + 2] += v.z * f, o[4 * e + 3] += v.w * f;
            }
          }
          store32(c, o);
        }
        flush_rows();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool MOD, bool REST, bool FOUR>
cudaError_t launch_d(const Kv8AttnArgs& a, cudaStream_t st) {
  auto kern = kv8_prefill_kernel<D, MOD, REST, FOUR>;
  constexpr int kBytes = Cfg<D, REST, FOUR>::SMEM;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (e != cudaSuccess) return e;
  // not a dependent launch: waiting blocks would take whole SMs, 6 % slower on batches of short prompts
  const int64_t blocks = a.whole + (static_cast<int64_t>(a.tiles) * a.g.n_kv_heads - a.whole) * a.max_splits;
  kern<<<static_cast<unsigned>(blocks), kThreads, kBytes, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

void kv8_prefill_plan(const Kv8Geom& g, int32_t batch, int32_t n_tokens, int32_t max_new, int32_t max_kv, int32_t num_sms,
                      int32_t* tiles, int32_t* whole, int32_t* chunk, int32_t* splits, double* end_out) {
  const int32_t G = g.n_q_heads / g.n_kv_heads;
  const int64_t n = static_cast<int64_t>(max_new) * G <= kRows ? batch : static_cast<int64_t>(n_tokens) * G / kRows + batch;
  const int64_t units = n * g.n_kv_heads, tiles_kv = (max_kv + kKeys - 1) / kKeys;
  // One block per SM at a time; kFixed and kPart: a block's fixed work, and a partial result's writing
  // and its share of the merge, in tiles. The lengths are on the device; where the sequences bring about
  // as many new rows each (n_tokens near batch * max_new), they are taken as alike, and waves count. Else
  // the blocks are taken as of every length, spread evenly but for a third of one.
  constexpr double kFixed = 3.0, kPart = 2.0, kMerge = 0.7;
  const int64_t of_one = (static_cast<int64_t>(max_new) * G + kRows - 1) / kRows;
  const int64_t full = std::min(units, of_one * batch * g.n_kv_heads);  // tiles that can have rows
  const double even = static_cast<double>(n_tokens) / (static_cast<double>(batch) * max_new);
  const double average = (even < 1.0 ? even : 1.0) * (static_cast<double>(tiles_kv) - 0.5 * max_new / kKeys);
  const bool alike = even > 0.9 && 3 * static_cast<int64_t>(max_new) < max_kv;
  int64_t best = 1, best_whole = 0;
  double best_end = 1e30;
  for (int64_t s = 1; s <= 32 && (s == 1 || tiles_kv / s >= 4); ++s) {
    const double block = static_cast<double>((tiles_kv + s - 1) / s) + kFixed + (s > 1 ? kPart : 0.0);
    double end = block;
    if (even > 0.9) {
      end = static_cast<double>((full * s + num_sms - 1) / num_sms) * block;
    } else {
      const double spread = full * (average + even * s * (block - (tiles_kv + s - 1) / s)) / num_sms + 0.35 * block;
      if (spread > end) end = spread;
    }
    if (s > 1) end += kMerge * s;
    if (end < best_end * 0.97) {
      best_end = end;
      best = s;
      best_whole = 0;
    }
    // Units alike that fill some waves and part of one more: only what is left over is split. Measured
    // against none split: 152 units of 103 tiles 318 -> 275 us, 320 of 90 477 -> 419, 192 of 28 136 -> 117,
    // 256 of 128 508 -> 497.
    const int64_t waves = full / num_sms;
    if (s > 1 && alike && waves > 0) {
      end = static_cast<double>(waves) * (static_cast<double>(tiles_kv) + kFixed) +
            static_cast<double>(((full - waves * num_sms) * s + num_sms - 1) / num_sms) * block + kMerge * s;
      if (end < best_end * 0.97) {
        best_end = end;
        best = s;
        best_whole = waves * num_sms * units / full;  // with its share of the tiles that turn out empty
      }
    }
  }
  if (units - best_whole > kKv8Counters) best = 1, best_whole = 0;
  const int64_t c = (tiles_kv + best - 1) / best;
  *end_out = best_end;
  *tiles = static_cast<int32_t>(n);
  *whole = static_cast<int32_t>(best_whole);
  *chunk = static_cast<int32_t>(c * kKeys);
  *splits = static_cast<int32_t>((tiles_kv + c - 1) / c);
}

int32_t kv8_prefill_rows() { return kRows; }

template <bool FOUR>
static cudaError_t launch_prompts(const Kv8AttnArgs& a, cudaStream_t st) {
  const bool mod = a.score_cap > 0.0f || a.alibi_slopes;
  if (a.g.head_dim == 64) return mod ? launch_d<64, true, true, FOUR>(a, st) : launch_d<64, false, true, FOUR>(a, st);
  if (a.exact_q) return mod ? launch_d<128, true, true, FOUR>(a, st) : launch_d<128, false, true, FOUR>(a, st);
  return mod ? launch_d<128, true, false, FOUR>(a, st) : launch_d<128, false, false, FOUR>(a, st);
}

cudaError_t launch_kv8_prefill(const Kv8AttnArgs& a, cudaStream_t st) { return launch_prompts<false>(a, st); }
cudaError_t launch_kv4_prefill(const Kv8AttnArgs& a, cudaStream_t st) { return launch_prompts<true>(a, st); }

}  // namespace aihost
