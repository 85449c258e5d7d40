// kv4_attn.cu — attention of few query rows over the 4-bit paged cache (decode, drafts, fp32 tensors).
//
// A cached row of a head is D codes c of 4 bits and a pair (low, step): value = low + step c. With it
//   q.k = step (q.c) + low sum(q)        o = sum_j (p_j step_j) c_j + sum_j p_j low_j
// so the products run over the codes alone, exactly, and the pairs enter in fp32 outside.
//
// The work is split as over the 8-bit cache (kv8_attn.cu): a block takes R = 8 or 16 query rows of one KV head
// and a chunk of the cache rows, its four warps walk 32-row steps of the chunk with mma.sync m16n8k16 on
// transposed products (S^T = K Q^T, O^T += V^T P^T), each with a ring of its own in shared memory
// (cp.async); warps merge through shared memory, chunks through partials.
//
// A word holds 8 codes, nibble n element 2 (n mod 4) + n / 4. Two nibbles 16 bits apart, moved to bits 4 to 7 and masked,
// are two neighbours as the fp16 numbers 16 c 2^-24 (below the normal ones, exact): no conversion. V comes by
// ldmatrix.trans, a register holding 16 bits (four codes) of one row and of the next; its last operand is the whole upper
// byte, with the code before in the lower bits, whose tile takes that out of it in the end.
// V's codes have to enter less their mean, value = (low + 7.5 step) + step (c - 7.5): else O carries 7.5 step times the sum of P,
// many times a result that averages thousands of rows, and cancels in the end. So each step's sum of P (a product with
// ones, thus of what P was rounded to) is taken off O 7.5 times, between the step's two blocks of rows, where O
// is smallest beside it. Measured, error of the 32 x 32768 rows below against 64 bits: with the eight left in 5.6e-4; with
// the codes at bits 0 to 3 3.5e-4 (a product's rounding goes by the exponent 2^-14 of numbers below the normal
// ones); so 2.5e-4; c - 8 by one fp16 fma each 2.6e-4, 15 % slower. The fp16 plain form has 2.1e-4.
// fp32 tensors: K's operands are c - 8 so made, V's c - 7.5, whose mean is 0, and a step's sums go to O by fp32 additions: the
// tensor core's cut what falls below the accumulator's last bit. Error 3e-7 whatever the length (plain form 2e-7 to 2e-6);
// with c - 8 for V and O as the accumulator it grew with the rows, 1.2e-5 at 32000 and 2.7e-5 at 64000; with c - 7.5 alone
// 1.6e-6 and 1.8e-6. 16 sequences of 8000 rows, 32/8 heads, rotated, 70 us (68 without either).
//
// A cached row is used by R query rows, 2 R products a code: bytes and instructions bound it, not the tensor pipe.
// Measured, head_dim 128, 8 KV heads: 64 sequences of 256 to 8192 rows, q rotated, 96 us (319 MB, 3.3 TB/s, 51 % of a
// copy's measured 6.57); 32 of 32768 with 64 query heads and capped scores 249 us, 279 under sustained load (1.14 GB: 4.6
// and 4.1 TB/s); one of 130001 57 us, one of 513 7. A 32-row step takes ~560 warp instructions, its share of a block's fixed work
// among them, half of them on the ALU pipe (of a word's codes, K's take three shifts and four masks, V's two shifts, three
// masks and a permutation), issued in 50 % of the slots; at a copy's rate a scheduler would have ~730 cycles for it, and it
// takes ~1110. Not better: four blocks an SM with three stages of the ring and 128 registers a thread (98 and 257 us for the
// first two); with these, V's words loaded by rows and permuted, or c - 8 made for V in registers (each 20 us more for the
// second).
#include <type_traits>

#include "common.cuh"
#include "kv8.h"
#include "kv8_tile.cuh"
#include "kv_split.cuh"

namespace aihost {
namespace {

constexpr int kStages = 4;  // of the warp's ring
constexpr int kBlocks = 3;  // on an SM, of 8 query rows (of 16: two)
constexpr int kChunkMax = 8192;
constexpr float kCodeUnit = 1048576.0f;  // a code enters times 2^-20
constexpr uint32_t kOnes = 0x3c003c00u;

// The operands of K and V: nibbles n and n + 4 of x times 2^-20; V's n = 3 with nibble 2 / 16. fp32 tensors: K's less 8, V's less
// their mean.
template <int PREC>
__device__ __forceinline__ uint32_t k_codes(uint32_t x, int n) {
  if constexpr (PREC == kPairQP) return codes_less_8(x, n);
  return (n == 0 ? x << 4 : n == 1 ? x : n == 2 ? x >> 4 : x >> 8) & 0x00f000f0u;
}
template <int PREC>
__device__ __forceinline__ uint32_t v_codes(uint32_t x, int n) {
  if constexpr (PREC == kPairQP) return codes_less_mean(x, n);
  return n == 3 ? __byte_perm(x, 0, 0x4341) : k_codes<PREC>(x, n);
}
__host__ __device__ constexpr float v_mean(int n) { return (n == 3 ? 7.5f + 7.5f / 16.0f : 7.5f) / kCodeUnit; }

// copy16 with offsets in the instruction.
template <uint32_t TO, uint32_t FROM>
__device__ __forceinline__ void copy16_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(TO), "n"(FROM) : "memory");
}
template <int N>
using Int = std::integral_constant<int, N>;
// f(Int<0>()) .. f(Int<N - 1>())
template <int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (N > 0) {
    unrolled<N - 1>(f);
    f(Int<N - 1>());
  }
}

// Four 8 x 8 matrices of 16 bits, transposed: lane (g, t4) gets column g of rows 2 t4 and 2 t4 + 1 of each; lane i of the
// eight for a matrix names row i.
template <uint32_t OFFSET>
__device__ __forceinline__ void load_transposed(uint32_t (&x)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4 + %5];"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
               : "r"(at), "n"(OFFSET)
               : "memory");
}

// P enters times V's step times kVUnit. The running maximum is that of score + floor(log2 step), so that the product
// is at most 2^(kSlack + 1) kVUnit = 2^15 whatever the step (fp16: 2^-24 to 2^16), and a row's own largest
// one at least kVUnit: its weights keep their bits whatever steps other rows have.
template <int PREC>
constexpr float kVUnit = PREC == kPairQP ? 16384.0f : 64.0f;

// floor(log2 |step|), -25 for 0: fp16 in fp32, so a normal number or zero.
__device__ __forceinline__ float exp_of(float step) {
  const uint32_t e = (__float_as_uint(step) >> 23) & 0xffu;
  return static_cast<float>(static_cast<int32_t>(max(e, 102u)) - 127);
}

// Where 16-byte chunk c of a step's row r lies (rows of D/2 bytes): what is loaded together, whole lines of K and a
// chunk of eight rows of V, falls into different banks.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if (D == 128) return static_cast<uint32_t>((r >> 1) * 128 + (((r & 1) * 4 + (c ^ ((r >> 1) & 3))) << 4));
  return static_cast<uint32_t>((r >> 2) * 128 + (((r & 3) * 2 + (c ^ ((r >> 2) & 1))) << 4));
}

template <int D, int NT>
struct SplitSmem {  // the rings, and over them the merge's O
  static constexpr int kCodes = kStep * D / 2;                  // a step's codes of K or V
  static constexpr int kStageBytes = 2 * kCodes + 2 * kStep * 4;  // with the ranges after them
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kMerge = kWarps * NT * 8 * (D + 4) * 4;
  static constexpr int kBytes = kRing > kMerge ? kRing : kMerge;
};

// FOLD: at most four query rows, whose rotated q's two parts take the eight columns together, the fp16 the first four and
// the rest the others; their scores are added across lanes, and both halves go on with the same rows. Half the products
// of K and half the registers for q: 6 us less for the 64 sequences above.
template <int D, int NT, int PREC, bool MOD, bool FOLD>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? kBlocks : 2) kv4_mma_kernel(const __grid_constant__ Kv8AttnArgs a) {
  using S = SplitSmem<D, NT>;
  constexpr int R = NT * 8;
  constexpr int KS = D / 16;       // k steps of S^T = K Q^T
  constexpr int KW = D / 32;       // words of a K row per lane
  constexpr int MT = D / 16;       // 16-row tiles of O^T
  constexpr int VP = D / 64;       // pairs of 16-byte chunks of a V row: four tiles each
  constexpr int NQ = PREC == kPlain || FOLD ? 1 : 2;
  static_assert(!FOLD || (NT == 1 && PREC == kPairQ), "four rows of a rotated fp16 q");
  constexpr float kCodeScale = PREC == kPairQP ? 1.0f : kCodeUnit;
  extern __shared__ __align__(128) uint8_t ring[];
  float(*const o_sh)[R][D + 4] = reinterpret_cast<float(*)[R][D + 4]>(ring);
  __shared__ float ml_sh[kWarps][R][2];
  // a step's rows: K's factor and offset, V's, each twice, for packed fp32, and floor(log2) of V's step
  __shared__ float4 k_sh[kWarps][kStep], v_sh[kWarps][kStep];
  __shared__ float e_sh[kWarps][kStep];
  __shared__ int32_t last_sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int32_t H = a.g.n_kv_heads, G = a.g.n_q_heads / H, ps = a.g.page_shift;
  const int32_t h = static_cast<int32_t>(blockIdx.x % H);
  const int64_t tile = blockIdx.x / H;
  const int32_t split = static_cast<int32_t>(blockIdx.y);
  griddep_wait();
  griddep_launch_dependents();
  // One tile a sequence and no documents: the sequence and the first row of this chunk are known before
  // the lengths, so the table entry of this lane's first block of rows comes along with them.
  const bool known = static_cast<int64_t>(a.max_new) * G <= R && !a.row_first;
  int32_t entry_early = 0;
  if (known) {
    const int64_t row = static_cast<int64_t>(split) * a.chunk + warp * kStep + (lane >> 1) * (kWarps * kStep) + (lane & 1) * kSub;
    if ((row >> ps) < a.g.max_pages) entry_early = a.block_table[tile * a.g.max_pages + (row >> ps)];
  }
  const Tile tl = find_tile(a, tile, G, R, lane);
  if (!tl.ok) return;
  const int32_t n_rows = min(R, tl.n_new * G - tl.row0);

  // ---- which cache rows each query row sees; this lane's two columns per N tile, and the tile's range
  int32_t c_first[NT][2], c_end[NT][2];
  float c_pos[NT][2], c_slope[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = (nt * 8 + 2 * t4 + c) & (FOLD ? 3 : 15);
      int32_t pos;
      row_range(a, tl, G, n_rows, r, c_first[nt][c], c_end[nt][c], pos);
      c_pos[nt][c] = static_cast<float>(pos);
      c_slope[nt][c] =
          MOD && a.alibi_slopes ? a.alibi_slopes[h * G + (tl.row0 + min(r, n_rows - 1)) % G] * kLog2e : 0.0f;
    }
  int32_t lo, hi, lo_max, hi_min;
  {
    int32_t first, end, pos;
    row_range(a, tl, G, n_rows, lane & (FOLD ? 3 : R - 1), first, end, pos);
    lo = __reduce_min_sync(0xffffffffu, first);
    lo_max = __reduce_max_sync(0xffffffffu, first);
    hi = __reduce_max_sync(0xffffffffu, end);
    hi_min = __reduce_min_sync(0xffffffffu, end);
  }
  const int32_t base = min(lo, hi) & ~(kSub - 1);
  const int32_t n_splits = (hi - base - 1) / a.chunk + 1;  // base <= hi; one for an empty range
  if (split >= n_splits) return;
  const int32_t k_begin = base + split * a.chunk, k_end = k_begin + min(hi - k_begin, a.chunk);
  const int32_t* const table = a.block_table + static_cast<int64_t>(tl.b) * a.g.max_pages;
  bool stray = false;  // a page id outside the pool reads page 0 and sets the status

  // ---- this warp's steps: step i is rows [k_of(i), k_of(i) + 32), as blocks of 16 rows 2 i and 2 i + 1
  const int32_t k_mine = k_begin + warp * kStep;
  const int32_t n_steps = k_mine < k_end ? (k_end - k_mine - 1) / (kWarps * kStep) + 1 : 0;
  auto row_of = [&](int32_t sub) { return k_mine + (sub >> 1) * (kWarps * kStep) + (sub & 1) * kSub; };
  // lane j: the pool row where block 32 * round + j begins (none past the end)
  constexpr int64_t kNowhere = -1;
  auto place_at = [&](int32_t row, int32_t entry) -> int64_t {
    return ((page_or_first(entry, a.g.n_pages, stray) * H + h) << ps) + (row & (a.g.page_rows - 1));
  };
  auto place_of = [&](int32_t sub) -> int64_t {
    const int32_t row = row_of(sub);
    return (sub >> 1) >= n_steps || row >= k_end ? kNowhere : place_at(row, table[row >> ps]);
  };
  int64_t place = kNowhere;
  if (!known) place = place_of(lane);
  else if ((lane >> 1) < n_steps && row_of(lane) < k_end) place = place_at(row_of(lane), entry_early);
  int64_t place_next = n_steps > 16 ? place_of(32 + lane) : kNowhere;
  uint8_t* const my_ring = ring + warp * (kStages * S::kStageBytes);
  // a half-warp copies one of a step's two blocks: chunks j * 16 + lane of its K and V rows, and 64 bytes of either's
  // ranges
  constexpr int CR = D / 32;                  // chunks per row
  constexpr int NC = kSub * CR / 16;          // per lane
  const int half = lane >> 4, l16 = lane & 15;
  uint32_t to[2];  // the swizzle repeats every 8 rows (16): two patterns of destinations (one)
#pragma unroll
  for (int j = 0; j < 2; ++j)
    to[j] = smem_u32(my_ring) + half * (kSub * D / 2) + chunk_at<D>((j * 16 + l16) / CR, (j * 16 + l16) % CR) - j * 256;
  const uint32_t to_range = smem_u32(my_ring) + 2 * S::kCodes + ((l16 >> 2) & 1) * (kStep * 4) + half * (kSub * 4) + (l16 & 3) * 16;
  const uint32_t* const range_from = (l16 & 4 ? a.v_range : a.k_range) + (l16 & 3) * 4;
  auto fetch = [&](int32_t i, int32_t round, uint32_t dst) {  // step i into the stage at dst
    const int32_t sub = 2 * i + half;
    const int64_t at = __shfl_sync(0xffffffffu, (i >> 4) == round ? place : place_next, sub & 31);
    if (i < n_steps && at != kNowhere) {
      const int8_t *kp = a.k_pool + at * (D / 2) + l16 * 16, *vp = a.v_pool + at * (D / 2) + l16 * 16;
      const uint32_t to0 = to[0] + dst, to1 = to[1] + dst;
      unrolled<NC>([&](auto index) {
        constexpr int j = decltype(index)::value;
        copy16_at<j * 256, j * 256>(j & 1 ? to1 : to0, kp);
        copy16_at<S::kCodes + j * 256, j * 256>(j & 1 ? to1 : to0, vp);
      });
      if (l16 < 8) copy16(to_range + dst, range_from + at);
    }
    copies_commit();
  };
  // ldmatrix: matrix lane / 8 is rows 0 to 7 or 8 to 15 of a chunk, or of the next one
  const uint32_t v_row = static_cast<uint32_t>((lane & 7) + (lane & 8)), v_chunk = static_cast<uint32_t>(lane >> 4);
  const uint32_t v_at = smem_u32(my_ring) + S::kCodes + chunk_at<D>(v_row, v_chunk);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i, 0, i * S::kStageBytes);

  uint32_t qf[NQ][NT][KS][2];
  float q_unit[NT][2];  // what the scores of this lane's two columns take back
  if constexpr (FOLD) {
    uint32_t parts[2][NT][KS][2];
    load_q<D, NT, PREC, true>(a, tl, G, h, n_rows, g & 3, t4, parts, q_unit);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[0][0][k][e] = g < 4 ? parts[0][0][k][e] : parts[1][0][k][e];
  } else {
    load_q<D, NT, PREC, true>(a, tl, G, h, n_rows, g, t4, qf, q_unit);
  }
  float q_sum[NT][2];  // the columns' sums of q, as it enters
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float sum = 0.0f;
#pragma unroll
    for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qf[n][nt][k][e]));
          sum += f.x + f.y;
        }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);  // row g's
    if (FOLD) sum += __shfl_xor_sync(0xffffffffu, sum, 16);
#pragma unroll
    for (int c = 0; c < 2; ++c) q_sum[nt][c] = __shfl_sync(0xffffffffu, sum, (2 * t4 + c) * 4);
  }

  float o[MT][NT][4];
  float m[NT][2], l[NT][2], z[NT][2];  // z: the sum of p times V's lows
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = kNoMax;
    l[nt][0] = l[nt][1] = z[nt][0] = z[nt][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
  }
  const bool capped = MOD && a.score_cap > 0.0f;
  const float q_scale = a.scale * (1.0f / kQUnit<PREC>), s_unit = capped ? q_scale / a.score_cap : q_scale * kLog2e;
  const float cap2 = a.score_cap * kLog2e;

  uint32_t at = 0, at_next = (kStages - 1) * S::kStageBytes;  // this step's stage, and that of the step to fetch
  for (int32_t i = 0, round = 0; i < n_steps; ++i) {
    if (i == 16 * (round + 1)) {
      ++round;
      place = place_next;
      if (i + 16 < n_steps) place_next = place_of(2 * i + 32 + lane);
    }
    fetch(i + kStages - 1, round, at_next);
    copies_wait<kStages - 1>();
    __syncwarp();
    const uint8_t* const stage = my_ring + at;
    const uint32_t v_stage = v_at + at;
    at_next = at;
    at = at == (kStages - 1) * S::kStageBytes ? 0 : at + S::kStageBytes;
    const uint32_t* const ranges = reinterpret_cast<const uint32_t*>(stage + 2 * S::kCodes);
    const int32_t k = row_of(2 * i);
    {  // a lane takes one row's ranges
      const uint32_t kr = ranges[lane], vr = ranges[kStep + lane];
      const float2 kv = __half22float2(*reinterpret_cast<const __half2*>(&kr));
      const float2 vv = __half22float2(*reinterpret_cast<const __half2*>(&vr));
      // a range of V's that is no number marks its row through K's, as one of K's does: of a hidden row, whose weight is 0,
      // nothing may come, and an infinite score of a row seen could be -infinity
      const bool fine = fabsf(vv.x) + fabsf(vv.y) < INFINITY;
      const float kf = fine && fabsf(kv.x) + fabsf(kv.y) < INFINITY ? kv.y * (s_unit * kCodeScale) : __uint_as_float(0x7fffffffu);
      const float kz = (PREC == kPairQP ? fmaf(8.0f, kv.y, kv.x) : kv.x) * s_unit;
      const float vf = fine ? vv.y * kVUnit<PREC> : 0.0f, vz = fine ? fmaf(7.5f, vv.y, vv.x) : 0.0f;
      k_sh[warp][lane] = make_float4(kf, kf, kz, kz);
      v_sh[warp][lane] = make_float4(vf, vf, vz, vz);
      e_sh[warp][lane] = exp_of(vv.y);
    }
    // ---- S^T = K Q^T
    float s[2][NT][4], s_odd[2][NT][4];  // in two sums, for chains half as long
    uint32_t w0[2][KW], w1[2][KW];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][nt][e] = s_odd[u][nt][e] = 0.0f;
      if constexpr (KW == 4) {
        const uint4 r0 = *reinterpret_cast<const uint4*>(stage + chunk_at<D>(u * kSub + g, t4));
        const uint4 r1 = *reinterpret_cast<const uint4*>(stage + chunk_at<D>(u * kSub + g + 8, t4));
        w0[u][0] = r0.x, w0[u][1] = r0.y, w0[u][2] = r0.z, w0[u][3] = r0.w;
        w1[u][0] = r1.x, w1[u][1] = r1.y, w1[u][2] = r1.z, w1[u][3] = r1.w;
      } else {
        const uint2 r0 = *reinterpret_cast<const uint2*>(stage + chunk_at<D>(u * kSub + g, t4 >> 1) + (t4 & 1) * 8);
        const uint2 r1 = *reinterpret_cast<const uint2*>(stage + chunk_at<D>(u * kSub + g + 8, t4 >> 1) + (t4 & 1) * 8);
        w0[u][0] = r0.x, w0[u][1] = r0.y, w1[u][0] = r1.x, w1[u][1] = r1.y;
      }
    }
#pragma unroll
    for (int j = 0; j < KW; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {  // elements 0, 1, 4, 5 of the word, then 2, 3, 6, 7
          const uint32_t a0 = k_codes<PREC>(w0[u][j], k2), a1 = k_codes<PREC>(w1[u][j], k2);
          const uint32_t a2 = k_codes<PREC>(w0[u][j], k2 + 2), a3 = k_codes<PREC>(w1[u][j], k2 + 2);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
              mma16816(k2 ? s_odd[u][nt] : s[u][nt], a0, a1, a2, a3, qf[n][nt][2 * j + k2][0], qf[n][nt][2 * j + k2][1]);
        }
    // ---- scores (log2 units), masks, running maximum
    __syncwarp();
    const bool edge = k < lo_max || k + kStep > hi_min;
    bool grow = false;
    float far = 0.0f;  // the largest of the lane's scores, in units of the cap
    of_pairs<NT>(s, [&](float2 x, int u, int nt, int e) {
      const float4 r = k_sh[warp][u * kSub + (e >> 1) * 8 + g];
      x = fadd2(make_float2(s_odd[u][nt][e], s_odd[u][nt][e + 1]), x);
      if constexpr (FOLD) x = fadd2(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, 2), __shfl_xor_sync(0xffffffffu, x.y, 2)));
      x = ffma2(x, make_float2(r.x, r.y), fmul2(make_float2(q_sum[nt][0], q_sum[nt][1]), make_float2(r.z, r.w)));
      if (PREC == kPairQP) x = fmul2(x, make_float2(q_unit[nt][0], q_unit[nt][1]));
      if (MOD) far = fmaxf(far, fmaxf(fabsf(x.x), fabsf(x.y)));
      return x;
    });
    if constexpr (MOD) modify_scores<NT>(a, capped, cap2, far, k, g, c_slope, c_pos, s);
    if (edge) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int32_t row = k + u * kSub + g + (e >> 1) * 8;
            if (row < c_first[nt][e & 1] || row >= c_end[nt][e & 1]) s[u][nt][e] = -INFINITY;
          }
    }
    float most[NT][2];  // of the lane's rows, score + exponent
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float2 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float ve = e_sh[warp][(j >> 1) * kSub + (j & 1) * 8 + g];
        x[j] = make_float2(s[j >> 1][nt][2 * (j & 1)] + ve, s[j >> 1][nt][2 * (j & 1) + 1] + ve);
      }
      most[nt][0] = fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x));
      most[nt][1] = fmaxf(fmaxf(x[0].y, x[1].y), fmaxf(x[2].y, x[3].y));
#pragma unroll
      for (int c = 0; c < 2; ++c) grow |= most[nt][c] > m[nt][c] + kSlack<PREC>;
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = most[nt][c];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float m_new = fmaxf(m[nt][c], mx), f = ex2_approx(m[nt][c] - m_new);
          m[nt][c] = m_new;
          l[nt][c] *= f;
          z[nt][c] *= f;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            o[t][nt][c] *= f;
            o[t][nt][c + 2] *= f;
          }
        }
    }
    // ---- P and its fragments
    constexpr int NP = PREC == kPairQP ? 2 : 1;
    uint32_t pf[2][NP][NT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float4 r = v_sh[warp][u * kSub + (e >> 1) * 8 + g];
          const float2 x = fadd2(make_float2(s[u][nt][e], s[u][nt][e + 1]), make_float2(-m[nt][0], -m[nt][1]));
          const float2 v = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          const float2 sum = fadd2(make_float2(l[nt][0], l[nt][1]), v), pv = fmul2(v, make_float2(r.x, r.y));
          const float2 zs = ffma2(v, make_float2(r.z, r.w), make_float2(z[nt][0], z[nt][1]));
          l[nt][0] = sum.x, l[nt][1] = sum.y, z[nt][0] = zs.x, z[nt][1] = zs.y;
          p[e] = pv.x, p[e + 1] = pv.y;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t hi2 = pack2(p[2 * c], p[2 * c + 1]);
          pf[u][0][nt][c] = movmatrix_t(hi2);
          if constexpr (PREC == kPairQP) pf[u][NP - 1][nt][c] = movmatrix_t(pack2_rest(p[2 * c], p[2 * c + 1], hi2));
        }
      }
    // ---- O^T += V^T P^T: tile 4 w + n is operands n of chunks 2 w and 2 w + 1
    if constexpr (PREC == kPairQP) {  // a step's sums apart, added to O in fp32
      unrolled<VP>([&](auto index) {
        constexpr int w = decltype(index)::value;
        uint32_t x[2][4];
        load_transposed<0>(x[0], w ? v_stage ^ 32u : v_stage);
        load_transposed<kSub * D / 2>(x[1], w ? v_stage ^ 32u : v_stage);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float part[4] = {};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t a0 = v_codes<PREC>(x[u][0], n), a1 = v_codes<PREC>(x[u][2], n);
              const uint32_t a2 = v_codes<PREC>(x[u][1], n), a3 = v_codes<PREC>(x[u][3], n);
#pragma unroll
              for (int n2 = 0; n2 < NP; ++n2) mma16816(part, a0, a1, a2, a3, pf[u][n2][nt][0], pf[u][n2][nt][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float2 y = fadd2(make_float2(part[e], part[e + 1]), make_float2(o[4 * w + n][nt][e], o[4 * w + n][nt][e + 1]));
              o[4 * w + n][nt][e] = y.x, o[4 * w + n][nt][e + 1] = y.y;
            }
          }
      });
    } else {
      float total[NT][4] = {};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < 2; ++u) mma16816(total[nt], kOnes, kOnes, kOnes, kOnes, pf[u][0][nt][0], pf[u][0][nt][1]);
      unrolled<2 * VP>([&](auto index) {
        constexpr int u = decltype(index)::value / VP, w = decltype(index)::value % VP;
        if constexpr (u == 1) {
#pragma unroll
          for (int i = 4 * w; i < 4 * w + 4; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float mean = -v_mean(i & 3);
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const float2 y = ffma2(make_float2(total[nt][0], total[nt][1]), make_float2(mean, mean),
                                       make_float2(o[i][nt][e], o[i][nt][e + 1]));
                o[i][nt][e] = y.x, o[i][nt][e + 1] = y.y;
              }
            }
        }
        uint32_t x[4];  // rows 0 to 7 and 8 to 15 of the first chunk, then of the second
        load_transposed<u * (kSub * D / 2)>(x, w ? v_stage ^ 32u : v_stage);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t a0 = v_codes<PREC>(x[0], n), a1 = v_codes<PREC>(x[2], n);
          const uint32_t a2 = v_codes<PREC>(x[1], n), a3 = v_codes<PREC>(x[3], n);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[4 * w + n][nt], a0, a1, a2, a3, pf[u][0][nt][0], pf[u][0][nt][1]);
        }
      });
    }
    __syncwarp();  // every lane has its rows: the slot may be filled again
  }
  if (stray) atomicOr(a.status, kStatusBadIndex);

  copies_wait<0>();
  __syncthreads();  // the rings become the merge's space
  // ---- merge the four warps: lane (g, t4) holds, of rows 2 t4 and 2 t4 + 1, in tile 4 w + n elements 2 n + (g & 1) of
  // words 8 w + g / 2 and, 8 rows on in the tile, 8 w + 4 + g / 2
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
        z[nt][c] += __shfl_xor_sync(0xffffffffu, z[nt][c], d);
      }
      const int r = nt * 8 + 2 * t4 + c;
      if (g == 0) ml_sh[warp][r][0] = m[nt][c], ml_sh[warp][r][1] = l[nt][c];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          float& v = o[i][nt][c + 2 * b];
          if (PREC != kPairQP && (i & 3) == 3) v = fmaf(o[i - 1][nt][c + 2 * b], -0.0625f, v);
          o_sh[warp][r][((i >> 2) * 8 + b * 4 + (g >> 1)) * 8 + (i & 3) * 2 + (g & 1)] =
              fmaf(v, kCodeScale / kVUnit<PREC>, z[nt][c]);
        }
    }
  __syncthreads();
  merge_block<D, NT>(a, tl, G, h, n_rows, split, n_splits, o_sh, ml_sh, last_sh);
}

template <int D, int NT, int PREC, bool MOD, bool FOLD>
cudaError_t launch_one(const Kv8AttnArgs& a, cudaStream_t st) {
  constexpr int kBytes = SplitSmem<D, NT>::kBytes;
  auto kern = kv4_mma_kernel<D, NT, PREC, MOD, FOLD>;
  if (kBytes > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) return e;
  }
  return launch_dependent(kern, dim3(static_cast<unsigned>(a.tiles) * a.g.n_kv_heads, a.max_splits), kWarps * 32, kBytes, st, a);
}

template <int D, int NT, int PREC, bool FOLD = false>
cudaError_t launch_mod(const Kv8AttnArgs& a, cudaStream_t st) {
  return a.score_cap > 0.0f || a.alibi_slopes ? launch_one<D, NT, PREC, true, FOLD>(a, st) : launch_one<D, NT, PREC, false, FOLD>(a, st);
}

template <int D, int NT>
cudaError_t launch_prec(const Kv8AttnArgs& a, cudaStream_t st) {
  if (a.q_dtype == AIHOST_F32) return launch_mod<D, NT, kPairQP>(a, st);
  if (a.rope_mode != AIHOST_ROPE_NONE) {
    if constexpr (NT == 1) {
      if (static_cast<int64_t>(a.max_new) * (a.g.n_q_heads / a.g.n_kv_heads) <= 4) return launch_mod<D, NT, kPairQ, true>(a, st);
    }
    return launch_mod<D, NT, kPairQ>(a, st);
  }
  return launch_mod<D, NT, kPlain>(a, st);
}

}  // namespace

void kv4_mma_plan(const Kv8Geom& g, int32_t batch, int32_t n_tokens, int32_t max_new, int32_t max_kv, int32_t num_sms,
                  int32_t* tiles, int32_t* chunk, int32_t* splits) {
  const int32_t R = kv8_mma_rows(g, max_new), G = g.n_q_heads / g.n_kv_heads;
  const int64_t n = static_cast<int64_t>(max_new) * G <= R ? batch : static_cast<int64_t>(n_tokens) * G / R + batch;
  const int64_t units = n * g.n_kv_heads;
  // Chunks of 128 rows (a step a warp) and more: the size with the least of the blocks' rows over the places for
  // blocks, a block's fixed work counted as 512 more, half a block for the uneven end, and 10 for each part to
  // merge. Measured, chunks of 1024, 2048, 4096 and 8192, and the one taken: 32 x 32768 rows, 64 query heads, 301, 258, 240, 241 and
  // 250 us (4736 rows); 64 x 256 to 8192 rows 110, 94, 98, 103 and 98 (2816); one of 130001 64, 55, 61, 60 and 57 (2176); 24 of
  // 1000 to 9000 with 2 to 5 new ones, 16-row tiles, 107, 90, 88, 112 and 88.
  const int64_t slots = static_cast<int64_t>(num_sms) * (R == 8 ? kBlocks : 2);
  int64_t c = kChunkMin;
  double best = 1e30;
  for (int64_t rows = kChunkMin; rows <= kChunkMax; rows += kChunkMin) {
    const double n_split = static_cast<double>((max_kv + rows - 1) / rows), block = static_cast<double>(rows) + 512.0;
    const double end = static_cast<double>(units) * n_split * block / static_cast<double>(slots) + 0.5 * block + 10.0 * n_split;
    if (end < best) {
      best = end;
      c = rows;
    }
  }
  int64_t s = (max_kv + c - 1) / c;
  if (units > kKv8Counters || s > 65535) {
    c = (static_cast<int64_t>(max_kv) + kChunkMin - 1) / kChunkMin * kChunkMin;
    s = 1;
  }
  *tiles = static_cast<int32_t>(n);
  *chunk = static_cast<int32_t>(c);
  *splits = static_cast<int32_t>(s);
}

cudaError_t launch_kv4_mma(const Kv8AttnArgs& a, cudaStream_t st) {
  const bool eight = kv8_mma_rows(a.g, a.max_new) == 8;
  if (a.g.head_dim == 64) return eight ? launch_prec<64, 1>(a, st) : launch_prec<64, 2>(a, st);
  return eight ? launch_prec<128, 1>(a, st) : launch_prec<128, 2>(a, st);
}

}  // namespace aihost
