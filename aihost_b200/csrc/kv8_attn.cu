// kv8_attn.cu — attention of few query rows over the 8-bit paged cache (decode, short prompts).
//
// One block takes R = 8 or 16 query rows (tokens x heads of one KV head, so the cache is read once
// for the whole head group), one KV head and a chunk of the cache rows; its four warps walk 32-row
// steps of the chunk. Per step, with the transposed products that make cache rows the M = 16 of
// mma.sync m16n8k16 and query rows its N = 8:
//   S^T = K Q^T     K's int8 go to fp16 in registers, one fp32 factor per page afterwards
//   online softmax  running maximum per query row, moved only when it grows by more than 2^8
//   O^T += V^T P^T  V likewise exact; P carries the page's scale relative to the chunk's largest, which
//                   the running maximum counts in
// The k order of either product is free, so it is chosen such that every lane takes 16 bytes of a
// cache row at a time and no transpose is needed. Each warp copies its own steps' rows into a ring of
// its own in shared memory (cp.async, a step ahead, chunks swizzled against bank conflicts): no warp
// waits for another in the loop. A lane holds the place and scales of one of the warp's next 32 blocks
// of 16 rows (the smallest page). Warps merge through shared memory, chunks through partials that the
// last block to arrive merges (no block waits for another).
//
// A cache value is used by R query rows, 2 R products a byte, far below what the tensor cores need:
// the bytes bound it, and mma.sync from registers is enough. Measured, head_dim 128, 8 KV heads: 64
// sequences of 256 to 8192 rows 105 us (599 MB, 5.7 TB/s, 87 % of a copy's measured 6.55), 32 of 16384
// with 64 query heads and capped scores 177 us (1.07 GB, 6.1 TB/s, 93 %); under sustained load 112 and
// 197. One sequence of 513 rows takes 6.9 us in a graph, 7.2 to 7.6 called one at a time: table entry, scales,
// rows, partial, counter and merge are dependent trips to L2. Not better: three stages of the ring with two blocks an SM instead
// of two with three (197 against 177 us for the 32 x 16384), rows loaded straight into registers (135
// against 127 for the 64), 16-row steps (127 against 113), prefetch hints on the copies (no change).
#include <type_traits>

#include "common.cuh"
#include "kv8.h"
#include "kv8_tile.cuh"
#include "kv_split.cuh"
#include "rows.cuh"

namespace aihost {
namespace {

constexpr int kStages = 2;        // of the warp's ring
constexpr int kChunkMax = 2048;

// P enters times v scale / (the chunk's largest v scale) * kVUnit, at most 2^15 (the maximum counts that ratio in: v_exp_of):
// inside fp16's range with as much as possible above its smallest step.
template <int PREC>
constexpr float kVUnit = PREC == kPairQP ? 32768.0f : 128.0f;

// Where 16-byte chunk c of a step's row r lies: lanes that load together, 8 chunks of two rows (K) or
// one or two chunks of four rows two apart (V), fall into different banks.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if (D == 128) return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4));
  return static_cast<uint32_t>((r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (r & 6)) << 4));
}

template <int D, int NT>
struct SplitSmem {  // the rings, and over them the merge's O
  static constexpr int kStageBytes = 2 * kStep * D;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kMerge = kWarps * NT * 8 * (D + 4) * 4;
  static constexpr int kBytes = kRing > kMerge ? kRing : kMerge;
};

template <int D, int NT, int PREC, bool MOD>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) kv8_mma_kernel(const __grid_constant__ Kv8AttnArgs a) {
  constexpr int R = NT * 8;
  constexpr int KS = D / 16;       // k steps of S^T = K Q^T
  constexpr int KC = D / 64;       // 16-byte chunks of a K row per lane
  constexpr int MT = D / 16;       // 16-row tiles of O^T
  constexpr int VW = D / 32;       // 32-bit words of a V row per lane
  constexpr int NQ = PREC == kPlain ? 1 : 2;
  extern __shared__ __align__(128) uint8_t ring[];
  float(*const o_sh)[R][D + 4] = reinterpret_cast<float(*)[R][D + 4]>(ring);
  __shared__ float ml_sh[kWarps][R][2];
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
    const int32_t row = split * a.chunk + warp * kStep + (lane >> 1) * (kWarps * kStep) + (lane & 1) * kSub;
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
      const int r = nt * 8 + 2 * t4 + c;
      int32_t pos;
      row_range(a, tl, G, n_rows, r, c_first[nt][c], c_end[nt][c], pos);
      c_pos[nt][c] = static_cast<float>(pos);
      c_slope[nt][c] =
          MOD && a.alibi_slopes ? a.alibi_slopes[h * G + (tl.row0 + min(r, n_rows - 1)) % G] * kLog2e : 0.0f;
    }
  int32_t lo, hi, lo_max, hi_min;
  {
    int32_t first, end, pos;
    row_range(a, tl, G, n_rows, lane & (R - 1), first, end, pos);
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
  // lane j: where block 32 * round + j lies (its offset in either pool; none past the end), its scales
  constexpr int64_t kNowhere = -1;
  auto place_at = [&](int32_t row, int32_t entry, int64_t& ph) -> int64_t {
    ph = page_or_first(entry, a.g.n_pages, stray) * H + h;
    return ((ph << ps) + (row & (a.g.page_rows - 1))) * D;
  };
  auto place_of = [&](int32_t sub, int64_t& ph) -> int64_t {
    const int32_t row = row_of(sub);
    ph = 0;
    return (sub >> 1) >= n_steps || row >= k_end ? kNowhere : place_at(row, table[row >> ps], ph);
  };
  int64_t ph = 0, ph_next = 0, place = kNowhere;
  if (!known) place = place_of(lane, ph);
  else if ((lane >> 1) < n_steps && row_of(lane) < k_end) place = place_at(row_of(lane), entry_early, ph);
  int64_t place_next = n_steps > 16 ? place_of(32 + lane, ph_next) : kNowhere;
  constexpr int kStageBytes = SplitSmem<D, NT>::kStageBytes;
  uint8_t* const my_ring = ring + warp * (kStages * kStageBytes);
  // copies of a 16-row block: chunk j * 32 + lane of its K and V rows each
  constexpr int CR = D / 16;  // chunks per row
  uint32_t to[2];             // the swizzle repeats every 8 rows: two patterns of destinations
#pragma unroll
  for (int j = 0; j < 2; ++j)
    to[j] = smem_u32(my_ring) + chunk_at<D>((j * 32 + lane) / CR, (j * 32 + lane) % CR) - j * 512;
  auto fetch = [&](int32_t i, int32_t round) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int32_t sub = 2 * i + u;
      const int64_t at = __shfl_sync(0xffffffffu, (sub >> 5) == round ? place : place_next, sub & 31);
      if (i < n_steps && at != kNowhere) {
        const uint32_t dst = (i % kStages) * kStageBytes + u * (kSub * D);
        const int8_t *kp = a.k_pool + at + lane * 16, *vp = a.v_pool + at + lane * 16;
#pragma unroll
        for (int j = 0; j < kSub * CR / 32; ++j) {
          copy16(to[j & 1] + dst + j * 512, kp + j * 512);
          copy16(to[j & 1] + dst + kStep * D + j * 512, vp + j * 512);
        }
      }
    }
    copies_commit();
  };
  fetch(0, 0);
  float ks = 0.0f, vs = 0.0f, ve = 0.0f;
  auto scales = [&] {
    ks = vs = 0.0f;
    if (place != kNowhere) {
      ks = __ldg(a.k_scale + ph);
      vs = __ldg(a.v_scale + ph);
    }
  };
  scales();
  // the blocks' largest V scale: P is scaled relative to it (a NaN scale is passed over here and reaches
  // the result through its own page's factor)
  float vmax = fmaxf(vs, 0.0f);
  for (int32_t sub = 32 + lane; sub < 2 * n_steps; sub += 32) {
    int64_t at;
    if (place_of(sub, at) != kNowhere) vmax = fmaxf(vmax, __ldg(a.v_scale + at));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
  const float v_rcp = v_reciprocal(vmax);
  auto relate = [&] {
    vs *= v_rcp;
    ve = v_exp_of(vs);
    vs *= kVUnit<PREC>;
  };
  relate();

  uint32_t qf[NQ][NT][KS][2];
  float q_unit[NT][2];  // what the scores of this lane's two columns take back
  load_q<D, NT, PREC, false>(a, tl, G, h, n_rows, g, t4, qf, q_unit);

  // Where q is fp16, K's bytes can enter as (128 + k) 2^-24, fp16 numbers below the normal ones that take no
  // arithmetic to make, with S starting at -128 sum q. The terms then cancel in fp32: each of the D / 16
  // products is off by at most 2^-23 of 128 |sum of q so far| and of its own 255 sum |q|. So pages enter where all
  // of that is below 2^-12 in the score (in log2 units; P's own rounding is 2^-11), and as k itself where
  // their scale or q is too large for it. Measured, 64 sequences and 32 of 16384 as above:
  // 104.6 and 176.4 us, k itself throughout 106.7 and 179.6. k itself is used where the registers have no
  // room for more: with two tiles of query rows (8 sequences of 8192 rows, 8 new ones each: 90.9, so 92.1)
  // and with a rotated q and a cap or bias (32 sequences of 4000 to 9000 rows: 98.2, so 100.1).
  constexpr bool kOffset = NT == 1 && (PREC == kPlain || (PREC == kPairQ && !MOD));
  constexpr float kTiny = 1.0f / 16777216.0f;
  constexpr float kOffsetMost = 8388608.0f / 4096.0f;  // of a page's factor times q_size
  float s_init[NT][2], q_size = 0.0f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float sum = 0.0f, most = 0.0f, all = 0.0f;
    if (kOffset) {
#pragma unroll
      for (int k = 0; k < KS; ++k) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qf[n][nt][k][e]));
            sum += f.x + f.y;
            if (n == 0) all += fabsf(f.x) + fabsf(f.y);
          }
        most = fmaxf(most, fabsf(sum));
      }
      q_size = fmaxf(q_size, 128.0f * KS * most + 255.0f * all);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);  // row g's
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) s_init[nt][c] = -128.0f * kTiny * __shfl_sync(0xffffffffu, sum, (2 * t4 + c) * 4);
  }
  // four lanes hold a row: at most four times the largest share (bits of numbers >= 0 compare as numbers)
  if (kOffset) q_size = 4.0f * __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(q_size)));

  float o[MT][NT][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = kNoMax;
    l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
  }
  const bool capped = MOD && a.score_cap > 0.0f;
  const float q_scale = a.scale * (1.0f / kQUnit<PREC>), s_unit = capped ? q_scale / a.score_cap : q_scale * kLog2e;
  const float cap2 = a.score_cap * kLog2e;
  // of this lane's next 32 blocks of rows together, so that it is settled once in 16 steps
  bool small = false;
  float k_unit = s_unit;
  auto settle = [&] {
    if (kOffset) {
      small = __all_sync(0xffffffffu, ks * (q_scale * kLog2e) * q_size <= kOffsetMost);
      k_unit = small ? s_unit / kTiny : s_unit;
    }
  };
  settle();

  for (int32_t i = 0, round = 0; i < n_steps; ++i) {
    if (i == 16 * (round + 1)) {
      ++round;
      place = place_next;
      ph = ph_next;
      scales();
      relate();
      settle();
      if (i + 16 < n_steps) place_next = place_of(2 * i + 32 + lane, ph_next);
    }
    fetch(i + 1, round);
    copies_wait<1>();
    __syncwarp();
    const uint8_t* const stage = my_ring + (i % kStages) * kStageBytes;
    const int32_t k = row_of(2 * i);
    // ---- S^T = K Q^T
    float s[2][NT][4], kf[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) kf[u] = __shfl_sync(0xffffffffu, ks, (2 * i + u) & 31) * k_unit;
    auto products = [&](auto with) {
      constexpr bool offset = decltype(with)::value;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint8_t* const kt = stage + u * (kSub * D);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][nt][e] = offset ? s_init[nt][e & 1] : 0.0f;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const uint4 r0 = *reinterpret_cast<const uint4*>(kt + chunk_at<D>(g, KC * t4 + c));
          const uint4 r1 = *reinterpret_cast<const uint4*>(kt + chunk_at<D>(g + 8, KC * t4 + c));
          const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t u0 = w0[j] ^ 0x80808080u, u1 = w1[j] ^ 0x80808080u;
            uint32_t a0, a1, a2, a3;
            if constexpr (offset) {
              a0 = __byte_perm(u0, 0, 0x4140), a1 = __byte_perm(u1, 0, 0x4140);
              a2 = __byte_perm(u0, 0, 0x4342), a3 = __byte_perm(u1, 0, 0x4342);
            } else {
              a0 = half2_of(u0, 0x4140), a1 = half2_of(u1, 0x4140);
              a2 = half2_of(u0, 0x4342), a3 = half2_of(u1, 0x4342);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int n = 0; n < NQ; ++n)
                mma16816(s[u][nt], a0, a1, a2, a3, qf[n][nt][4 * c + j][0], qf[n][nt][4 * c + j][1]);
          }
        }
      }
    };
    if (kOffset && small) products(std::true_type());
    else products(std::false_type());
    // ---- scores (log2 units), masks, running maximum
    const bool edge = k < lo_max || k + kStep > hi_min;
    bool grow = false;
    const float ve0 = __shfl_sync(0xffffffffu, ve, (2 * i) & 31), ve1 = __shfl_sync(0xffffffffu, ve, (2 * i + 1) & 31);
    auto most_of = [&](int nt, int c) {
      return fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]) + ve0, fmaxf(s[1][nt][c], s[1][nt][c + 2]) + ve1);
    };
    float far = 0.0f;  // the largest of the lane's scores, in units of the cap
    of_pairs<NT>(s, [&](float2 x, int u, int nt, int) {
      float2 f = make_float2(kf[u], kf[u]);
      if (PREC == kPairQP) f = fmul2(f, make_float2(q_unit[nt][0], q_unit[nt][1]));
      x = fmul2(x, f);
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
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        grow |= most_of(nt, c) > m[nt][c] + kSlack<PREC>;
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = most_of(nt, c);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float m_new = fmaxf(m[nt][c], mx), f = ex2_approx(m[nt][c] - m_new);
          m[nt][c] = m_new;
          l[nt][c] *= f;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            o[t][nt][c] *= f;
            o[t][nt][c + 2] *= f;
          }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // ---- P and its fragments
      const float vf = __shfl_sync(0xffffffffu, vs, (2 * i + u) & 31);
      uint32_t pf[PREC == kPairQP ? 2 : 1][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float2 x = fadd2(make_float2(s[u][nt][e], s[u][nt][e + 1]), make_float2(-m[nt][0], -m[nt][1]));
          const float2 v = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          const float2 sum = fadd2(make_float2(l[nt][0], l[nt][1]), v), pv = fmul2(v, make_float2(vf, vf));
          l[nt][0] = sum.x, l[nt][1] = sum.y;
          p[e] = pv.x, p[e + 1] = pv.y;
        }
        if (edge) {  // a hidden row adds nothing even where its page's scale is NaN
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (s[u][nt][e] == -INFINITY) p[e] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t hi2 = pack2(p[2 * c], p[2 * c + 1]);
          pf[0][nt][c] = movmatrix_t(hi2);
          if constexpr (PREC == kPairQP) pf[1][nt][c] = movmatrix_t(pack2_rest(p[2 * c], p[2 * c + 1], hi2));
        }
      }
      // ---- O^T += V^T P^T
      const uint8_t* const vt = stage + kStep * D + u * (kSub * D);
      uint32_t vw[4][VW];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 2 * t4 + (r & 1) + (r >> 1) * 8;
        if constexpr (VW == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(vt + chunk_at<D>(row, g));
          vw[r][0] = v.x, vw[r][1] = v.y, vw[r][2] = v.z, vw[r][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(vt + chunk_at<D>(row, g >> 1) + (g & 1) * 8);
          vw[r][0] = v.x, vw[r][1] = v.y;
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const uint32_t w0 = vw[0][w] ^ 0x80808080u, w1 = vw[1][w] ^ 0x80808080u;
        const uint32_t w2 = vw[2][w] ^ 0x80808080u, w3 = vw[3][w] ^ 0x80808080u;
        const uint32_t x0 = __byte_perm(w0, w1, 0x5140), x1 = __byte_perm(w0, w1, 0x7362);
        const uint32_t y0 = __byte_perm(w2, w3, 0x5140), y1 = __byte_perm(w2, w3, 0x7362);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t x = t ? x1 : x0, y = t ? y1 : y0;
          const uint32_t a0 = half2_of(x, 0x4140), a1 = half2_of(x, 0x4342);
          const uint32_t a2 = half2_of(y, 0x4140), a3 = half2_of(y, 0x4342);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(o[2 * w + t][nt], a0, a1, a2, a3, pf[0][nt][0], pf[0][nt][1]);
            if constexpr (PREC == kPairQP) mma16816(o[2 * w + t][nt], a0, a1, a2, a3, pf[1][nt][0], pf[1][nt][1]);
          }
        }
      }
    }
    __syncwarp();  // every lane has its rows: the slot may be filled again
  }
  if (stray) atomicOr(a.status, kStatusBadIndex);

  copies_wait<0>();
  __syncthreads();  // the rings become the merge's space
  // ---- merge the four warps: lane (g, t4) holds elements [g * D/8, (g + 1) * D/8) of rows 2 t4 and 2 t4 + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
      const int r = nt * 8 + 2 * t4 + c;
      if (g == 0) ml_sh[warp][r][0] = m[nt][c], ml_sh[warp][r][1] = l[nt][c];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        o_sh[warp][r][g * (D / 8) + 2 * i] = o[i][nt][c] * (1.0f / kVUnit<PREC>) * vmax;  // each warp's own
        o_sh[warp][r][g * (D / 8) + 2 * i + 1] = o[i][nt][c + 2] * (1.0f / kVUnit<PREC>) * vmax;
      }
    }
  __syncthreads();
  merge_block<D, NT>(a, tl, G, h, n_rows, split, n_splits, o_sh, ml_sh, last_sh);
}

template <int D, int NT, int PREC, bool MOD>
cudaError_t launch_one(const Kv8AttnArgs& a, cudaStream_t st) {
  constexpr int kBytes = SplitSmem<D, NT>::kBytes;
  auto kern = kv8_mma_kernel<D, NT, PREC, MOD>;
  if (kBytes > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) return e;
  }
  return launch_dependent(kern, dim3(static_cast<unsigned>(a.tiles) * a.g.n_kv_heads, a.max_splits), kWarps * 32, kBytes, st, a);
}

template <int D, int NT, int PREC>
cudaError_t launch_mod(const Kv8AttnArgs& a, cudaStream_t st) {
  return a.score_cap > 0.0f || a.alibi_slopes ? launch_one<D, NT, PREC, true>(a, st) : launch_one<D, NT, PREC, false>(a, st);
}

template <int D, int NT>
cudaError_t launch_prec(const Kv8AttnArgs& a, cudaStream_t st) {
  if (a.q_dtype == AIHOST_F32) return launch_mod<D, NT, kPairQP>(a, st);
  if (a.rope_mode != AIHOST_ROPE_NONE) return launch_mod<D, NT, kPairQ>(a, st);
  return launch_mod<D, NT, kPlain>(a, st);
}

}  // namespace

int32_t kv8_mma_rows(const Kv8Geom& g, int32_t max_new) {
  return static_cast<int64_t>(max_new) * (g.n_q_heads / g.n_kv_heads) <= 8 ? 8 : 16;
}

void kv8_mma_plan(const Kv8Geom& g, int32_t batch, int32_t n_tokens, int32_t max_new, int32_t max_kv, int32_t num_sms,
                  int32_t* tiles, int32_t* chunk, int32_t* splits) {
  const int32_t R = kv8_mma_rows(g, max_new), G = g.n_q_heads / g.n_kv_heads;
  const int64_t n = static_cast<int64_t>(max_new) * G <= R ? batch : static_cast<int64_t>(n_tokens) * G / R + batch;
  const int64_t units = n * g.n_kv_heads;
  // Chunks of 128 rows (a step a warp) to 2048: the size with the least waves of blocks (three or two on
  // an SM) times a block's rows, its fixed work counted as 256 more, and 5 for each part to merge. (Measured
  // for 32 x 16384 rows: chunks of 512 take 230 us, of 1024 193, of 1920 184; for one sequence of 513 rows
  // chunks of 128 to 512 are alike.)
  const int64_t slots = static_cast<int64_t>(num_sms) * (R == 8 ? 3 : 2);
  int64_t c = kChunkMin, best = INT64_MAX;
  for (int64_t rows = kChunkMin; rows <= kChunkMax; rows += kChunkMin) {
    const int64_t n_split = (max_kv + rows - 1) / rows;
    const int64_t cost = (units * n_split + slots - 1) / slots * (rows + 256) + 5 * n_split;
    if (cost <= best) {
      best = cost;
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

cudaError_t launch_kv8_mma(const Kv8AttnArgs& a, cudaStream_t st) {
  const bool eight = kv8_mma_rows(a.g, a.max_new) == 8;
  if (a.g.head_dim == 64) return eight ? launch_prec<64, 1>(a, st) : launch_prec<64, 2>(a, st);
  return eight ? launch_prec<128, 1>(a, st) : launch_prec<128, 2>(a, st);
}

}  // namespace aihost
