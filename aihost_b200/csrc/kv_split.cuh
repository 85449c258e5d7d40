// kv_split.cuh — what the split-cache attention kernels over the 8-bit and the 4-bit paged cache share: the
// products' forms, the query rows as operands, and the merge of a block's warps and of a tile's chunks.
#pragma once

#include "common.cuh"
#include "kv8.h"
#include "kv8_tile.cuh"
#include "rows.cuh"

namespace aihost {

constexpr int kWarps = 4;         // of a block
constexpr int kSub = 16;          // cache rows of one MMA, and of the smallest page
constexpr int kStep = 2 * kSub;   // cache rows of a step; a block's warps take steps in turn
constexpr int kChunkMin = kWarps * kStep;

// What the products take. fp16 tensors: an unrotated q is exact in fp16, a rotated one (in fp32) enters
// as a pair, its fp16 and the fp16 of what that leaves, both of one half of it, since turning (x, y) may
// pass fp16's range; P is rounded to fp16 once, as the output is. fp32
// tensors: q and P as pairs, 22 bits; a row of q is brought to 2^13 first by a power of two, which the
// scores take back, or rows beyond fp16's range would be infinite and small ones lose the pair's
// lower half. The cache's integers are exact in fp16; sums are fp32.
enum { kPlain = 0, kPairQ = 1, kPairQP = 2 };

// The maximum may lag by 2^kSlack before O is rescaled. A pair's rest has fp16's smallest step, so pairs keep the
// maximum up to date and use the whole range.
template <int PREC>
constexpr float kSlack = PREC == kPairQP ? 0.0f : 8.0f;
template <int PREC>
constexpr float kQUnit = PREC == kPairQ ? 0.5f : 1.0f;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// f(scores of two columns, block of 16 rows, N tile, first of the fragment's two) for a step's scores, in packed fp32.
template <int NT, typename F>
__device__ __forceinline__ void of_pairs(float (&s)[2][NT][4], F&& f) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float2 x = f(make_float2(s[u][nt][e], s[u][nt][e + 1]), u, nt, e);
        s[u][nt][e] = x.x, s[u][nt][e + 1] = x.y;
      }
}

// Cap (the scores come in units of it, far the largest of the lane's) and distance bias, into log2 units.
template <int NT>
__device__ __forceinline__ void modify_scores(const Kv8AttnArgs& a, bool capped, float cap2, float far, int32_t k, int g,
                                              const float (&c_slope)[NT][2], const float (&c_pos)[NT][2],
                                              float (&s)[2][NT][4]) {
  if (capped) {  // without exponentials where the warp has small ones only
    if (__any_sync(0xffffffffu, far > kTanhSmall))
      of_pairs<NT>(s, [&](float2 x, int, int, int) { return make_float2(cap2 * tanh_of(x.x), cap2 * tanh_of(x.y)); });
    else
      of_pairs<NT>(s, [&](float2 x, int, int, int) {
        const float2 y = fmul2(x, x);
        float2 p = ffma2(make_float2(kTanh3, kTanh3), y, make_float2(kTanh2, kTanh2));
        p = ffma2(p, y, make_float2(kTanh1, kTanh1));
        p = ffma2(p, y, make_float2(kTanh0, kTanh0));
        return fmul2(fmul2(x, make_float2(cap2, cap2)), p);
      });
  }
  if (a.alibi_slopes)
    of_pairs<NT>(s, [&](float2 x, int u, int nt, int e) {
      const float row = static_cast<float>(k + u * kSub + g + (e >> 1) * 8);
      return make_float2(fmaf(-c_slope[nt][0], fabsf(c_pos[nt][0] - row), x.x),
                         fmaf(-c_slope[nt][1], fabsf(c_pos[nt][1] - row), x.y));
    });
}

// The tile's query rows, rotated, as B fragments: lane (g, t4) holds row g's elements [t4 * D/4, (t4 + 1) * D/4).
// FOUR: in the order of the 4-bit cache's words, whose products take elements 0, 1, 4, 5 of eight and 2, 3, 6, 7.
template <int D, int NT, int PREC, bool FOUR>
__device__ __forceinline__ void load_q(const Kv8AttnArgs& a, const Tile& tl, int32_t G, int32_t h, int32_t n_rows, int g, int t4,
                                       uint32_t (&qf)[PREC == kPlain ? 1 : 2][NT][D / 16][2], float (&q_unit)[NT][2]) {
  constexpr int KS = D / 16, NQ = PREC == kPlain ? 1 : 2;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    constexpr int E = D / 4;
    float x[E];
    float back = 1.0f;
    const int r = nt * 8 + g;
    const int32_t row = tl.row0 + min(r, n_rows - 1), i = row / G;
    const uint8_t* src = static_cast<const uint8_t*>(a.q) + (tl.start + static_cast<int64_t>(i)) * a.q_token_stride;
    const int64_t el = static_cast<int64_t>(h * G + row % G) * D + t4 * E;
    if (a.q_dtype == AIHOST_F16) {
      const uint4* p = reinterpret_cast<const uint4*>(src + el * 2);
#pragma unroll
      for (int k = 0; k < E / 8; ++k) {
        const uint4 v = p[k];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[m]));
          x[8 * k + 2 * m] = f.x, x[8 * k + 2 * m + 1] = f.y;
        }
      }
    } else {
      const float4* p = reinterpret_cast<const float4*>(src + el * 4);
#pragma unroll
      for (int k = 0; k < E / 4; ++k) {
        const float4 v = p[k];
        x[4 * k] = v.x, x[4 * k + 1] = v.y, x[4 * k + 2] = v.z, x[4 * k + 3] = v.w;
      }
    }
    if constexpr (PREC == kPairQP) {
      float most = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) most = fmaxf(most, fabsf(x[e]));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // biased exponents: e for the row's largest element, from 14 on so that both powers are normal numbers
      const uint32_t e_most = max(__float_as_uint(most) >> 23, 14u);
      const float bring = __uint_as_float((267u - e_most) << 23);
      back = __uint_as_float((e_most - 13u) << 23);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] *= bring;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) q_unit[nt][c] = PREC == kPairQP ? __shfl_sync(0xffffffffu, back, (2 * t4 + c) * 4) : 1.0f;
    if (PREC != kPlain && a.rope_mode != AIHOST_ROPE_NONE) {
      const float pos = static_cast<float>(tl.pos0 + i);
      if (a.rope_mode == AIHOST_ROPE_INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          float sn, cs;
          sincos_near(__fmul_rn(pos, a.freqs.f[(t4 * E + e) >> 1]), &sn, &cs);
          rotate_pair(x[e], x[e + 1], cs * kQUnit<PREC>, sn * kQUnit<PREC>);
        }
      } else {  // pairs D/2 apart: lanes t4 and t4 ^ 2
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float other = __shfl_xor_sync(0xffffffffu, x[e], 2);
          float sn, cs;
          sincos_near(__fmul_rn(pos, a.freqs.f[(t4 & 1) * E + e]), &sn, &cs);
          float x1 = t4 < 2 ? x[e] : other, x2 = t4 < 2 ? other : x[e];
          rotate_pair(x1, x2, cs * kQUnit<PREC>, sn * kQUnit<PREC>);
          x[e] = t4 < 2 ? x1 : x2;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int e0 = FOUR ? 8 * (k >> 1) + 2 * (k & 1) : 4 * k, e1 = FOUR ? e0 + 4 : e0 + 2;
      qf[0][nt][k][0] = pack2(x[e0], x[e0 + 1]);
      qf[0][nt][k][1] = pack2(x[e1], x[e1 + 1]);
      if constexpr (NQ == 2) {
        qf[1][nt][k][0] = pack2_rest(x[e0], x[e0 + 1], qf[0][nt][k][0]);
        qf[1][nt][k][1] = pack2_rest(x[e1], x[e1 + 1], qf[0][nt][k][1]);
      }
    }
  }
}

// The block's result from its warps' parts: o_sh, relative to 2^m, and ml_sh (m, sum), all written. A tile of one chunk
// is stored; else the chunk's part goes to a.part_o and a.part_ml, and the last block to arrive merges the chunks.
template <int D, int NT>
__device__ __forceinline__ void merge_block(const Kv8AttnArgs& a, const Tile& tl, int32_t G, int32_t h, int32_t n_rows,
                                            int32_t split, int32_t n_splits, const float (*o_sh)[NT * 8][D + 4],
                                            const float (*ml_sh)[NT * 8][2], int32_t& last_sh) {
  constexpr int R = NT * 8;
  auto store = [&](int r, int d, float v0, float v1) {
    const int32_t row = tl.row0 + r;
    const int64_t at = ((tl.start + static_cast<int64_t>(row / G)) * a.g.n_q_heads + h * G + row % G) * D + d;
    if (a.out_dtype == AIHOST_F16)
      *reinterpret_cast<__half2*>(static_cast<__half*>(a.out) + at) = __floats2half2_rn(v0, v1);
    else
      *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(v0, v1);
  };
  const int64_t unit = static_cast<int64_t>(blockIdx.x);
  for (int i = threadIdx.x; i < n_rows * (D / 2); i += kWarps * 32) {
    const int r = i / (D / 2), d = i % (D / 2) * 2;
    float mm = kNoMax;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ml_sh[w][r][0]);
    float ll = 0.0f, v0 = 0.0f, v1 = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2_approx(ml_sh[w][r][0] - mm);
      ll += ml_sh[w][r][1] * f;
      v0 += o_sh[w][r][d] * f;
      v1 += o_sh[w][r][d + 1] * f;
    }
    if (n_splits == 1) {
      const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;  // NaN stays NaN
      store(r, d, v0 * inv, v1 * inv);
    } else {
      const int64_t at = (unit * a.max_splits + split) * R + r;
      *reinterpret_cast<float2*>(a.part_o + at * D + d) = make_float2(v0, v1);
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(mm, ll);
    }
  }
  if (n_splits == 1) return;

  // ---- merge the chunks: the last block of this tile and head to arrive
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last_sh = last_to_arrive(a.counters + unit, n_splits);
  __syncthreads();
  if (!last_sh) return;
  __threadfence();
  const int64_t first_part = unit * a.max_splits * R;
  constexpr int kVec = R * (D / 4) / (kWarps * 32);  // float4 of the result per thread
  constexpr int kAtOnce = 8;                         // chunks whose parts are in flight together
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    const int at = v * (kWarps * 32) + threadIdx.x, r = at / (D / 4), d4 = at % (D / 4);
    if (r >= n_rows) continue;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float mm = kNoMax, ll = 0.0f;
    for (int32_t s0 = 0; s0 < n_splits; s0 += kAtOnce) {
      const int64_t p0 = first_part + static_cast<int64_t>(s0) * R + r;
      float2 ml[kAtOnce];
      float4 x[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const bool on = s0 + q < n_splits;
        ml[q] = on ? __ldcg(reinterpret_cast<const float2*>(a.part_ml) + p0 + q * R) : make_float2(kNoMax, 0.0f);
        x[q] = on ? __ldcg(reinterpret_cast<const float4*>(a.part_o) + (p0 + q * R) * (D / 4) + d4)
                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      float top = mm;
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) top = fmaxf(top, ml[q].x);
      const float f0 = ex2_approx(mm - top);
      mm = top;
      ll *= f0;
      acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const float f = ex2_approx(ml[q].x - top);
        ll += ml[q].y * f;
        acc.x += x[q].x * f, acc.y += x[q].y * f, acc.z += x[q].z * f, acc.w += x[q].w * f;
      }
    }
    const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
    store(r, 4 * d4, acc.x * inv, acc.y * inv);
    store(r, 4 * d4 + 2, acc.z * inv, acc.w * inv);
  }
}

}  // namespace aihost
