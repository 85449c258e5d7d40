// kv8_tile.cuh — where a tile of query rows of the ragged batch lies, and small pieces that the
// kernels over the 8-bit cache share.
#pragma once

#include "common.cuh"
#include "kv8.h"

namespace aihost {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -3.402823466e38f;  // the lowest number: no score is below it but a hidden one's -infinity

// A KV head's query rows of sequence b are its tokens' heads, token by token: row = token * G + head
// in the group. Tiles of R rows of sequence b start at floor(row_start[b] * G / R) + b: room for every
// tile whatever the lengths, so the grid needs only host-known bounds and each block finds its
// sequence by itself. (One tile per sequence where max_new * G <= R.)
struct Tile {
  int32_t b, n_new, start, row0, kv_len, pos0;  // pos0: cache row of the sequence's first new token
  bool ok;
};

// The tile's place; ok is false for a tile without rows and for one whose lengths are out of bounds
// (which sets the status). Called by whole warps.
__device__ __forceinline__ Tile find_tile(const Kv8AttnArgs& a, int64_t tile, int32_t G, int32_t R, int lane) {
  Tile t;
  t.ok = false;
  t.row0 = 0;
  const bool one = static_cast<int64_t>(a.max_new) * G <= R;
  if (one) {
    t.b = static_cast<int32_t>(tile);
  } else {
    int32_t lo = 0, n = a.batch;
    while (n > 1) {  // 32 candidates at a time
      const int32_t step = (n + 31) / 32, i = lo + lane * step;
      const bool at = i < lo + n && static_cast<int64_t>(a.row_start[i]) * G / R + i <= tile;
      const int32_t c = __popc(__ballot_sync(0xffffffffu, at));
      const int32_t skip = (c > 0 ? c - 1 : 0) * step;
      lo += skip;
      n = min(step, n - skip);
    }
    t.b = lo;
  }
  t.start = a.row_start[t.b];
  t.n_new = a.row_start[t.b + 1] - t.start;
  t.kv_len = a.kv_len[t.b];
  t.pos0 = t.kv_len - t.n_new;
  if (t.n_new == 0) return t;
  if (t.n_new < 0 || t.start < 0 || static_cast<int64_t>(t.start) + t.n_new > a.n_tokens || t.n_new > a.max_new ||
      t.pos0 < 0 || t.kv_len > a.max_kv || t.kv_len > static_cast<int64_t>(a.g.max_pages) << a.g.page_shift) {
    if (lane == 0) atomicOr(a.status, kStatusBadIndex);
    return t;
  }
  if (!one) {
    const int64_t k = tile - (static_cast<int64_t>(t.start) * G / R + t.b);
    if (k < 0 || k * R >= static_cast<int64_t>(t.n_new) * G) return t;
    t.row0 = static_cast<int32_t>(k * R);
  }
  t.ok = true;
  return t;
}

// The cache rows [first, end) that the tile's row r sees, and its position. r is clamped to n_rows - 1.
__device__ __forceinline__ void row_range(const Kv8AttnArgs& a, const Tile& t, int32_t G, int32_t n_rows, int r,
                                          int32_t& first, int32_t& end, int32_t& pos) {
  const int32_t i = (t.row0 + min(r, n_rows - 1)) / G;
  pos = t.pos0 + i;
  end = pos + 1;
  if (a.prefix_len) end = max(end, min(a.prefix_len[t.b], t.kv_len));
  first = a.row_first ? max(a.row_first[t.start + i], 0) : 0;
}

// Bytes 0,1 (sel 0x4140) or 2,3 (0x4342) of `u` as exact fp16 integers: u holds value + 128, the
// byte becomes the mantissa of 1024 + u, and 1152 comes off again.
__device__ __forceinline__ uint32_t half2_of(uint32_t u, uint32_t sel) {
  const uint32_t h = __byte_perm(u, 0x64646464u, sel);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The rest of (lo, hi) after the fp16 pair `h`, in fp16.
__device__ __forceinline__ uint32_t pack2_rest(float lo, float hi, uint32_t h) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pack2(lo - f.x, hi - f.y);
}

// Packed fp32 pairs: one instruction for two.
__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 ra, rb, rc, rd;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %5};\n mov.b64 rc, {%6, %7};\n"
      " fma.rn.f32x2 rd, ra, rb, rc;\n mov.b64 {%0, %1}, rd;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 ra, rb, rd;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %5};\n add.rn.f32x2 rd, ra, rb;\n"
      " mov.b64 {%0, %1}, rd;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 ra, rb, rd;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %5};\n mul.rn.f32x2 rd, ra, rb;\n"
      " mov.b64 {%0, %1}, rd;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// tanh for the score cap, whose error is to go by the score and not by the cap: up to kTanhSmall x P(x^2), P of
// degree 3 (our weighted least-squares fit on [0, 0.35], 4e-8 off, 1.8e-7 of x near 0); beyond,
// 1 - 2 / (1 + e^2x), absolute error ~1e-7.
constexpr float kTanhSmall = 0.35f;
constexpr float kTanh0 = 0.9999998211860657f, kTanh1 = -0.3333165645599365f, kTanh2 = 0.13283322751522064f,
                kTanh3 = -0.048376914113759995f;
__device__ __forceinline__ float tanh_small(float x) {
  const float y = x * x;
  return x * fmaf(fmaf(fmaf(kTanh3, y, kTanh2), y, kTanh1), y, kTanh0);
}
__device__ __forceinline__ float tanh_far(float x) {
  const float e = ex2_approx(x * (2.0f * kLog2e));
  return 1.0f - __fdividef(2.0f, 1.0f + e);
}
__device__ __forceinline__ float tanh_of(float x) { return fabsf(x) <= kTanhSmall ? tanh_small(x) : tanh_far(x); }

// sin and cos to 1.1e-7 for |angle| <= 1e6 (beyond, the library's): Cody-Waite reduction by pi/2 in three
// parts (W. J. Cody and W. Waite, Software Manual for the Elementary Functions, 1980), each step one
// fma, then odd and even polynomials, our weighted least-squares fits on [-pi/4, pi/4].
__device__ __noinline__ inline float2 sincos_far(float a) {
  float2 v;
  sincosf(a, &v.x, &v.y);
  return v;
}

__device__ __forceinline__ void sincos_near(float a, float* s, float* c) {
  if (fabsf(a) > 1e6f) {
    const float2 v = sincos_far(a);
    *s = v.x;
    *c = v.y;
    return;
  }
  const float k = rintf(a * 0.636619772367581343f);
  float r = fmaf(-k, 1.5707963705062866f, a);
  r = fmaf(-k, -4.371138828673793e-08f, r);
  r = fmaf(-k, -1.7151245100058819e-15f, r);
  const float y = r * r;
  const float ps = fmaf(fmaf(-0.00019517235341481864f, y, 0.008332177996635437f), y, -0.16666655242443085f);
  const float pc = fmaf(fmaf(2.4438379114144482e-05f, y, -0.0013887366512790322f), y, 0.04166664555668831f);
  const float sn = fmaf(r * y, ps, r), cs = fmaf(pc * y, y, fmaf(-0.5f, y, 1.0f));
  const int q = static_cast<int>(k);
  const float u = q & 1 ? cs : sn, v = q & 1 ? sn : cs;
  *s = q & 2 ? -u : u;
  *c = (q + 1) & 2 ? -v : v;
}

// How a page's V scale enters. P carries it relative to the largest of the chunk, times kVUnit, so that it stays
// in fp16's range. But a row may see only pages far below the largest (other rows' documents set it), or
// give the pages near it next to no weight. So a row's running maximum is that of score + v_exp, with
// v_exp = log2 of the relative scale: then the row's own largest weight times scale comes to about kVUnit,
// whichever page it lies on, and what is rounded off is small beside that. exp2(score - maximum) may be up to
// 2^90 times what it were with the largest score there; its sum and the merges are fp32.
__device__ __forceinline__ float v_exp_of(float relative) {
  return fmaxf(__log2f(fabsf(relative)), -90.0f);  // pages below 2^-90 of the largest count as that: sums stay below 2^127
}
// 1 / the chunk's largest V scale; 0 where that is 0 or the quotient infinite (the append stores zeros there).
__device__ __forceinline__ float v_reciprocal(float top) { return top > 2.94e-39f ? 1.0f / top : 0.0f; }

// Launch that may begin before the kernel ahead of it on the stream has ended: every kernel launched so
// calls griddep_wait() before it touches memory (the kernel ahead is then complete and visible), and
// griddep_launch_dependents() at its own start, so that the next one's set-up overlaps its work.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Whether this is the last of n arrivals, by one thread of each block after its own writes and a fence.
// The counter wraps to zero with the last, ready for the next launch (and for a replayed one). No block
// waits for another.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, int32_t n) {
  return atomicInc(counter, static_cast<uint32_t>(n - 1)) == static_cast<uint32_t>(n - 1);
}

// Page id of a table entry; one outside the pool becomes page 0 and sets `stray`.
__device__ __forceinline__ int64_t page_or_first(int32_t p, int32_t n_pages, bool& stray) {
  if (p >= 0 && p < n_pages) return p;
  stray = true;
  return 0;
}

}  // namespace aihost
