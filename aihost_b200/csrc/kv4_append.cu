// kv4_append.cu — new K and V rows into the 4-bit paged cache, and rows of it back out.
//
// A row x of one head (K rotated first) is stored by itself, in fp32:
//   low  = fp16(min x)       step = max(fp16((max x - low) / 15), 2^-24)
//   code = min(max(rint((x - low) / step), 0), 15)
// with 1 / 15 and 1 / step rounded first, every operation rounded once and the rotation's cosines and sines the fp32
// numbers nearest to the true ones: the codes are defined to the bit, and no older row is ever touched.
// A row with a NaN or an infinity in it, or whose low or step passes fp16's range, gets NaN for both.
// A row needs nothing of another, so a warp takes a token's heads two (D = 128) or four at a time, a lane eight elements, and the
// bytes bound it where there are many. Measured with the two reads of what was written, 8 heads x 128: 6.7 K prompt
// rows of 4 sequences 25.6 us (62 MB in and out, 2.4 TB/s: three dependent kernels of 20 to 40 MB each), 64 single tokens
// 10.4 us (three launches and their enqueue). The angles' sines and cosines in fp64 cost a token about 45 instructions
// of a warp on a pipe that is otherwise idle, and make the codes the same wherever they are worked out.
#include "common.cuh"
#include "kv8.h"
#include "kv8_tile.cuh"
#include "rows.cuh"

namespace aihost {
namespace {

constexpr int kWarpsHere = 8;
constexpr int kE = 8;  // elements of a row per lane: one word of codes

__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// sin and cos of an fp32 angle, in fp64 and rounded once: reduction by pi / 2 in two parts (W. J. Cody and W. Waite,
// Software Manual for the Elementary Functions, 1980), each one fma, then the Taylor series to x^15 and x^14 (2e-15 off
// at pi / 4).
__device__ __forceinline__ void sincos_rounded(float angle, float* s, float* c) {
  const double a = static_cast<double>(angle), k = rint(a * 0.63661977236758134308);
  double r = fma(-k, 1.57079632679489655800, a);
  r = fma(-k, 6.12323399573676603587e-17, r);
  const double y = r * r;
  double ps = fma(y, -1.0 / 1307674368000.0, 1.0 / 6227020800.0), pc = fma(y, -1.0 / 87178291200.0, 1.0 / 479001600.0);
  ps = fma(y, ps, -1.0 / 39916800.0), pc = fma(y, pc, -1.0 / 3628800.0);
  ps = fma(y, ps, 1.0 / 362880.0), pc = fma(y, pc, 1.0 / 40320.0);
  ps = fma(y, ps, -1.0 / 5040.0), pc = fma(y, pc, -1.0 / 720.0);
  ps = fma(y, ps, 1.0 / 120.0), pc = fma(y, pc, 1.0 / 24.0);
  ps = fma(y, ps, -1.0 / 6.0), pc = fma(y, pc, -0.5);
  const float sn = static_cast<float>(fma(r * y, ps, r)), cs = static_cast<float>(fma(y, pc, 1.0));
  const int q = static_cast<int>(static_cast<long long>(k) & 3);
  const float u = q & 1 ? cs : sn, v = q & 1 ? sn : cs;
  *s = q & 2 ? -u : u;
  *c = (q + 1) & 2 ? -v : v;
}

// A lane's eight elements of a row: 8 in_row .. + 8, or, where pairs lie D/2 apart, 4 in_row .. + 4 of either half.
template <bool HALVES, int D>
__device__ __forceinline__ void load_row(const float* row, int in_row, uint4 (&v)[2]) {
  const float* p = row + in_row * (HALVES ? 4 : 8);
  v[0] = __ldg(reinterpret_cast<const uint4*>(p));
  v[1] = __ldg(reinterpret_cast<const uint4*>(p + (HALVES ? D / 2 : 4)));
}
template <bool HALVES, int D>
__device__ __forceinline__ void load_row(const __half* row, int in_row, uint4 (&v)[1]) {
  if constexpr (HALVES) {
    const uint2 a = __ldg(reinterpret_cast<const uint2*>(row + in_row * 4)), b = __ldg(reinterpret_cast<const uint2*>(row + D / 2 + in_row * 4));
    v[0] = make_uint4(a.x, a.y, b.x, b.y);
  } else {
    v[0] = __ldg(reinterpret_cast<const uint4*>(row + in_row * 8));
  }
}
__device__ __forceinline__ void as_floats(const uint4 (&v)[2], float (&x)[kE]) {
  const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
}
__device__ __forceinline__ void as_floats(const uint4 (&v)[1], float (&x)[kE]) {
  const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    x[2 * k] = f.x, x[2 * k + 1] = f.y;
  }
}

// A warp takes one token's NI * RP heads of K and of V, RP = 32 / LPR rows at a time, D / 8 = LPR lanes to a row. A
// lane's elements hold the pairs 4 in_row .. + 4 of the rotation either way, so the warp works out its token's cosines
// and sines once, each of the RP lanes of a place a share of the four.
template <int D, int NI, typename T, int ROPE>
__global__ void __launch_bounds__(kWarpsHere * 32) kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a, int32_t groups) {
  constexpr int LPR = D / kE, RP = 32 / LPR, NV = sizeof(T) / 2;
  constexpr bool kHalves = ROPE == AIHOST_ROPE_NEOX;
  __shared__ float freq[64];
  const int lane = threadIdx.x & 31, in_row = lane % LPR, sub = lane / LPR;
  const int32_t H = a.g.n_kv_heads;
  if (ROPE != AIHOST_ROPE_NONE) {  // a parameter indexed by lane costs a turn per distinct index
    if (threadIdx.x < D / 2) freq[threadIdx.x] = a.freqs.f[threadIdx.x];
    __syncthreads();
  }
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarpsHere + (threadIdx.x >> 5);
  const int32_t t = static_cast<int32_t>(unit / groups), h0 = static_cast<int32_t>(unit - static_cast<int64_t>(t) * groups) * (NI * RP);
  griddep_wait();
  griddep_launch_dependents();
  if (t >= a.n_tokens) return;
  const int64_t slot = a.slots[t];
  uint4 raw[2][NI][NV] = {};
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int32_t h = h0 + i * RP + sub;
    if (h < H) {
      const int64_t off = t * a.token_stride + static_cast<int64_t>(h) * D * static_cast<int64_t>(sizeof(T));
      load_row<kHalves, D>(reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.k_new) + off), in_row, raw[0][i]);
      load_row<kHalves, D>(reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.v_new) + off), in_row, raw[1][i]);
    }
  }
  if (slot < 0 || slot >= (static_cast<int64_t>(a.g.n_pages) << a.g.page_shift)) {
    if (slot != -1 && lane == 0) atomicOr(a.status, kStatusBadIndex);
    return;
  }
  float cs[4], sn[4];
  if constexpr (ROPE != AIHOST_ROPE_NONE) {
    const float pos = static_cast<float>(a.positions[t]);
    constexpr int kOwn = 4 / RP;  // pairs that this lane works out
    float c[kOwn], s[kOwn];
#pragma unroll
    for (int e = 0; e < kOwn; ++e) sincos_rounded(__fmul_rn(pos, freq[in_row * 4 + sub * kOwn + e]), &s[e], &c[e]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cs[e] = __shfl_sync(0xffffffffu, c[e % kOwn], e / kOwn * LPR + in_row);
      sn[e] = __shfl_sync(0xffffffffu, s[e % kOwn], e / kOwn * LPR + in_row);
    }
  }
  const int64_t row0 = ((slot >> a.g.page_shift) * H << a.g.page_shift) + (slot & (a.g.page_rows - 1));
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int32_t h = h0 + i * RP + sub;
    const int64_t row = row0 + (static_cast<int64_t>(h) << a.g.page_shift);
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float x[kE];
      as_floats(raw[v][i], x);
      if (ROPE != AIHOST_ROPE_NONE && v == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (kHalves) rotate_pair(x[e], x[e + 4], cs[e], sn[e]);
          else rotate_pair(x[2 * e], x[2 * e + 1], cs[e], sn[e]);
        }
      }
      float lo = x[0], hi = x[0];
#pragma unroll
      for (int e = 1; e < kE; ++e) lo = min_nan(lo, x[e]), hi = max_nan(hi, x[e]);
#pragma unroll
      for (int d = 1; d < LPR; d <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
      }
      __half low = __float2half_rn(lo);
      const float low32 = __half2float(low);
      __half step = __float2half_rn(__fmul_rn(__fsub_rn(hi, low32), 1.0f / 15.0f));
      float step32 = fmaxf(__half2float(step), 5.9604644775390625e-8f);
      step = __float2half_rn(step32);
      if (!(hi < INFINITY && fabsf(low32) < INFINITY && step32 < INFINITY)) {  // the codes of such a row: 0
        low = step = __ushort_as_half(0x7fff);
        step32 = INFINITY;
      }
      const float inv = __frcp_rn(step32);
      uint32_t q[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float y = fminf(fmaxf(__fmul_rn(__fsub_rn(x[e], low32), inv), 0.0f), 15.0f);
        q[e] = __float_as_uint(__fadd_rn(y, 8388608.0f)) & 15u;  // the nearest integer, in the low bits
      }
      uint32_t word;
      if constexpr (kHalves) {
        // elements 4 in_row .. + 4 of either half: half a word each, the other half with the next lane
        const uint32_t first = q[0] | q[1] << 16 | q[2] << 4 | q[3] << 20, second = q[4] | q[5] << 16 | q[6] << 4 | q[7] << 20;
        const bool odd = in_row & 1;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? first : second, 1);
        word = odd ? other | second << 8 : first | other << 8;
      } else {
        word = q[0] | q[1] << 16 | q[2] << 4 | q[3] << 20 | q[4] << 8 | q[5] << 24 | q[6] << 12 | q[7] << 28;
      }
      const int at_word = kHalves ? (in_row >> 1) + (in_row & 1) * (LPR / 2) : in_row;
      if (h < H) {
        reinterpret_cast<uint32_t*>(v ? a.v_pool : a.k_pool)[row * LPR + at_word] = word;
        if (in_row == 0)
          (v ? a.v_range : a.k_range)[row] = static_cast<uint32_t>(__half_as_ushort(low)) | static_cast<uint32_t>(__half_as_ushort(step)) << 16;
      }
    }
  }
}

// Rows of a pool as the values they stand for: a thread takes one word (eight codes) of kRowsAt rows.
constexpr int kRowsAt = 4;
template <typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4ReadArgs a, uint32_t per_row, uint32_t per_head_shift) {
  const int64_t n_slots = static_cast<int64_t>(a.g.n_pages) << a.g.page_shift;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y) * kRowsAt;
  if (first >= a.n_rows) return;
  int64_t at[kRowsAt];
#pragma unroll
  for (int k = 0; k < kRowsAt; ++k) {
    const int64_t slot = first + k < a.n_rows ? a.slots[first + k] : -1;
    const bool on = slot >= 0 && slot < n_slots;
    if (!on && slot != -1 && threadIdx.x == 0) atomicOr(a.status, kStatusBadIndex);
    at[k] = on ? ((slot >> a.g.page_shift) * a.g.n_kv_heads << a.g.page_shift) + (slot & (a.g.page_rows - 1)) : -1;
  }
  for (uint32_t i = threadIdx.x; i < per_row; i += blockDim.x) {
    const uint32_t h = i >> per_head_shift, c = i - (h << per_head_shift);
    uint32_t w[kRowsAt], r[kRowsAt];
#pragma unroll
    for (int k = 0; k < kRowsAt; ++k) {
      w[k] = r[k] = 0;
      if (at[k] >= 0) {
        const int64_t row = at[k] + (static_cast<int64_t>(h) << a.g.page_shift);
        w[k] = __ldg(reinterpret_cast<const uint32_t*>(a.pool) + (row << per_head_shift) + c);
        r[k] = __ldg(a.range + row);
      }
    }
#pragma unroll
    for (int k = 0; k < kRowsAt; ++k) {
      if (first + k >= a.n_rows) break;
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[k]));
      alignas(16) T o[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e)
        st_from_float(&o[e], fmaf(static_cast<float>((w[k] >> ((e >> 1) * 4 + (e & 1) * 16)) & 15u), f.y, f.x));
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + ((first + k) * per_row + i) * kE);
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(o) / 16); ++j) dst[j] = reinterpret_cast<const uint4*>(o)[j];
    }
  }
}

template <int D, int NI, typename T, int ROPE>
cudaError_t launch_append_n(const Kv4AppendArgs& a, cudaStream_t st) {
  constexpr int kHeadsAt = NI * 32 * kE / D;  // heads of a warp
  const int32_t groups = (a.g.n_kv_heads + kHeadsAt - 1) / kHeadsAt;
  const int64_t blocks = (static_cast<int64_t>(a.n_tokens) * groups + kWarpsHere - 1) / kWarpsHere;
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_dependent(kv4_append_kernel<D, NI, T, ROPE>, static_cast<unsigned>(blocks), kWarpsHere * 32, 0, st, a, groups);
}

template <int D, typename T, int ROPE>
cudaError_t launch_append_r(const Kv4AppendArgs& a, cudaStream_t st) {
  // Few tokens: a warp a pair (four) of heads, for more warps. Many: four times as many, for more loads in flight and a
  // token's cosines for all of them.
  return a.n_tokens < 1024 ? launch_append_n<D, 1, T, ROPE>(a, st) : launch_append_n<D, 4, T, ROPE>(a, st);
}

template <int D, typename T>
cudaError_t launch_append_t(const Kv4AppendArgs& a, cudaStream_t st) {
  if (a.rope_mode == AIHOST_ROPE_NONE) return launch_append_r<D, T, AIHOST_ROPE_NONE>(a, st);
  if (a.rope_mode == AIHOST_ROPE_NEOX) return launch_append_r<D, T, AIHOST_ROPE_NEOX>(a, st);
  return launch_append_r<D, T, AIHOST_ROPE_INTERLEAVED>(a, st);
}

template <int D>
cudaError_t launch_append_d(const Kv4AppendArgs& a, cudaStream_t st) {
  return a.io_dtype == AIHOST_F32 ? launch_append_t<D, float>(a, st) : launch_append_t<D, __half>(a, st);
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4AppendArgs& a, cudaStream_t st) {
  return a.g.head_dim == 64 ? launch_append_d<64>(a, st) : launch_append_d<128>(a, st);
}

cudaError_t launch_kv4_read(const Kv4ReadArgs& a, cudaStream_t st) {
  const uint32_t shift = a.g.head_dim == 64 ? 3 : 4, per_row = static_cast<uint32_t>(a.g.n_kv_heads) << shift;
  uint32_t x = 8;  // threads across a row: as many as it has words, up to the block's
  while (x < per_row && x < 256) x *= 2;
  const dim3 block(x, 256 / x);
  const int64_t at_once = static_cast<int64_t>(block.y) * kRowsAt;
  const unsigned blocks = static_cast<unsigned>((a.n_rows + at_once - 1) / at_once);
  return launch_dependent(a.out_dtype == AIHOST_F16 ? kv4_read_kernel<__half> : kv4_read_kernel<float>, blocks, block, 0, st, a,
                          per_row, shift);
}

}  // namespace aihost
