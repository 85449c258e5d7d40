// kv8_append.cu — new K and V rows into the 8-bit paged cache, and rows of it back out.
//
// For each page and head that gets new rows x (K rotated first), in fp32:
//   had   = the page's scale, or 0 where its row 0 is among them (a page begun anew)
//   scale = max(had, amax|x| / 127)
//   older rows  q <- rint(q * (had / scale))   (only where the scale grew)
//   new rows    q  = rint(x * (1 / scale))
// The work unit is a run: the consecutive tokens whose slots are consecutive rows of one page. A run is
// read once and kept in registers while its maximum comes together, so 2 (fp16) or 4 bytes a value come
// in and 1 goes out.
// Measured with the two reads of what was written, 8 heads x 128: 64 one-token sequences 12.3 us; the three
// dependent kernels take 11.7 in a graph (5 + 2 x 2.8 us and their hand-over), the host's enqueue as long.
// 6.7 K prompt rows of 4 sequences 41.6 us, of which the append 27 (41 MB in and out: 1.5 TB/s where a copy
// reaches 6.55) and the reads 7 each (21 MB: 45 % of a copy's rate; one load in flight a thread, whose
// neighbours store 32 bytes apart). The append issues about 140 warp instructions per row and head
// (conversion, rotation, maximum, scaling, rounding, packing; a token's sine and cosine anew for every two
// heads) in 53 % of the issue slots: a run's load, its maximum across the warps and its store follow one
// another. (One pass over memory for the maximum and another for the rounding: 70 us for the three
// calls.)
#include "common.cuh"
#include "kv8.h"
#include "kv8_tile.cuh"
#include "rows.cuh"

namespace aihost {
namespace {

constexpr int kWarps = 16;
constexpr int kHeads = 2;      // heads of K or V that one block handles
constexpr int kMaxPage = 128;
constexpr uint32_t kInfBits = 0x7f800000u;

// |x| against a running maximum in which a NaN stays.
__device__ __forceinline__ float max_abs(float top, float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(top), "f"(fabsf(x)));
  return y;
}

// N consecutive elements (8, 4 or 2) as floats.
template <int N>
__device__ __forceinline__ void load_some(const float* p, float* x) {
  if constexpr (N == 8) {
    load_some<4>(p, x);
    load_some<4>(p + 4, x + 4);
  } else if constexpr (N == 4) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const float2 v = __ldg(reinterpret_cast<const float2*>(p));
    x[0] = v.x, x[1] = v.y;
  }
}
template <int N>
__device__ __forceinline__ void load_some(const __half* p, float* x) {
  uint32_t w[N / 2];
  if constexpr (N == 8) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 4) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    x[2 * k] = f.x, x[2 * k + 1] = f.y;
  }
}

// Int8 from the low bytes of q: four, then N of them.
__device__ __forceinline__ uint32_t pack_bytes(const uint32_t* q) {
  return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}
template <int N>
__device__ __forceinline__ void store_bytes(int8_t* p, const uint32_t* q) {
  if constexpr (N == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bytes(q), pack_bytes(q + 4));
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint32_t*>(p) = pack_bytes(q);
  } else {
    *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(__byte_perm(q[0], q[1], 0x0040));
  }
}

// Four int8 q -> rint(q * ratio), ratio <= 1 (adding 1.5 * 2^23 rounds to the nearest integer).
__device__ __forceinline__ uint32_t rescale4(uint32_t word, float ratio) {
  uint32_t q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = static_cast<float>(static_cast<int8_t>(word >> (8 * e)));
    q[e] = __float_as_uint(__fadd_rn(__fmul_rn(x, ratio), 12582912.0f));
  }
  return pack_bytes(q);
}

// The runs that start in one window of tokens, for two heads of K or V. The 16 warps split into groups,
// as many as the window starts runs (up to 16), and a group takes a run at a time: all warps on one
// page's rows for prompts, a warp per row for decode. LPR lanes take a row, so a warp RP = 32 / LPR at a
// time, and it keeps ROWS such loads of HEADS heads in registers: 16 warps read a page once, whole,
// before its scale is known (64 rows of 2 heads, or 128 of one), and a token's sine and cosine serve both
// heads. A lane holds E = D / LPR elements of a row: consecutive ones, or (rotation by halves) as many from either half, so that pairs stay in a lane.
template <int D, int LPR, int ROWS, int HEADS, typename T, int ROPE>
__global__ void __launch_bounds__(kWarps * 32, 2) kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a, int32_t window) {
  constexpr int RP = 32 / LPR, E = D / LPR, PART = ROPE == AIHOST_ROPE_NEOX ? E / 2 : E;  // elements a lane, in how large parts
  __shared__ int64_t slot_sh[1 + 2 * kMaxPage];  // the token before the window, the window, a page more
  __shared__ int32_t run_at[kMaxPage];
  __shared__ int32_t run_count;
  __shared__ uint32_t warp_max[HEADS][kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in_row = lane % LPR, sub = lane / LPR;
  const int32_t t0 = static_cast<int32_t>(blockIdx.x) * window;
  const bool is_k = (blockIdx.y & 1) == 0;
  const int32_t P = a.g.page_rows, H = a.g.n_kv_heads, h_begin = static_cast<int32_t>(blockIdx.y >> 1) * kHeads;
  const int64_t n_slots = static_cast<int64_t>(a.g.n_pages) << a.g.page_shift;
  const bool rotate = ROPE != AIHOST_ROPE_NONE && is_k;

  griddep_wait();
  griddep_launch_dependents();
  if (threadIdx.x < 1 + window + P) {
    const int64_t t = static_cast<int64_t>(t0) + threadIdx.x - 1;
    slot_sh[threadIdx.x] = t >= 0 && t < a.n_tokens ? a.slots[t] : -1;
  }
  float freq[E / 2];  // of the lane's pairs: the same ones in either layout
#pragma unroll
  for (int p = 0; p < E / 2; ++p) freq[p] = rotate ? a.freqs.f[in_row * (E / 2) + p] : 0.0f;
  __syncthreads();
  if (warp == 0) {
    int32_t count = 0;
    for (int32_t i0 = 0; i0 < window; i0 += 32) {
      const int32_t i = i0 + lane;
      bool head = false;
      if (i < window) {
        const int64_t s = slot_sh[1 + i];
        if (s < -1 || s >= n_slots) {
          if (blockIdx.y == 0) atomicOr(a.status, kStatusBadIndex);
        } else if (s >= 0) {
          head = (s & (P - 1)) == 0 || slot_sh[i] != s - 1;
        }
      }
      const uint32_t m = __ballot_sync(0xffffffffu, head);
      if (head) run_at[count + __popc(m & ((1u << lane) - 1))] = i;
      count += __popc(m);
    }
    if (lane == 0) run_count = count;
  }
  __syncthreads();

  const int32_t n_runs = run_count;
  const int nw = n_runs <= 1 ? 16 : n_runs == 2 ? 8 : n_runs <= 4 ? 4 : n_runs <= 8 ? 2 : 1;  // warps of a group
  const int group = warp / nw, w = warp % nw;
  auto group_sync = [&] {
    if (nw > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(nw * 32) : "memory");
    else __syncwarp();
  };
  int8_t* const pool = is_k ? a.k_pool : a.v_pool;
  float* const scales = is_k ? a.k_scale : a.v_scale;
  const T* const src = static_cast<const T*>(is_k ? a.k_new : a.v_new) + in_row * PART;
  const int64_t stride = a.token_stride / static_cast<int64_t>(sizeof(T));

  for (int r = group; r < n_runs; r += kWarps / nw) {
    const int32_t at = run_at[r];
    const int32_t t = t0 + at;
    const int64_t slot = slot_sh[1 + at];
    const int64_t page = slot >> a.g.page_shift;
    const int32_t row0 = static_cast<int32_t>(slot & (P - 1));
    // the run's length: tokens t + i at slot + i, up to the page's end (past the last token stands -1)
    const int32_t most = P - row0;
    int32_t n = most;
    for (int32_t i0 = 0; i0 < most; i0 += 32) {
      const uint32_t off = __ballot_sync(0xffffffffu, i0 + lane < most && slot_sh[1 + at + i0 + lane] != slot + i0 + lane);
      if (off) {
        n = i0 + __ffs(off) - 1;
        break;
      }
    }
    const int32_t batch = RP * ROWS * nw, last = (n - 1) / batch * batch;
    for (int32_t h0 = h_begin; h0 < min(H, h_begin + kHeads); h0 += HEADS) {
      float had[HEADS];
#pragma unroll
      for (int j = 0; j < HEADS; ++j) had[j] = row0 == 0 || h0 + j >= H ? 0.0f : scales[page * H + h0 + j];
      float x[ROWS][HEADS][E];
      const T* const from = src + t * stride + h0 * D;
      const bool two = HEADS == 1 || h0 + 1 < H;
      auto load = [&](int32_t first) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int32_t k = first + RP * (i * nw + w) + sub;  // the group's rows first + RP i nw + (0 .. RP nw - 1)
          const T* const row = from + k * stride;
#pragma unroll
          for (int j = 0; j < HEADS; ++j) {
            const bool on = k < n && (j == 0 || two);
#pragma unroll
            for (int e = 0; e < E; e += PART) {
              if (on) {
                load_some<PART>(row + j * D + (e ? D / 2 : 0), &x[i][j][e]);
              } else {
#pragma unroll
                for (int q = 0; q < PART; ++q) x[i][j][e + q] = 0.0f;
              }
            }
          }
        }
        if constexpr (ROPE != AIHOST_ROPE_NONE) {
          if (rotate) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
              const int32_t k = first + RP * (i * nw + w) + sub;
              if (k >= n) continue;
              const float pos = static_cast<float>(a.positions[t + k]);
#pragma unroll
              for (int p = 0; p < E / 2; ++p) {
                float sn, cs;
                sincos_near(__fmul_rn(pos, freq[p]), &sn, &cs);
#pragma unroll
                for (int j = 0; j < HEADS; ++j) {
                  if (ROPE == AIHOST_ROPE_NEOX) rotate_pair(x[i][j][p], x[i][j][p + E / 2], cs, sn);
                  else rotate_pair(x[i][j][2 * p], x[i][j][2 * p + 1], cs, sn);
                }
              }
            }
          }
        }
      };
      // amax, then as bits: infinities and NaN compare above every number
      uint32_t top[HEADS];
      {
        float most_abs[HEADS];
#pragma unroll
        for (int j = 0; j < HEADS; ++j) most_abs[j] = 0.0f;
        for (int32_t first = 0; first < n; first += batch) {
          load(first);
#pragma unroll
          for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int j = 0; j < HEADS; ++j)
#pragma unroll
              for (int e = 0; e < E; ++e) most_abs[j] = max_abs(most_abs[j], x[i][j][e]);
        }
#pragma unroll
        for (int j = 0; j < HEADS; ++j) top[j] = __reduce_max_sync(0xffffffffu, __float_as_uint(most_abs[j]));
      }
      if (nw > 1) {
        if (lane == 0)
#pragma unroll
          for (int j = 0; j < HEADS; ++j) warp_max[j][warp] = top[j];
        group_sync();
#pragma unroll
        for (int j = 0; j < HEADS; ++j) top[j] = __reduce_max_sync(0xffffffffu, warp_max[j][group * nw + lane % nw]);
      }
      float inv[HEADS];
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        inv[j] = 0.0f;
        if (h0 + j >= H) continue;
        const float need =
            top[j] >= kInfBits ? __uint_as_float(0x7fffffffu) : __fmul_rn(__uint_as_float(top[j]), 1.0f / 127.0f);
        const float scale = had[j] != had[j] || need != need ? __uint_as_float(0x7fffffffu) : fmaxf(had[j], need);
        // 0 for a NaN scale (its values do not matter) and where 1 / scale overflows (values below 2^-121)
        const float rcp = scale > 0.0f ? __frcp_rn(scale) : 0.0f;
        inv[j] = rcp < __uint_as_float(kInfBits) ? rcp : 0.0f;
        if (scale > had[j] && row0 > 0) {  // the older rows in the new scale (false for NaN)
          const float ratio = __fdiv_rn(had[j], scale);
          uint8_t* const base = reinterpret_cast<uint8_t*>(pool + ((page * H + h0 + j) << a.g.page_shift) * D);
          const int32_t bytes = row0 * D, step = nw * 512;  // the rows lie together: 16 bytes a lane
          for (int32_t b0 = (w * 32 + lane) * 16; b0 < bytes; b0 += 4 * step) {
            uint4 v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (b0 + q * step < bytes) v[q] = *reinterpret_cast<const uint4*>(base + b0 + q * step);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (b0 + q * step < bytes) {
                v[q] = make_uint4(rescale4(v[q].x, ratio), rescale4(v[q].y, ratio), rescale4(v[q].z, ratio),
                                  rescale4(v[q].w, ratio));
                *reinterpret_cast<uint4*>(base + b0 + q * step) = v[q];
              }
          }
        }
        // every lane and warp of the group has read the scale before the maximum came together
        if (lane == 0 && w == 0) scales[page * H + h0 + j] = scale;
      }
      const int32_t head_bytes = P * D;
      int8_t* const to = pool + (((page * H + h0) << a.g.page_shift) + row0) * D + in_row * PART;
      for (int32_t first = last; first >= 0; first -= batch) {  // backwards: the last rows are still held
        if (first != last) load(first);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int32_t k = first + RP * (i * nw + w) + sub;
          if (k >= n) continue;
          int8_t* const row = to + k * D;
#pragma unroll
          for (int j = 0; j < HEADS; ++j) {
            if (j && !two) continue;
            // |x / scale| <= 127 but for rounding: adding 1.5 * 2^23 rounds it to the nearest integer, in the
            // low bits
            uint32_t q[E];
#pragma unroll
            for (int e = 0; e < E; ++e) q[e] = __float_as_uint(__fadd_rn(__fmul_rn(x[i][j][e], inv[j]), 12582912.0f));
#pragma unroll
            for (int e = 0; e < E; e += PART) store_bytes<PART>(row + j * head_bytes + (e ? D / 2 : 0), &q[e]);
          }
        }
      }
      group_sync();  // warp_max is free again
    }
  }
}

// Rows of a pool as the values they stand for: 16 int8 (one 16-byte load) per thread, the heads' chunks of
// a row side by side.
template <typename T>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8ReadArgs a, uint32_t per_row, uint32_t per_head_shift) {
  const int64_t n_slots = static_cast<int64_t>(a.g.n_pages) << a.g.page_shift;
  griddep_wait();
  griddep_launch_dependents();
  for (int32_t row = blockIdx.x * blockDim.y + threadIdx.y; row < a.n_rows; row += gridDim.x * blockDim.y) {
    const int64_t slot = a.slots[row];
    const bool on = slot >= 0 && slot < n_slots;
    if (!on && slot != -1 && threadIdx.x == 0) atomicOr(a.status, kStatusBadIndex);
    for (uint32_t i = threadIdx.x; i < per_row; i += blockDim.x) {
      const uint32_t h = i >> per_head_shift, c = i - (h << per_head_shift);
      int4 v = make_int4(0, 0, 0, 0);
      float s = 0.0f;
      if (on) {
        const int64_t ph = (slot >> a.g.page_shift) * a.g.n_kv_heads + h;
        const int64_t at = ((ph << a.g.page_shift) + (slot & (a.g.page_rows - 1))) * a.g.head_dim + c * 16;
        v = __ldg(reinterpret_cast<const int4*>(a.pool + at));
        s = __ldg(a.scale + ph);
      }
      const int32_t w[4] = {v.x, v.y, v.z, v.w};
      alignas(16) T o[16];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        st_from_float(&o[e], __fmul_rn(static_cast<float>(static_cast<int8_t>(w[e / 4] >> (8 * (e % 4)))), s));
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (static_cast<int64_t>(row) * per_row + i) * 16);
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(o) / 16); ++k) dst[k] = reinterpret_cast<const uint4*>(o)[k];
    }
  }
}

template <int D, typename T, int ROPE>
cudaError_t launch_append_r(const Kv8AppendArgs& a, cudaStream_t st) {
  // Few tokens: windows of 16, for more blocks. Many: a page's rows, so that no block of a prompt's
  // window starts no run, and at least 32 or 64, so that its warps' registers are full (6.7 K rows in pages
  // of 16 with their reads 43 us, by windows of 16 77; 1100 single tokens 31 us, by windows of 16 29, of 64 37).
  const int32_t least = a.n_tokens < 1024 ? 16 : a.n_tokens < 4096 ? 32 : 64;
  const int32_t window = a.n_tokens < 1024 || a.g.page_rows < least ? least : a.g.page_rows;
  const dim3 grid((a.n_tokens + window - 1) / window, 2 * ((a.g.n_kv_heads + kHeads - 1) / kHeads));
  // Sixteen lanes to a row where there are many, for half the instructions (5 K rows of head_dim 128 in pages
  // of 128, unrotated, with their reads: 47 us, with a warp to a row 55); a warp to a row of 128 where
  // there are few and the way through one counts (64 single tokens: 11.6 us in a graph against 12.1).
  constexpr int kFew = D == 128 ? 32 : 16, kR = 32 / kFew;
  const bool few = a.n_tokens < 1024;
  auto kern = a.g.page_rows == 128
                  ? (few ? kv8_append_kernel<D, kFew, 8 / kR, 1, T, ROPE> : kv8_append_kernel<D, 16, 4, 1, T, ROPE>)
                  : (few ? kv8_append_kernel<D, kFew, 4 / kR, 2, T, ROPE> : kv8_append_kernel<D, 16, 2, 2, T, ROPE>);
  return launch_dependent(kern, grid, kWarps * 32, 0, st, a, window);
}

template <int D, typename T>
cudaError_t launch_append_t(const Kv8AppendArgs& a, cudaStream_t st) {
  if (a.rope_mode == AIHOST_ROPE_NONE) return launch_append_r<D, T, AIHOST_ROPE_NONE>(a, st);
  if (a.rope_mode == AIHOST_ROPE_NEOX) return launch_append_r<D, T, AIHOST_ROPE_NEOX>(a, st);
  return launch_append_r<D, T, AIHOST_ROPE_INTERLEAVED>(a, st);
}

template <int D>
cudaError_t launch_append_d(const Kv8AppendArgs& a, cudaStream_t st) {
  return a.io_dtype == AIHOST_F32 ? launch_append_t<D, float>(a, st) : launch_append_t<D, __half>(a, st);
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t st) {
  return a.g.head_dim == 64 ? launch_append_d<64>(a, st) : launch_append_d<128>(a, st);
}

cudaError_t launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t st) {
  const uint32_t per_row = a.g.n_kv_heads * (a.g.head_dim / 16), shift = a.g.head_dim == 64 ? 2 : 3;
  uint32_t x = 4;  // threads across a row: as many as it has chunks, up to the block's
  while (x < per_row && x < 256) x *= 2;
  const dim3 block(x, 256 / x);
  const int64_t want = (a.n_rows + block.y - 1) / block.y;
  const int blocks = static_cast<int>(want < 148 * 16 ? want : 148 * 16);
  return launch_dependent(a.out_dtype == AIHOST_F16 ? kv8_read_kernel<__half> : kv8_read_kernel<float>, blocks, block, 0, st, a,
                          per_row, shift);
}

}  // namespace aihost
