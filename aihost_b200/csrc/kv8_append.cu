// kv8_append.cu — new K and V rows into the 8-bit paged cache, and rows of it back out.
//
// For each page and head that gets new rows x (K rotated first), in fp32:
//   had   = the page's scale, or 0 where its row 0 is among them (a page begun anew)
//   scale = max(had, amax|x| / 127)
//   older rows  q <- rint(q * (had / scale))   (only where the scale grew)
//   new rows    q  = rint(x * (1 / scale))
// The work unit is a run: the consecutive tokens whose slots are consecutive rows of one page.
#include "common.cuh"
#include "kv8.h"
#include "rows.cuh"

namespace aihost {
namespace {

constexpr int kWindow = 16;       // tokens whose runs one block handles
constexpr int kWarps = 8;
constexpr int kRowsPerWarp = 8;   // rows of a run that a warp holds in registers at a time
constexpr uint32_t kInfBits = 0x7f800000u;

// The runs that start in one window of tokens, for one head of K or V: all warps share a run where
// the window starts few (prompts: pages of consecutive rows), one warp takes a run where it starts
// many (decode: one row per sequence).
template <int D>
__global__ void __launch_bounds__(kWarps * 32) kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a) {
  constexpr int E = D / 32;
  __shared__ int32_t run_at[kWindow];
  __shared__ int32_t n_runs;
  __shared__ uint32_t warp_max[kWarps];
  __shared__ int32_t warp_len[kWarps];
  __shared__ float freqs[D / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t t0 = static_cast<int32_t>(blockIdx.x) * kWindow;
  const int32_t h = static_cast<int32_t>(blockIdx.y) >> 1;
  const bool is_k = (blockIdx.y & 1) == 0;
  const int32_t P = a.g.page_rows, H = a.g.n_kv_heads;
  const int64_t n_slots = static_cast<int64_t>(a.g.n_pages) << a.g.page_shift;
  const int32_t rope = is_k ? a.rope_mode : AIHOST_ROPE_NONE;

  if (rope != AIHOST_ROPE_NONE)
    for (int i = threadIdx.x; i < D / 2; i += blockDim.x) freqs[i] = a.freqs.f[i];
  if (warp == 0) {
    const int32_t t = t0 + lane;
    bool head = false;
    if (lane < kWindow && t < a.n_tokens) {
      const int64_t s = a.slots[t];
      if (s < -1 || s >= n_slots) {
        if (blockIdx.y == 0) atomicOr(a.status, kStatusBadIndex);
      } else if (s >= 0) {
        head = t == 0 || (s & (P - 1)) == 0 || a.slots[t - 1] != s - 1;
      }
    }
    const uint32_t m = __ballot_sync(0xffffffffu, head);
    if (head) run_at[__popc(m & ((1u << lane) - 1))] = t;
    if (lane == 0) n_runs = __popc(m);
  }
  __syncthreads();

  const bool shared = n_runs <= 2;  // all warps on each run, else a warp per run
  const int nw = shared ? kWarps : 1, w = shared ? warp : 0;
  int8_t* const pool = is_k ? a.k_pool : a.v_pool;
  float* const scales = is_k ? a.k_scale : a.v_scale;
  const uint8_t* const src = static_cast<const uint8_t*>(is_k ? a.k_new : a.v_new) +
                             static_cast<int64_t>(h) * D * (a.io_dtype == AIHOST_F32 ? 4 : 2);

  for (int r = shared ? 0 : warp; r < n_runs; r += shared ? 1 : kWarps) {
    const int32_t t = run_at[r];
    const int64_t slot = a.slots[t];
    const int64_t page = slot >> a.g.page_shift;
    const int32_t row0 = static_cast<int32_t>(slot & (P - 1));
    // the run's length: tokens t + i at slot + i, up to the page's end
    int32_t n = 1;
    const int32_t most = min(P - row0, a.n_tokens - t);
    if (most > 1) {
      int32_t len = most;
      for (int32_t i0 = 32 * w; i0 < most; i0 += 32 * nw) {
        const int32_t i = i0 + lane;
        const uint32_t off = __ballot_sync(0xffffffffu, i < most && a.slots[t + i] != slot + i);
        if (off) {
          len = i0 + __ffs(off) - 1;
          break;
        }
      }
      if (shared) {
        if (lane == 0) warp_len[warp] = len;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWarps; ++i) len = min(len, warp_len[i]);
      }
      n = len;
    }
    float x[kRowsPerWarp][E];
    auto load = [&](int32_t first) {
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i) {
        const int32_t k = first + i * nw + w;
        if (k < n) load_row_warp<E>(src + (t + k) * a.token_stride, a.io_dtype, lane, x[i]);
      }
      if (rope != AIHOST_ROPE_NONE) {
#pragma unroll
        for (int i = 0; i < kRowsPerWarp; ++i) {
          const int32_t k = first + i * nw + w;
          if (k < n) rope_row_warp<E>(x[i], lane, static_cast<float>(a.positions[t + k]), rope, freqs);
        }
      }
    };
    // amax as bits of |x|: infinities and NaN compare above every number
    uint32_t top = 0;
    const int32_t batch = kRowsPerWarp * nw, last = (n - 1) / batch * batch;
    for (int32_t first = 0; first < n; first += batch) {
      load(first);
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i)
        if (first + i * nw + w < n)
#pragma unroll
          for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (shared) {
      if (lane == 0) warp_max[warp] = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWarps; ++i) top = max(top, warp_max[i]);
    }
    float* const sp = scales + page * H + h;
    const float had = row0 == 0 ? 0.0f : *sp;
    const float need = top >= kInfBits ? __uint_as_float(0x7fffffffu) : __fmul_rn(__uint_as_float(top), 1.0f / 127.0f);
    const float scale = had != had || need != need ? __uint_as_float(0x7fffffffu) : fmaxf(had, need);
    // 0 for a NaN scale (its values do not matter) and where 1 / scale overflows (values below 2^-121)
    const float rcp = scale > 0.0f ? __frcp_rn(scale) : 0.0f;
    const float inv = rcp < __uint_as_float(kInfBits) ? rcp : 0.0f;
    int8_t* const base = pool + ((page * H + h) << a.g.page_shift) * D;
    if (scale > had && row0 > 0) {  // the older rows in the new scale (false for NaN)
      const float ratio = __fdiv_rn(had, scale);
      for (int32_t k = w; k < row0; k += nw) {
        int8_t* p = base + static_cast<int64_t>(k) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] = static_cast<int8_t>(__float2int_rn(__fmul_rn(static_cast<float>(p[e]), ratio)));
      }
    }
    for (int32_t first = last; first >= 0; first -= batch) {  // backwards: the last rows are still held
      if (first != last) load(first);
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i) {
        const int32_t k = first + i * nw + w;
        if (k < n) {
          uint32_t word = 0;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const int q = __float2int_rn(fminf(fmaxf(__fmul_rn(x[i][e], inv), -127.0f), 127.0f));
            word |= (static_cast<uint32_t>(q) & 0xffu) << (8 * e);
          }
          int8_t* p = base + static_cast<int64_t>(row0 + k) * D + lane * E;
          if (E == 4) *reinterpret_cast<uint32_t*>(p) = word;
          else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(word);
        }
      }
    }
    if (shared) __syncthreads();  // every warp has read the scale
    else __syncwarp();
    if (lane == 0 && w == 0) *sp = scale;
  }
}

// Rows of a pool as the values they stand for: 16 int8 (one 16-byte load) per thread and step.
template <typename T>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8ReadArgs a) {
  const int32_t per_row = a.g.n_kv_heads * (a.g.head_dim / 16), per_head = a.g.head_dim / 16;
  const int64_t n = static_cast<int64_t>(a.n_rows) * per_row;
  const int64_t n_slots = static_cast<int64_t>(a.g.n_pages) << a.g.page_shift;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / per_row;
    const int32_t rest = static_cast<int32_t>(i - row * per_row);
    const int32_t h = rest / per_head, c = rest % per_head;
    const int64_t slot = a.slots[row];
    int4 v = make_int4(0, 0, 0, 0);
    float s = 0.0f;
    if (slot >= 0 && slot < n_slots) {
      const int64_t ph = (slot >> a.g.page_shift) * a.g.n_kv_heads + h;
      const int64_t at = ((ph << a.g.page_shift) + (slot & (a.g.page_rows - 1))) * a.g.head_dim + c * 16;
      v = *reinterpret_cast<const int4*>(a.pool + at);
      s = a.scale[ph];
    } else if (slot != -1) {
      atomicOr(a.status, kStatusBadIndex);
    }
    const int32_t w[4] = {v.x, v.y, v.z, v.w};
    alignas(16) T o[16];
#pragma unroll
    for (int e = 0; e < 16; ++e)
      st_from_float(&o[e], __fmul_rn(static_cast<float>(static_cast<int8_t>(w[e / 4] >> (8 * (e % 4)))), s));
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + i * 16);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(o) / 16); ++k) dst[k] = reinterpret_cast<const uint4*>(o)[k];
  }
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t st) {
  const dim3 grid((a.n_tokens + kWindow - 1) / kWindow, 2 * a.g.n_kv_heads);
  if (a.g.head_dim == 64) kv8_append_kernel<64><<<grid, kWarps * 32, 0, st>>>(a);
  else kv8_append_kernel<128><<<grid, kWarps * 32, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t st) {
  const int64_t n = static_cast<int64_t>(a.n_rows) * a.g.n_kv_heads * (a.g.head_dim / 16);
  const int64_t want = (n + 255) / 256;
  const int blocks = static_cast<int>(want < 148 * 16 ? want : 148 * 16);
  if (a.out_dtype == AIHOST_F16) kv8_read_kernel<__half><<<blocks, 256, 0, st>>>(a);
  else kv8_read_kernel<float><<<blocks, 256, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace aihost
