// kv8_pages.cu — page bookkeeping of a serving step on the GPU: block tables, slots and positions
// from the requests' lengths (aihost_page_map), and the return of finished requests' pages
// (aihost_page_release).
//   row_start[b] = sum of n_new before b,   kv_len[b] = seq_len[b] + n_new[b]
//   position of token i of b = seq_len[b] + i,   slot = table[b][position / P] * P + position % P
// and the pages that b newly needs come off the free stack at (sum of the pages taken before b).
// Integer work of 12 bytes a token, bound by the dependent reads lengths -> running sums -> table or
// stack entry -> slot. So the running sums are 64-bit scans in one block's registers and shared memory,
// and each block repeats them for itself, which is cheaper than a second launch or a grid barrier.
// Measured: 64 one-token sequences 3.1 us in a graph, 512 with 73 K tokens in all 5.7 us; either called
// one at a time 5.5 us, the host's enqueue. (Blocks that wait for one that scans: 9.2 us; Python's page loop
// with its copies: 304.)
#include "common.cuh"
#include "kv8.h"
#include "kv8_tile.cuh"

namespace aihost {
namespace {

struct Sums {
  int64_t tokens, pages;
};

__device__ __forceinline__ Sums add(Sums a, Sums b) { return {a.tokens + b.tokens, a.pages + b.pages}; }

__device__ __forceinline__ Sums warp_scan(Sums v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums u = {__shfl_up_sync(0xffffffffu, v.tokens, o), __shfl_up_sync(0xffffffffu, v.pages, o)};
    if (lane >= o) v = add(v, u);
  }
  return v;
}

// Running sums over the block's threads: returns the exclusive sum, *total the block's sum.
__device__ __forceinline__ Sums block_scan(Sums v, Sums* warp_sums, Sums* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const Sums in = warp_scan(v, lane);
  if (lane == 31) warp_sums[warp] = in;
  __syncthreads();
  if (warp == 0) {
    const Sums w = warp_scan(lane < warps ? warp_sums[lane] : Sums{0, 0}, lane);
    __syncwarp();
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[warps - 1];
  Sums ex = warp ? warp_sums[warp - 1] : Sums{0, 0};
  ex = add(ex, {in.tokens - v.tokens, in.pages - v.pages});
  __syncthreads();
  return ex;
}

__device__ __forceinline__ int32_t pages_of(int64_t rows, int32_t shift) {
  return static_cast<int32_t>((rows + (1 << shift) - 1) >> shift);
}

// Every block adds up the whole batch for itself (a few sums per thread), so no block waits for
// another; then each takes its share of the tokens. Nothing a block reads is written by another,
// but for kv_len and free_count_out where they are seq_len and free_count themselves: those two
// are written by the last block to have read them.
__global__ void __launch_bounds__(1024) page_map_kernel(const PageMapArgs a) {
  extern __shared__ int32_t sums[];  // [batch + 1] token starts, [batch] pages taken before
  int32_t* start = sums;
  int32_t* taken = sums + a.batch + 1;
  __shared__ Sums warp_sums[32];
  __shared__ int32_t last_block;
  griddep_wait();
  griddep_launch_dependents();
  const int32_t avail = *a.free_count;
  Sums carry = {0, 0};
  bool bad = avail < 0 || avail > a.n_pages;
  for (int32_t b0 = 0; b0 < a.batch; b0 += blockDim.x) {
    const int32_t b = b0 + threadIdx.x;
    Sums v = {0, 0};
    if (b < a.batch) {
      const int64_t n = a.n_new[b], c = a.seq_len[b];
      if (n < 0 || c < 0 || (c + n) > (static_cast<int64_t>(a.max_pages) << a.page_shift)) bad = true;
      else v = {n, pages_of(c + n, a.page_shift) - pages_of(c, a.page_shift)};
    }
    Sums total;
    const Sums ex = add(carry, block_scan(v, warp_sums, &total));
    carry = add(carry, total);
    if (b < a.batch) {  // sums past 2^31 are refused below and never read
      start[b] = static_cast<int32_t>(ex.tokens);
      taken[b] = static_cast<int32_t>(ex.pages);
    }
  }
  bad = __syncthreads_or(bad || carry.tokens > a.max_tokens);
  const bool refused = bad || carry.pages > avail;
  const int32_t n_tokens = refused ? 0 : static_cast<int32_t>(carry.tokens);

  bool stray = false;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; t < a.max_tokens;
       t += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int64_t slot = -1;
    int32_t pos = 0;
    if (t < n_tokens) {
      int32_t lo = 0, hi = a.batch;  // the last sequence that starts at or before t
      while (hi - lo > 1) {
        const int32_t mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int32_t c = a.seq_len[lo], have = pages_of(c, a.page_shift);
      pos = c + static_cast<int32_t>(t) - start[lo];
      const int32_t p = pos >> a.page_shift, row = pos & ((1 << a.page_shift) - 1);
      int32_t* entry = a.block_table + static_cast<int64_t>(lo) * a.max_pages + p;
      int32_t page;
      if (p < have) {
        page = *entry;
      } else {
        page = a.free_pages[avail - 1 - (taken[lo] + p - have)];
        if (row == 0) *entry = page;  // a page's row 0 is new in the step that takes the page
      }
      if (page >= 0 && page < a.n_pages) slot = (static_cast<int64_t>(page) << a.page_shift) + row;
      else stray = true;
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
  if (stray) atomicOr(a.status, kStatusBadIndex);

  if (blockIdx.x == 0) {
    for (int32_t b = threadIdx.x; b <= a.batch; b += blockDim.x)
      a.row_start[b] = refused ? 0 : b < a.batch ? start[b] : n_tokens;
    if (threadIdx.x == 0 && refused) atomicOr(a.status, bad ? kStatusBadIndex : kStatusNoPages);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last_block = gridDim.x == 1 || last_to_arrive(a.ticket, gridDim.x);
  }
  __syncthreads();
  if (!last_block) return;
  for (int32_t b = threadIdx.x; b < a.batch; b += blockDim.x)
    a.kv_len[b] = refused ? a.seq_len[b] : a.seq_len[b] + a.n_new[b];
  if (threadIdx.x == 0) *a.free_count_out = refused ? avail : avail - static_cast<int32_t>(carry.pages);
}

// One block: the pages of all ended sequences go on the stack in order. Checked first, so that a
// table with a page outside the pool, or a stack that would overflow, changes nothing.
__global__ void __launch_bounds__(1024) page_release_kernel(const PageReleaseArgs a) {
  extern __shared__ int32_t before[];  // [batch] pages returned before
  __shared__ Sums warp_sums[32];
  griddep_wait();
  griddep_launch_dependents();
  const int32_t have = *a.free_count;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  bool bad = have < 0;
  Sums carry = {0, 0};
  for (int32_t b0 = 0; b0 < a.batch; b0 += blockDim.x) {
    const int32_t b = b0 + threadIdx.x;
    Sums v = {0, 0};
    if (b < a.batch && a.done[b]) {
      const int64_t c = a.seq_len[b];
      if (c < 0 || c > (static_cast<int64_t>(a.max_pages) << a.page_shift)) bad = true;
      else v.pages = pages_of(c, a.page_shift);
    }
    Sums total;
    const Sums ex = add(carry, block_scan(v, warp_sums, &total));
    carry = add(carry, total);
    if (b < a.batch) before[b] = static_cast<int32_t>(ex.pages);
  }
  bad = __syncthreads_or(bad || have + carry.pages > a.n_pages);
  if (!bad) {
    bool stray = false;
    for (int32_t b = warp; b < a.batch; b += warps) {
      if (!a.done[b]) continue;
      const int32_t n = pages_of(a.seq_len[b], a.page_shift);
      for (int32_t p = lane; p < n; p += 32) {
        const int32_t page = a.block_table[static_cast<int64_t>(b) * a.max_pages + p];
        stray |= page < 0 || page >= a.n_pages;
      }
    }
    bad = __syncthreads_or(stray);
  }
  if (bad) {
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadIndex);
    return;
  }
  for (int32_t b = warp; b < a.batch; b += warps) {
    if (!a.done[b]) continue;
    const int32_t n = pages_of(a.seq_len[b], a.page_shift);
    for (int32_t p = lane; p < a.max_pages; p += 32) {
      int32_t* entry = a.block_table + static_cast<int64_t>(b) * a.max_pages + p;
      if (p < n) a.free_pages[have + before[b] + p] = *entry;
      *entry = -1;
    }
    __syncwarp();
    if (lane == 0) a.seq_len[b] = 0;
  }
  if (threadIdx.x == 0) *a.free_count = have + static_cast<int32_t>(carry.pages);
}

}  // namespace

static int page_map_threads(const PageMapArgs& a) { return a.batch <= 256 && a.max_tokens <= 256 ? 256 : 1024; }

int page_map_blocks(const PageMapArgs& a) {
  const int threads = page_map_threads(a);
  const int64_t blocks = (static_cast<int64_t>(a.max_tokens) + threads - 1) / threads;
  return blocks < 1 ? 1 : blocks > 148 ? 148 : static_cast<int>(blocks);
}

cudaError_t launch_page_map(const PageMapArgs& a, cudaStream_t st) {
  const int threads = page_map_threads(a), blocks = page_map_blocks(a);
  const size_t smem = (2 * static_cast<size_t>(a.batch) + 1) * sizeof(int32_t);
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(page_map_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  return launch_dependent(page_map_kernel, blocks, threads, smem, st, a);
}

cudaError_t launch_page_release(const PageReleaseArgs& a, cudaStream_t st) {
  return launch_dependent(page_release_kernel, 1, a.batch <= 256 ? 256 : 1024,
                          static_cast<size_t>(a.batch) * sizeof(int32_t), st, a);
}

}  // namespace aihost
