// kv8.h — launch interface of the 8-bit and the 4-bit paged cache: page bookkeeping, append, read, attention.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace aihost {

constexpr int64_t kKv8Counters = 1 << 16;      // tiles x heads whose chunks can be merged in one launch
constexpr int32_t kPageMapMaxBatch = 8192;  // two running sums of the batch are kept in shared memory

// Geometry of one layer's cache; page_rows = 1 << page_shift (16 .. 128). 8 bits: pools
// [n_pages][n_kv_heads][page_rows][head_dim], scales [n_pages][n_kv_heads]. 4 bits: pools
// [n_pages][n_kv_heads][page_rows][head_dim / 2] and, a 32-bit word each, ranges [n_pages][n_kv_heads][page_rows].
struct Kv8Geom {
  int32_t n_q_heads, n_kv_heads, head_dim;
  int32_t page_rows, page_shift, n_pages, max_pages;
};

struct PageMapArgs {
  int32_t batch, page_shift, n_pages, max_pages, max_tokens;
  const int32_t* seq_len;
  const int32_t* n_new;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* block_table;
  int32_t* kv_len;
  int32_t* row_start;
  int64_t* slots;
  int32_t* positions;
  int32_t* free_count_out;
  uint32_t* ticket;  // arrival counter of the blocks, zero between launches
  int32_t* status;
};

struct PageReleaseArgs {
  int32_t batch, page_shift, n_pages, max_pages;
  const int32_t* done;
  int32_t* seq_len;
  int32_t* block_table;
  int32_t* free_pages;
  int32_t* free_count;
  int32_t* status;
};

struct Kv8AppendArgs {
  Kv8Geom g;
  int32_t n_tokens, io_dtype, rope_mode;
  int64_t token_stride;  // bytes between tokens of k_new / v_new
  const void* k_new;
  const void* v_new;
  const int64_t* slots;
  const int32_t* positions;
  int8_t* k_pool;
  int8_t* v_pool;
  float* k_scale;
  float* v_scale;
  int32_t* status;
  RopeFreqs freqs;
};

struct Kv8ReadArgs {
  Kv8Geom g;
  int32_t n_rows, out_dtype;
  const int64_t* slots;
  const int8_t* pool;
  const float* scale;
  void* out;
  int32_t* status;
};

struct Kv4AppendArgs {
  Kv8Geom g;
  int32_t n_tokens, io_dtype, rope_mode;
  int64_t token_stride;  // bytes between tokens of k_new / v_new
  const void* k_new;
  const void* v_new;
  const int64_t* slots;
  const int32_t* positions;
  uint8_t* k_pool;
  uint8_t* v_pool;
  uint32_t* k_range;  // fp16 pairs (low, step)
  uint32_t* v_range;
  int32_t* status;
  RopeFreqs freqs;
};

struct Kv4ReadArgs {
  Kv8Geom g;
  int32_t n_rows, out_dtype;
  const int64_t* slots;
  const uint8_t* pool;
  const uint32_t* range;
  void* out;
  int32_t* status;
};

// Attention over either cache.
struct Kv8AttnArgs {
  Kv8Geom g;
  int32_t batch, n_tokens, max_new, max_kv;
  int32_t q_dtype, out_dtype, rope_mode;
  bool exact_q;  // rotated, and not to be rounded to fp16
  int64_t q_token_stride;  // bytes
  const void* q;
  const int32_t* row_start;
  const int32_t* kv_len;
  const int32_t* block_table;
  const int8_t* k_pool;
  const int8_t* v_pool;
  const float* k_scale;     // 8 bits
  const float* v_scale;
  const uint32_t* k_range;  // 4 bits
  const uint32_t* v_range;
  const int32_t* prefix_len;   // or NULL
  const int32_t* row_first;    // or NULL
  const float* alibi_slopes;   // or NULL
  void* out;
  float scale, score_cap;
  int32_t* status;
  // split over the cache rows (mma kernel): chunk rows each, partials and arrival counters
  int32_t tiles, chunk, max_splits;
  int32_t whole;   // tcgen05 kernel: so many (tile, head) units ahead of the others stay in one block
  float* part_o;   // [unit][split][rows][head_dim]
  float* part_ml;  // [unit][split][rows][2]
  uint32_t* counters;  // one for each tile and head, zero between launches
  RopeFreqs freqs;
};

int page_map_blocks(const PageMapArgs& a);  // only several use the ticket
cudaError_t launch_page_map(const PageMapArgs& a, cudaStream_t st);
cudaError_t launch_page_release(const PageReleaseArgs& a, cudaStream_t st);
cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t st);
cudaError_t launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t st);

// The split-cache kernel (mma.sync, query rows per tile 8 or 16) and its plan over the cache rows:
// tiles of query rows, cache rows per chunk, chunks of the longest range.
int32_t kv8_mma_rows(const Kv8Geom& g, int32_t max_new);
void kv8_mma_plan(const Kv8Geom& g, int32_t batch, int32_t n_tokens, int32_t max_new, int32_t max_kv, int32_t num_sms,
                  int32_t* tiles, int32_t* chunk, int32_t* splits);
cudaError_t launch_kv8_mma(const Kv8AttnArgs& a, cudaStream_t st);

// The same over the 4-bit cache.
cudaError_t launch_kv4_append(const Kv4AppendArgs& a, cudaStream_t st);
cudaError_t launch_kv4_read(const Kv4ReadArgs& a, cudaStream_t st);
void kv4_mma_plan(const Kv8Geom& g, int32_t batch, int32_t n_tokens, int32_t max_new, int32_t max_kv, int32_t num_sms,
                  int32_t* tiles, int32_t* chunk, int32_t* splits);
cudaError_t launch_kv4_mma(const Kv8AttnArgs& a, cudaStream_t st);

// The tcgen05 kernel (query rows per block 256) and its plan; *end: its length as the plan sees it, in
// times of one 128-row cache tile (about 2.1 us at head_dim 128, 2.4 with a rotated q that is not rounded, and 1.7 at 64). *whole: so many units
// (tile, head), before the others, are not cut.
int32_t kv8_prefill_rows();
void kv8_prefill_plan(const Kv8Geom& g, int32_t batch, int32_t n_tokens, int32_t max_new, int32_t max_kv, int32_t num_sms,
                      int32_t* tiles, int32_t* whole, int32_t* chunk, int32_t* splits, double* end);
cudaError_t launch_kv8_prefill(const Kv8AttnArgs& a, cudaStream_t st);
cudaError_t launch_kv4_prefill(const Kv8AttnArgs& a, cudaStream_t st);  // over the 4-bit cache, with the same plan

}  // namespace aihost
