// kv8_api.cu — the extern "C" boundary of the 8-bit and the 4-bit paged cache (declared in include/aihost_attn.h):
// argument checks, resolved strides, the split plan and the launches. Allocates nothing.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "common.cuh"
#include "ctx.h"
#include "kv8.h"

using namespace aihost;

namespace {

constexpr int32_t kMaxKv = INT32_MAX - 8192;  // rows of a sequence: chunks of them are rounded up, within int32

int32_t page_shift_of(int32_t page_rows) {
  return page_rows == 16 ? 4 : page_rows == 32 ? 5 : page_rows == 64 ? 6 : page_rows == 128 ? 7 : -1;
}

// The frequency table of a description; the last one is kept (64 powers cost as much as a launch).
const RopeFreqs& freqs_of(aihost_attn_ctx* ctx, const aihost_kv8_desc* d) {
  if (ctx->freqs_dim != d->head_dim || ctx->freqs_theta != d->rope_theta) {
    ctx->freqs = make_freqs(d->rope_theta, d->head_dim);
    ctx->freqs_theta = d->rope_theta;
    ctx->freqs_dim = d->head_dim;
  }
  return ctx->freqs;
}

struct Resolved {
  Kv8Geom g;
  int32_t rope_mode;
  bool exact_q;  // rotated, and not to be rounded to fp16
  float scale;
  int64_t q_stride, kv_stride;  // bytes between tokens
};

aihost_status check_kv8(const aihost_kv8_desc* d, Resolved* r) {
  if (!d) return fail(AIHOST_EINVAL, "desc is NULL");
  if (d->n_q_heads < 1 || d->n_kv_heads < 1 || d->n_kv_heads > 32767)
    return fail(AIHOST_EINVAL, "n_q_heads (%d) and n_kv_heads (%d) must be >= 1 (n_kv_heads at most 32767)", d->n_q_heads,
                d->n_kv_heads);
  if (d->n_q_heads % d->n_kv_heads)
    return fail(AIHOST_EINVAL, "n_q_heads (%d) must be a multiple of n_kv_heads (%d)", d->n_q_heads, d->n_kv_heads);
  if (d->head_dim != 64 && d->head_dim != 128)
    return fail(AIHOST_EUNSUPPORTED, "head_dim %d is not supported (64 or 128)", d->head_dim);
  const int32_t shift = page_shift_of(d->page_rows);
  if (shift < 0) return fail(AIHOST_EUNSUPPORTED, "page_rows %d is not supported (16, 32, 64 or 128)", d->page_rows);
  if (d->n_pages < 1 || d->max_pages < 1)
    return fail(AIHOST_EINVAL, "n_pages (%d) and max_pages (%d) must be >= 1", d->n_pages, d->max_pages);
  if (d->io_dtype != AIHOST_F32 && d->io_dtype != AIHOST_F16)
    return fail(AIHOST_EINVAL, "io_dtype %d must be F32 (0) or F16 (1)", d->io_dtype);
  if (d->out_dtype != AIHOST_F32 && d->out_dtype != AIHOST_F16)
    return fail(AIHOST_EINVAL, "out_dtype %d must be F32 (0) or F16 (1)", d->out_dtype);
  r->rope_mode = d->rope_mode & ~AIHOST_KV8_ROUND_Q;
  if (r->rope_mode < AIHOST_ROPE_INTERLEAVED || r->rope_mode > AIHOST_ROPE_NONE)
    return fail(AIHOST_EINVAL, "rope_mode %d is not a valid aihost_rope_mode", d->rope_mode);
  r->exact_q = d->rope_mode == r->rope_mode && r->rope_mode != AIHOST_ROPE_NONE;
  if (r->rope_mode != AIHOST_ROPE_NONE && !(d->rope_theta > 0.0f && isfinite(d->rope_theta)))
    return fail(AIHOST_EINVAL, "rope_theta must be a positive finite number");
  if (!(isfinite(d->scale) && d->scale >= 0.0f)) return fail(AIHOST_EINVAL, "scale must be >= 0 and finite");
  if (!(isfinite(d->score_cap) && d->score_cap >= 0.0f)) return fail(AIHOST_EINVAL, "score_cap must be >= 0 and finite");
  const int64_t eb = d->io_dtype == AIHOST_F32 ? 4 : 2;
  const int64_t q_row = eb * d->n_q_heads * d->head_dim, kv_row = eb * d->n_kv_heads * d->head_dim;
  r->q_stride = d->q_token_stride ? d->q_token_stride : q_row;
  r->kv_stride = d->kv_token_stride ? d->kv_token_stride : kv_row;
  if (r->q_stride < q_row || r->kv_stride < kv_row)
    return fail(AIHOST_EINVAL, "q_token_stride and kv_token_stride must be at least one token's bytes (%lld and %lld)",
                static_cast<long long>(q_row), static_cast<long long>(kv_row));
  if (r->q_stride % 16 || r->kv_stride % 16)
    return fail(AIHOST_EINVAL, "q_token_stride and kv_token_stride must be multiples of 16 bytes");
  r->g = Kv8Geom{d->n_q_heads, d->n_kv_heads, d->head_dim, d->page_rows, shift, d->n_pages, d->max_pages};
  r->scale = d->scale != 0.0f ? d->scale : 1.0f / sqrtf(static_cast<float>(d->head_dim));
  return AIHOST_OK;
}

aihost_status check_pages(const aihost_attn_ctx* ctx, int32_t batch, int32_t page_rows, int32_t n_pages, int32_t max_pages,
                          int32_t* shift) {
  if (!ctx) return fail(AIHOST_EINVAL, "ctx is NULL");
  if (batch < 1) return fail(AIHOST_EINVAL, "batch (%d) must be >= 1", batch);
  if (batch > kPageMapMaxBatch) return fail(AIHOST_EUNSUPPORTED, "batch %d is over %d", batch, kPageMapMaxBatch);
  *shift = page_shift_of(page_rows);
  if (*shift < 0) return fail(AIHOST_EUNSUPPORTED, "page_rows %d is not supported (16, 32, 64 or 128)", page_rows);
  if (n_pages < 1 || max_pages < 1)
    return fail(AIHOST_EINVAL, "n_pages (%d) and max_pages (%d) must be >= 1", n_pages, max_pages);
  // positions and lengths are int32
  if ((static_cast<int64_t>(max_pages) << *shift) > INT32_MAX)
    return fail(AIHOST_EINVAL, "max_pages * page_rows must stay below 2^31");
  return AIHOST_OK;
}

// Which kernel an attention call runs, and its plan over the cache rows.
struct Plan {
  bool tensor;  // the tcgen05 kernel (many query rows a sequence, fp16), else the split-cache one
  int32_t rows, tiles, whole, chunk, splits;  // whole: units that are not split, before the others
  int64_t parts(const Kv8Geom& g) const { return (static_cast<int64_t>(tiles) * g.n_kv_heads - whole) * splits * rows; }
  size_t scratch(const Kv8Geom& g) const {
    return splits <= 1 ? 0 : static_cast<size_t>(parts(g)) * (g.head_dim + 2) * sizeof(float);
  }
};

Plan make_plan(const aihost_kv8_desc* d, const Resolved& r, bool four, int32_t batch, int32_t n_tokens, int32_t max_new,
               int32_t max_kv, int32_t num_sms) {
  // The tcgen05 kernel takes fp16 rows by 256 and has ~12 us of fixed work a block; the split-cache one
  // takes 16 and rereads the cache for each tile, ~50 ns (head_dim 64: 37) per tile and 1000 rows over the
  // whole GPU, and fills it with little work. Measured, head_dim 128, 32/8 heads, tcgen05 against split-cache,
  // q not rotated: 8 sequences of 8192 rows with 8 new ones 87 and 73 us, with 16 87 and 125; one sequence with
  // 32 43 and 43, with 64 45 and 70; 8 of 512 rows with 16 21 and 15, with 32 21 and 28. A rotated q costs the
  // split-cache kernel a quarter more, the other one 2 %: 89 and 93 us for the first of these.
  // The rule knows the batch, not its sequences: it takes the cached rows to be spread as the new ones are. A
  // step that mixes long prompts with single tokens over long caches runs on one kernel, and either is
  // wrong for a part of it: 63 single tokens over 256 to 8192 rows beside a prompt of 2048 take 526 us so, 573
  // on the tcgen05 kernel, and 115 + 58 as two calls.
  // Over the 4-bit cache, tcgen05 against split-cache, q not rotated: 8 sequences of 8192 rows with 8 new ones 159 and 75
  // us, with 16 160 and 111, with 32 160 and 201; one sequence with 32 56 and 46, with 64 61 and 75; 8 of 512 rows with 16
  // 31 and 15, with 32 31 and 28, with 64 36 and 52. Rotated: 146 and 139 for 8 of 8192 with 16, 148 and 227 with 32.
  // head_dim 64, the same steps: 118 and 52, 118 and 77, 119 and 139; 40 and 33, 46 and 52; 26 and 11, 26 and 19, 30 and 36;
  // rotated 123 and 89, 123 and 159; 14/2 heads, 8 of 8192 with 8 47 and 34, with 16 47 and 37, with 32 54 and 76. The constants
  // for 64 are a fit to 46 such pairs, of which none takes a kernel over 8 % slower than the other. At 128 16 new rows over
  // 8192 go to the slower one.
  Plan p;
  const Kv8Geom& g = r.g;
  max_kv = std::min(max_kv, kMaxKv);
  const int32_t rows = kv8_mma_rows(g, max_new), G = g.n_q_heads / g.n_kv_heads;
  p.tensor = false;
  if (d->io_dtype == AIHOST_F16 && static_cast<int64_t>(max_new) * G > rows) {
    double end;
    kv8_prefill_plan(g, batch, n_tokens, max_new, max_kv, num_sms, &p.tiles, &p.whole, &p.chunk, &p.splits, &end);
    const double even = static_cast<double>(n_tokens) / (static_cast<double>(batch) * max_new);
    const double by_tc = end * (four ? (g.head_dim == 64 ? 2.5 : r.exact_q ? 3.2 : 2.9) : g.head_dim == 64 ? 1.7 : r.exact_q ? 2.4 : 2.1);
    const double tiles16 = (static_cast<double>(n_tokens) * G / rows + 0.5 * batch) * g.n_kv_heads;
    const double row = four ? (g.head_dim == 64 ? 32e-6 : r.exact_q ? 54e-6 : 42e-6) : g.head_dim == 128 ? 50e-6 : 37e-6;
    const double by_mma = 8.0 + (four ? 1e-3 * max_kv : 0.0) + tiles16 * max_kv * (even > 0.9 ? 1.0 : even) * row;
    p.tensor = by_tc < by_mma;
  }
  if (p.tensor) {
    p.rows = kv8_prefill_rows();
  } else {
    p.rows = rows;
    p.whole = 0;
    (four ? kv4_mma_plan : kv8_mma_plan)(g, batch, n_tokens, max_new, max_kv, num_sms, &p.tiles, &p.chunk, &p.splits);
  }
  return p;
}

int32_t current_sms() {
  int sms = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Sizes of an attention call, from host-known bounds.
aihost_status check_sizes(int32_t batch, int32_t n_tokens, int32_t max_new, int32_t max_kv) {
  if (batch < 1) return fail(AIHOST_EINVAL, "batch (%d) must be >= 1", batch);
  if (n_tokens < 0) return fail(AIHOST_EINVAL, "n_tokens (%d) must be >= 0", n_tokens);
  if (max_new < 1 || max_kv < max_new)
    return fail(AIHOST_EINVAL, "max_new (%d) must be >= 1 and max_kv (%d) at least max_new", max_new, max_kv);
  return AIHOST_OK;
}

aihost_status tell_plan(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, bool four, int32_t batch, int32_t n_tokens,
                        int32_t max_new, int32_t max_kv, size_t* out_bytes, int32_t* out_kernel) {
  Resolved r;
  aihost_status s = check_kv8(desc, &r);
  if (s == AIHOST_OK) s = check_sizes(batch, n_tokens, max_new, max_kv);
  if (s != AIHOST_OK) return s;
  const Plan plan = make_plan(desc, r, four, batch, n_tokens, max_new, max_kv, ctx ? ctx->num_sms : current_sms());
  if (out_bytes) *out_bytes = plan.scratch(r.g);
  if (out_kernel) *out_kernel = plan.tensor ? AIHOST_KV8_TENSOR : AIHOST_KV8_SPLIT_CACHE;
  return AIHOST_OK;
}

// The caches differ in what the pools and their factors are.
struct CachePtrs {
  const void* k_pool;
  const void* v_pool;
  const void* k_factor;  // scales or ranges
  const void* v_factor;
};

aihost_status attention(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, bool four, int32_t batch, int32_t n_tokens,
                        int32_t max_new, int32_t max_kv, const void* q, const int32_t* row_start, const int32_t* kv_len,
                        const int32_t* block_table, const CachePtrs& c, const int32_t* prefix_len, const int32_t* row_first,
                        const float* alibi_slopes, void* out, void* stream) {
  if (!ctx) return fail(AIHOST_EINVAL, "ctx is NULL");
  Resolved r;
  aihost_status s = check_kv8(desc, &r);
  if (s == AIHOST_OK) s = check_sizes(batch, n_tokens, max_new, max_kv);
  if (s != AIHOST_OK) return s;
  if (n_tokens == 0) return AIHOST_OK;
  if (!q || !row_start || !kv_len || !block_table || !c.k_pool || !c.v_pool || !c.k_factor || !c.v_factor || !out)
    return fail(AIHOST_EINVAL, "every array but prefix_len, row_first and alibi_slopes must be non-NULL");
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(c.k_pool, 16) || !aligned(c.v_pool, 16) || !aligned(row_start, 4) ||
      !aligned(kv_len, 4) || !aligned(block_table, 4) || !aligned(c.k_factor, four ? 16 : 4) || !aligned(c.v_factor, four ? 16 : 4) ||
      !aligned(prefix_len, 4) || !aligned(row_first, 4) || !aligned(alibi_slopes, 4))
    return fail(AIHOST_EINVAL, four ? "q, out, the pools and the ranges must be 16-byte, other arrays 4-byte aligned"
                                   : "q, out and the pools must be 16-byte, other arrays 4-byte aligned");
  Kv8AttnArgs a;
  memset(&a, 0, sizeof(a));
  a.g = r.g;
  a.batch = batch;
  a.n_tokens = n_tokens;
  a.max_new = max_new;
  a.max_kv = std::min(max_kv, kMaxKv);
  a.q_dtype = desc->io_dtype;
  a.out_dtype = desc->out_dtype;
  a.rope_mode = r.rope_mode;
  a.exact_q = r.exact_q;
  a.q_token_stride = r.q_stride;
  a.q = q;
  a.row_start = row_start;
  a.kv_len = kv_len;
  a.block_table = block_table;
  a.k_pool = static_cast<const int8_t*>(c.k_pool);
  a.v_pool = static_cast<const int8_t*>(c.v_pool);
  if (four) {
    a.k_range = static_cast<const uint32_t*>(c.k_factor);
    a.v_range = static_cast<const uint32_t*>(c.v_factor);
  } else {
    a.k_scale = static_cast<const float*>(c.k_factor);
    a.v_scale = static_cast<const float*>(c.v_factor);
  }
  a.prefix_len = prefix_len;
  a.row_first = row_first;
  a.alibi_slopes = alibi_slopes;
  a.out = out;
  a.scale = r.scale;
  // cap tanh(s / cap) in fp32 wants scale / cap and cap log2(e) to be normal numbers: beyond 1e30 it is s itself,
  // below 1e-30 the scores are alike either way (1e-20 where the codes' unit 2^20 joins the factor)
  a.score_cap = desc->score_cap > 1e30f || desc->score_cap == 0.0f ? 0.0f : std::max(desc->score_cap, four ? 1e-20f : 1e-30f);
  a.status = ctx->d_status;
  if (r.rope_mode != AIHOST_ROPE_NONE) a.freqs = freqs_of(ctx, desc);
  const Plan plan = make_plan(desc, r, four, batch, n_tokens, max_new, max_kv, ctx->num_sms);
  a.tiles = plan.tiles;
  a.chunk = plan.chunk;
  a.max_splits = plan.splits;
  a.whole = plan.whole;
  if (static_cast<int64_t>(a.tiles) * r.g.n_kv_heads > INT32_MAX)
    return fail(AIHOST_EUNSUPPORTED, "n_tokens %d needs too many blocks", n_tokens);
  const size_t need = plan.scratch(r.g);
  if (need > ctx->scratch_bytes)
    return fail(AIHOST_ENOMEM, "attention needs %zu bytes of scratch, context has %zu (call aihost_attn_reserve)", need,
                ctx->scratch_bytes);
  if (need) {
    a.part_o = static_cast<float*>(ctx->scratch);
    a.part_ml = a.part_o + static_cast<size_t>(plan.parts(r.g)) * r.g.head_dim;
    a.counters = ctx->kv8_counters + 1;
  }
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(AIHOST_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SharedUse shared(ctx, st, need > 0);
  if (shared.error() != cudaSuccess) return cuda_fail(shared.error(), "ordering the scratch's uses");
  cudaError_t e = timed_launch(ctx, four ? AIHOST_KERNEL_KV4_ATTN : AIHOST_KERNEL_KV8_ATTN, st, [&] {
    if (four) return plan.tensor ? launch_kv4_prefill(a, st) : launch_kv4_mma(a, st);
    return plan.tensor ? launch_kv8_prefill(a, st) : launch_kv8_mma(a, st);
  });
  return e == cudaSuccess ? AIHOST_OK : cuda_fail(e, four ? "4-bit attention launch" : "8-bit attention launch");
}

}  // namespace

extern "C" {

aihost_status aihost_page_map(aihost_attn_ctx* ctx, int32_t batch, int32_t page_rows, int32_t n_pages, int32_t max_pages,
                              int32_t max_tokens, const int32_t* seq_len, const int32_t* n_new,
                              const int32_t* free_pages, const int32_t* free_count, int32_t* block_table,
                              int32_t* kv_len, int32_t* row_start, int64_t* slots, int32_t* positions,
                              int32_t* free_count_out, void* stream) {
  PageMapArgs a;
  aihost_status s = check_pages(ctx, batch, page_rows, n_pages, max_pages, &a.page_shift);
  if (s != AIHOST_OK) return s;
  if (max_tokens < 0) return fail(AIHOST_EINVAL, "max_tokens (%d) must be >= 0", max_tokens);
  if (!seq_len || !n_new || !free_pages || !free_count || !block_table || !kv_len || !row_start || !free_count_out ||
      (max_tokens > 0 && (!slots || !positions)))
    return fail(AIHOST_EINVAL, "every array must be non-NULL");
  if (!aligned(seq_len, 4) || !aligned(n_new, 4) || !aligned(free_pages, 4) || !aligned(free_count, 4) ||
      !aligned(block_table, 4) || !aligned(kv_len, 4) || !aligned(row_start, 4) || !aligned(slots, 8) ||
      !aligned(positions, 4) || !aligned(free_count_out, 4))
    return fail(AIHOST_EINVAL, "int32 arrays must be 4-byte and slots 8-byte aligned");
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(AIHOST_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
  a.batch = batch;
  a.n_pages = n_pages;
  a.max_pages = max_pages;
  a.max_tokens = max_tokens;
  a.seq_len = seq_len;
  a.n_new = n_new;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.block_table = block_table;
  a.kv_len = kv_len;
  a.row_start = row_start;
  a.slots = slots;
  a.positions = positions;
  a.free_count_out = free_count_out;
  a.ticket = ctx->kv8_counters;
  a.status = ctx->d_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SharedUse shared(ctx, st, page_map_blocks(a) > 1);  // the ticket
  if (shared.error() != cudaSuccess) return cuda_fail(shared.error(), "ordering the page maps");
  cudaError_t e = timed_launch(ctx, AIHOST_KERNEL_PAGES, st, [&] { return launch_page_map(a, st); });
  return e == cudaSuccess ? AIHOST_OK : cuda_fail(e, "page map launch");
}

aihost_status aihost_page_release(aihost_attn_ctx* ctx, int32_t batch, int32_t page_rows, int32_t n_pages,
                                  int32_t max_pages, const int32_t* done, int32_t* seq_len, int32_t* block_table,
                                  int32_t* free_pages, int32_t* free_count, void* stream) {
  PageReleaseArgs a;
  aihost_status s = check_pages(ctx, batch, page_rows, n_pages, max_pages, &a.page_shift);
  if (s != AIHOST_OK) return s;
  if (!done || !seq_len || !block_table || !free_pages || !free_count)
    return fail(AIHOST_EINVAL, "every array must be non-NULL");
  if (!aligned(done, 4) || !aligned(seq_len, 4) || !aligned(block_table, 4) || !aligned(free_pages, 4) ||
      !aligned(free_count, 4))
    return fail(AIHOST_EINVAL, "int32 arrays must be 4-byte aligned");
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(AIHOST_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
  a.batch = batch;
  a.n_pages = n_pages;
  a.max_pages = max_pages;
  a.done = done;
  a.seq_len = seq_len;
  a.block_table = block_table;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.status = ctx->d_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = timed_launch(ctx, AIHOST_KERNEL_PAGES, st, [&] { return launch_page_release(a, st); });
  return e == cudaSuccess ? AIHOST_OK : cuda_fail(e, "page release launch");
}

aihost_status aihost_kv8_append(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, int32_t n_tokens, const void* k_new,
                                const void* v_new, const int64_t* slots, const int32_t* positions, int8_t* k_pool,
                                int8_t* v_pool, float* k_scale, float* v_scale, void* stream) {
  if (!ctx) return fail(AIHOST_EINVAL, "ctx is NULL");
  Resolved r;
  aihost_status s = check_kv8(desc, &r);
  if (s != AIHOST_OK) return s;
  if (n_tokens < 0) return fail(AIHOST_EINVAL, "n_tokens (%d) must be >= 0", n_tokens);
  if (n_tokens == 0) return AIHOST_OK;
  if (!k_new || !v_new || !slots || !k_pool || !v_pool || !k_scale || !v_scale ||
      (!positions && r.rope_mode != AIHOST_ROPE_NONE))
    return fail(AIHOST_EINVAL, "every array must be non-NULL (positions may be NULL with rope_mode NONE)");
  if (!aligned(k_new, 16) || !aligned(v_new, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(slots, 8) ||
      !aligned(positions, 4) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return fail(AIHOST_EINVAL, "k_new, v_new and the pools must be 16-byte, slots 8-byte, other arrays 4-byte aligned");
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(AIHOST_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
  Kv8AppendArgs a;
  a.g = r.g;
  a.n_tokens = n_tokens;
  a.io_dtype = desc->io_dtype;
  a.rope_mode = r.rope_mode;
  a.token_stride = r.kv_stride;
  a.k_new = k_new;
  a.v_new = v_new;
  a.slots = slots;
  a.positions = positions;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.status = ctx->d_status;
  if (r.rope_mode != AIHOST_ROPE_NONE) a.freqs = freqs_of(ctx, desc);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = timed_launch(ctx, AIHOST_KERNEL_KV8_APPEND, st, [&] { return launch_kv8_append(a, st); });
  return e == cudaSuccess ? AIHOST_OK : cuda_fail(e, "8-bit append launch");
}

aihost_status aihost_kv8_read(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, int32_t n_rows, const int64_t* slots,
                              const int8_t* pool, const float* scale, void* out, int32_t out_dtype, void* stream) {
  if (!ctx) return fail(AIHOST_EINVAL, "ctx is NULL");
  Resolved r;
  aihost_status s = check_kv8(desc, &r);
  if (s != AIHOST_OK) return s;
  if (out_dtype != AIHOST_F32 && out_dtype != AIHOST_F16)
    return fail(AIHOST_EINVAL, "out_dtype %d must be F32 (0) or F16 (1)", out_dtype);
  if (n_rows < 0) return fail(AIHOST_EINVAL, "n_rows (%d) must be >= 0", n_rows);
  if (n_rows == 0) return AIHOST_OK;
  if (!slots || !pool || !scale || !out) return fail(AIHOST_EINVAL, "slots, pool, scale and out must be non-NULL");
  if (!aligned(slots, 8) || !aligned(pool, 16) || !aligned(scale, 4) || !aligned(out, 16))
    return fail(AIHOST_EINVAL, "pool and out must be 16-byte, slots 8-byte, scale 4-byte aligned");
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(AIHOST_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
  Kv8ReadArgs a{r.g, n_rows, out_dtype, slots, pool, scale, out, ctx->d_status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = timed_launch(ctx, AIHOST_KERNEL_KV8_APPEND, st, [&] { return launch_kv8_read(a, st); });
  return e == cudaSuccess ? AIHOST_OK : cuda_fail(e, "8-bit read launch");
}

aihost_status aihost_kv8_workspace_size(const aihost_kv8_desc* desc, int32_t batch, int32_t n_tokens, int32_t max_new,
                                        int32_t max_kv, size_t* out_bytes) {
  if (!out_bytes) return fail(AIHOST_EINVAL, "out_bytes is NULL");
  Resolved r;
  aihost_status s = check_kv8(desc, &r);
  if (s == AIHOST_OK) s = check_sizes(batch, n_tokens, max_new, max_kv);
  if (s != AIHOST_OK) return s;
  *out_bytes = make_plan(desc, r, false, batch, n_tokens, max_new, max_kv, current_sms()).scratch(r.g);
  return AIHOST_OK;
}

aihost_status aihost_kv8_plan(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, int32_t batch, int32_t n_tokens,
                              int32_t max_new, int32_t max_kv, size_t* out_bytes, int32_t* out_kernel) {
  return tell_plan(ctx, desc, false, batch, n_tokens, max_new, max_kv, out_bytes, out_kernel);
}
aihost_status aihost_kv8_attention(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, int32_t batch, int32_t n_tokens,
                                   int32_t max_new, int32_t max_kv, const void* q, const int32_t* row_start,
                                   const int32_t* kv_len, const int32_t* block_table, const int8_t* k_pool,
                                   const int8_t* v_pool, const float* k_scale, const float* v_scale,
                                   const int32_t* prefix_len, const int32_t* row_first, const float* alibi_slopes,
                                   void* out, void* stream) {
  return attention(ctx, desc, false, batch, n_tokens, max_new, max_kv, q, row_start, kv_len, block_table,
                   CachePtrs{k_pool, v_pool, k_scale, v_scale}, prefix_len, row_first, alibi_slopes, out, stream);
}

aihost_status aihost_kv4_append(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, int32_t n_tokens, const void* k_new,
                                const void* v_new, const int64_t* slots, const int32_t* positions, uint8_t* k_pool,
                                uint8_t* v_pool, void* k_range, void* v_range, void* stream) {
  if (!ctx) return fail(AIHOST_EINVAL, "ctx is NULL");
  Resolved r;
  aihost_status s = check_kv8(desc, &r);
  if (s != AIHOST_OK) return s;
  if (n_tokens < 0) return fail(AIHOST_EINVAL, "n_tokens (%d) must be >= 0", n_tokens);
  if (n_tokens == 0) return AIHOST_OK;
  if (!k_new || !v_new || !slots || !k_pool || !v_pool || !k_range || !v_range ||
      (!positions && r.rope_mode != AIHOST_ROPE_NONE))
    return fail(AIHOST_EINVAL, "every array must be non-NULL (positions may be NULL with rope_mode NONE)");
  if (!aligned(k_new, 16) || !aligned(v_new, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(k_range, 16) ||
      !aligned(v_range, 16) || !aligned(slots, 8) || !aligned(positions, 4))
    return fail(AIHOST_EINVAL, "k_new, v_new, the pools and the ranges must be 16-byte, slots 8-byte, positions 4-byte aligned");
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(AIHOST_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
  Kv4AppendArgs a;
  a.g = r.g;
  a.n_tokens = n_tokens;
  a.io_dtype = desc->io_dtype;
  a.rope_mode = r.rope_mode;
  a.token_stride = r.kv_stride;
  a.k_new = k_new;
  a.v_new = v_new;
  a.slots = slots;
  a.positions = positions;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_range = static_cast<uint32_t*>(k_range);
  a.v_range = static_cast<uint32_t*>(v_range);
  a.status = ctx->d_status;
  if (r.rope_mode != AIHOST_ROPE_NONE) a.freqs = freqs_of(ctx, desc);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = timed_launch(ctx, AIHOST_KERNEL_KV4_APPEND, st, [&] { return launch_kv4_append(a, st); });
  return e == cudaSuccess ? AIHOST_OK : cuda_fail(e, "4-bit append launch");
}

aihost_status aihost_kv4_read(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, int32_t n_rows, const int64_t* slots,
                              const uint8_t* pool, const void* range, void* out, int32_t out_dtype, void* stream) {
  if (!ctx) return fail(AIHOST_EINVAL, "ctx is NULL");
  Resolved r;
  aihost_status s = check_kv8(desc, &r);
  if (s != AIHOST_OK) return s;
  if (out_dtype != AIHOST_F32 && out_dtype != AIHOST_F16)
    return fail(AIHOST_EINVAL, "out_dtype %d must be F32 (0) or F16 (1)", out_dtype);
  if (n_rows < 0) return fail(AIHOST_EINVAL, "n_rows (%d) must be >= 0", n_rows);
  if (n_rows == 0) return AIHOST_OK;
  if (!slots || !pool || !range || !out) return fail(AIHOST_EINVAL, "slots, pool, range and out must be non-NULL");
  if (!aligned(slots, 8) || !aligned(pool, 16) || !aligned(range, 16) || !aligned(out, 16))
    return fail(AIHOST_EINVAL, "pool, range and out must be 16-byte, slots 8-byte aligned");
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(AIHOST_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
  Kv4ReadArgs a{r.g, n_rows, out_dtype, slots, pool, static_cast<const uint32_t*>(range), out, ctx->d_status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = timed_launch(ctx, AIHOST_KERNEL_KV4_APPEND, st, [&] { return launch_kv4_read(a, st); });
  return e == cudaSuccess ? AIHOST_OK : cuda_fail(e, "4-bit read launch");
}

aihost_status aihost_kv4_plan(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, int32_t batch, int32_t n_tokens,
                              int32_t max_new, int32_t max_kv, size_t* out_bytes, int32_t* out_kernel) {
  return tell_plan(ctx, desc, true, batch, n_tokens, max_new, max_kv, out_bytes, out_kernel);
}

aihost_status aihost_kv4_attention(aihost_attn_ctx* ctx, const aihost_kv8_desc* desc, int32_t batch, int32_t n_tokens,
                                   int32_t max_new, int32_t max_kv, const void* q, const int32_t* row_start,
                                   const int32_t* kv_len, const int32_t* block_table, const uint8_t* k_pool,
                                   const uint8_t* v_pool, const void* k_range, const void* v_range,
                                   const int32_t* prefix_len, const int32_t* row_first, const float* alibi_slopes,
                                   void* out, void* stream) {
  return attention(ctx, desc, true, batch, n_tokens, max_new, max_kv, q, row_start, kv_len, block_table,
                   CachePtrs{k_pool, v_pool, k_range, v_range}, prefix_len, row_first, alibi_slopes, out, stream);
}

}  // extern "C"
