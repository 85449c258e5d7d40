// ctx.h — the context behind aihost_attn_ctx and the host-side helpers that the C-ABI sources share.
#pragma once

#include <math.h>
#include <string.h>

#include <mutex>
#include <utility>
#include <vector>

#include "../../include/aihost_attn.h"
#include "kernels.h"

// Per-kernel-kind device-time accumulator (events recorded around each launch while enabled).
struct ProfSlot {
  std::vector<std::pair<cudaEvent_t, cudaEvent_t>> pending;
  int64_t launches = 0;
  double total_ms = 0.0;
};

struct aihost_attn_ctx {
  int32_t device = 0;
  int32_t num_sms = 148;
  int32_t* d_status = nullptr;
  void* scratch = nullptr;
  size_t scratch_bytes = 0;
  bool scratch_captured = false;   // a captured call holds the scratch's address
  std::vector<void*> outgrown;     // earlier scratch that captured calls hold: kept with the context
  bool shared_used = false;            // the scratch or the counters have been used,
  unsigned long long shared_stream = 0;  // last on the stream of this id;
  cudaEvent_t shared_done = nullptr;   // since a second stream came: after the last use
  unsigned long long* counters = nullptr;  // fused split merge: epoch-tagged arrival counts
  uint32_t epoch = 0;
  uint32_t* kv8_counters = nullptr;  // page map's ticket, then the 8-bit attention's arrival counts
  aihost::RopeFreqs freqs;                   // of (freqs_theta, freqs_dim), for the 8-bit cache's calls
  float freqs_theta = 0.0f;
  int32_t freqs_dim = 0;
  bool profiling = false;
  std::mutex prof_mu;
  ProfSlot prof[AIHOST_KERNEL_COUNT];
  std::vector<cudaEvent_t> event_pool;
};

namespace aihost {

aihost_status api_fail(aihost_status st, const char* fmt, ...);  // api.cu
#define fail api_fail

inline aihost_status cuda_fail(cudaError_t e, const char* what) {
  return fail(AIHOST_ECUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

// Runs `f` with the context's device current and restores the caller's device afterwards.
class DeviceGuard {
 public:
  explicit DeviceGuard(int32_t dev) {
    ok_ = cudaGetDevice(&prev_) == cudaSuccess;
    if (ok_ && prev_ != dev) ok_ = cudaSetDevice(dev) == cudaSuccess;
  }
  ~DeviceGuard() {
    int cur = -1;
    if (cudaGetDevice(&cur) == cudaSuccess && cur != prev_) cudaSetDevice(prev_);
  }
  bool ok() const { return ok_; }

 private:
  int prev_ = 0;
  bool ok_ = false;
};

// Held around the launches of a call that uses what its context has only once: the scratch and the arrival
// counters. Calls on one stream follow each other anyway. One on another stream than the last waits
// for it: the first of these for the whole device, as no event marks the call before, later ones for an
// event that every call records from then on (a context used on one stream pays for none). A captured call is
// ordered by its graph; it marks the scratch, whose address the graph holds.
class SharedUse {
 public:
  SharedUse(aihost_attn_ctx* ctx, cudaStream_t st, bool uses) : ctx_(ctx), st_(st) {
    if (uses) e_ = enter();
  }
  ~SharedUse() {
    if (entered_ && ctx_->shared_done) cudaEventRecord(ctx_->shared_done, st_);
  }
  SharedUse(const SharedUse&) = delete;
  SharedUse& operator=(const SharedUse&) = delete;
  cudaError_t error() const { return e_; }

 private:
  cudaError_t enter() {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(st_, &status);
    if (e != cudaSuccess) return e;
    if (status != cudaStreamCaptureStatusNone) {
      ctx_->scratch_captured = true;
      return cudaSuccess;
    }
    unsigned long long id = 0;  // unlike a handle, never used again for a later stream
    e = cudaStreamGetId(st_, &id);
    if (e != cudaSuccess) return e;
    if (ctx_->shared_used && id != ctx_->shared_stream) {
      if (ctx_->shared_done) {
        e = cudaStreamWaitEvent(st_, ctx_->shared_done, 0);
      } else {
        e = cudaDeviceSynchronize();
        if (e == cudaSuccess) e = cudaEventCreateWithFlags(&ctx_->shared_done, cudaEventDisableTiming);
      }
      if (e != cudaSuccess) return e;
    }
    ctx_->shared_used = true;
    ctx_->shared_stream = id;
    entered_ = true;
    return cudaSuccess;
  }

  aihost_attn_ctx* const ctx_;
  const cudaStream_t st_;
  cudaError_t e_ = cudaSuccess;
  bool entered_ = false;
};

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

inline RopeFreqs make_freqs(float theta, int32_t head_dim) {
  RopeFreqs f;
  memset(&f, 0, sizeof(f));
  for (int i = 0; i < head_dim / 2 && i < kMaxHeadDim / 2; ++i)
    f.f[i] = 1.0f / powf(theta, static_cast<float>(2 * i) / static_cast<float>(head_dim));
  return f;
}

inline cudaEvent_t take_event(aihost_attn_ctx* ctx) {
  if (!ctx->event_pool.empty()) {
    cudaEvent_t e = ctx->event_pool.back();
    ctx->event_pool.pop_back();
    return e;
  }
  cudaEvent_t e = nullptr;
  if (cudaEventCreate(&e) != cudaSuccess) return nullptr;
  return e;
}

// Launch through `fn`, bracketed by timing events on `st` when the profiler is on.
template <class F>
cudaError_t timed_launch(aihost_attn_ctx* ctx, int kind, cudaStream_t st, F&& fn) {
  if (!ctx->profiling) return fn();
  std::lock_guard<std::mutex> lk(ctx->prof_mu);
  cudaEvent_t a = take_event(ctx), b = take_event(ctx);
  if (!a || !b) return cudaErrorMemoryAllocation;
  cudaError_t e = cudaEventRecord(a, st);
  if (e != cudaSuccess) return e;
  e = fn();
  if (e != cudaSuccess) return e;
  e = cudaEventRecord(b, st);
  if (e != cudaSuccess) return e;
  ctx->prof[kind].pending.emplace_back(a, b);
  return cudaSuccess;
}

}  // namespace aihost
