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

// Called before work on `st` that is given the context's scratch: what a graph holds is not freed when the
// scratch grows.
inline cudaError_t note_scratch_use(aihost_attn_ctx* ctx, cudaStream_t st) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  const cudaError_t e = cudaStreamIsCapturing(st, &status);
  if (e == cudaSuccess && status != cudaStreamCaptureStatusNone) ctx->scratch_captured = true;
  return e;
}

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
