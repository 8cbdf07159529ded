// The context behind the C ABI and what its entry points share: error text,
// the device guard, workspaces by stream. Host side only.
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "../../include/c4s_sampling.h"
#include "c4s_internal.h"
#include "c4s_pool.hpp"

// The pools' runtime.
struct HipRt {
  using Stream = hipStream_t;
  using Event = hipEvent_t;
  hipError_t err = hipSuccess;   // of the last call
  bool ok(hipError_t e) {
    err = e;
    return e == hipSuccess;
  }
  // While any stream of the thread is being captured, hipMalloc is refused
  // (and the capture lost) unless the thread asks for the relaxed mode.
  bool alloc(void** p, size_t bytes) {
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    if (!ok(hipThreadExchangeStreamCaptureMode(&mode))) return false;
    const hipError_t e = hipMalloc(p, bytes);
    (void)hipThreadExchangeStreamCaptureMode(&mode);
    return ok(e);
  }
  bool release(void* p) { return ok(hipFree(p)); }
  bool create(hipEvent_t* e) { return ok(hipEventCreateWithFlags(e, hipEventDisableTiming)); }
  bool destroy(hipEvent_t e) { return ok(hipEventDestroy(e)); }
  bool record(hipEvent_t e, hipStream_t s) { return ok(hipEventRecord(e, s)); }
  bool wait(hipStream_t s, hipEvent_t e) { return ok(hipStreamWaitEvent(s, e, 0)); }
};

// That of a pool whose workspaces begin zeroed: by a kernel on a stream of its
// own, which is never captured.
struct ZeroedRt : HipRt {
  hipStream_t stream = nullptr;
  bool alloc(void** p, size_t bytes) {
    if (!HipRt::alloc(p, bytes)) return false;
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    bool fine = ok(hipThreadExchangeStreamCaptureMode(&mode));
    if (fine) {
      fine = ok(c4s::launch_zero(*p, bytes < c4s::kLayerZeroed ? bytes : c4s::kLayerZeroed, stream)) &&
             ok(hipStreamSynchronize(stream));
      const hipError_t e = err;
      (void)hipThreadExchangeStreamCaptureMode(&mode);
      err = e;
    }
    if (!fine) {
      const hipError_t e = err;
      (void)hipFree(*p);
      *p = nullptr;
      err = e;
    }
    return fine;
  }
};

struct c4s_ctx {
  int device = 0;
  std::string err;
  hipStream_t host_stream = nullptr;  // used by the synchronous host helpers
  void* ws = nullptr;                 // stream: exact steps' key buffers
  size_t ws_bytes = 0;
  c4s::StreamPool<HipRt> rows_ws;     // large-vocabulary rows: slices, lists, exact-pass keys
  c4s::StreamPool<HipRt> logits_ws;   // LM head + sample: logits when the caller gives none
  c4s::StreamPool<ZeroedRt> layer_ws; // decoder layer: counters, split sums' parts
  // host-helper staging: pinned host memory that the device maps
  void* hstage = nullptr;
  size_t hstage_bytes = 0;
  // two-phase stream: summaries of one chunk of steps, per-row carried state
  void* sum_ws = nullptr;
  size_t sum_bytes = 0;
  void* state_ws = nullptr;
  size_t state_bytes = 0;
  // second stream: the two fast chain kernels run side by side
  hipStream_t side = nullptr;
  // third stream: the scan of the next chunk of steps beside the chain of this one
  hipStream_t scan_s = nullptr;
  hipEvent_t ev_start = nullptr;
  // by summary buffer: its scan done, its list chain done, its full-vocabulary chain done
  hipEvent_t ev_scan[3] = {nullptr, nullptr, nullptr}, ev_chain[3] = {nullptr, nullptr, nullptr};
  hipEvent_t ev_side[3] = {nullptr, nullptr, nullptr};
  // Overlapped stream: the scan and the chains on disjoint sets of CUs (half
  // of every 32 CUs for the chains), created at first use.
  int n_cus = 0;
  bool cu_split_tried = false;
  hipStream_t scan_m = nullptr, chain_m = nullptr, side_m = nullptr;
  hipEvent_t ev_done = nullptr;
  // step segments of the pipelined row chain (rows without penalty)
  void* segres = nullptr;
  size_t segres_bytes = 0;
  // this device's address of the no-allocation entry point's static scratch
  // (null when the runtime could not give it)
  void* noalloc = nullptr;
  // The speculative chains' give-up report: a word of pinned host memory that
  // the kernels write through its device address, and the polls a bounded
  // wait makes before it gives up.
  volatile uint32_t* status_host = nullptr;
  uint32_t* status_dev = nullptr;
  int spin_max = c4s::kSpinMaxDefault;
};

namespace c4s {

inline int fail(c4s_ctx* ctx, int code, const std::string& msg) {
  if (ctx) ctx->err = msg;
  return code;
}

inline int hip_fail(c4s_ctx* ctx, hipError_t e, const char* what) {
  return fail(ctx, C4S_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}

struct DeviceGuard {
  int prev = -1;
  hipError_t err = hipSuccess;
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != dev) err = hipSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
  }
};

inline bool is_capturing(hipStream_t s) {
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(s, &cap) == hipSuccess && cap != hipStreamCaptureStatusNone;
}

// The stream's workspace of `pool` for a call about to be queued on `s`.
template <class Rt>
int pool_take(c4s_ctx* ctx, c4s::StreamPool<Rt>& pool, hipStream_t s, size_t need, const char* what, void** out) {
  switch (pool.take(s, is_capturing(s), need, out)) {
    case c4s::PoolResult::kOk: return C4S_OK;
    case c4s::PoolResult::kWouldGrow:
      return fail(ctx, C4S_EINVAL, std::string(what) +
                                       ": the workspace would grow during graph capture; make one call of "
                                       "this shape (or larger) outside the capture first");
    default: break;
  }
  const hipError_t e = pool.runtime().err;
  return e == hipErrorOutOfMemory ? fail(ctx, C4S_ENOMEM, std::string(what) + ": out of memory")
                                  : hip_fail(ctx, e, what);
}

}  // namespace c4s
