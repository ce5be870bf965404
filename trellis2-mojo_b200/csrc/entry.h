// Helpers shared by the C-ABI entry points: the device guard, the error
// path, the exception barrier and the checks of strided device buffers.
#pragma once
#include <atomic>
#include <new>
#include <string>

#include "internal.h"

namespace t2sc {

// Makes the context's device current for the duration of a call and
// restores the caller's device afterwards.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

// Allows this thread's allocations and frees while some stream is being
// captured into a graph (a handle that is made, or dropped by a garbage
// collector, meanwhile). The captured stream is not touched.
struct CaptureTolerant {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  CaptureTolerant() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~CaptureTolerant() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

inline int fail(t2sc_ctx *ctx, int code, const std::string &msg) {
  if (ctx) ctx->last_error = msg;
  return code;
}

#define T2SC_TRY(expr)                   \
  do {                                   \
    int _rc = (expr);                    \
    if (_rc != T2SC_OK) return _rc;      \
  } while (0)

// Runs an entry point's body; C++ exceptions never cross the C ABI.
template <class F>
int guarded(t2sc_ctx *ctx, F &&body) {
  bool oom = false;
  try {
    return body();
  } catch (const std::bad_alloc &) {
    oom = true;
  } catch (...) {
  }
  try {
    return oom ? fail(ctx, T2SC_ERR_OOM, "host allocation failed") : fail(ctx, T2SC_ERR_INVALID, "unexpected exception");
  } catch (...) {  // no memory for the message either
    return oom ? T2SC_ERR_OOM : T2SC_ERR_INVALID;
  }
}

// Lets `kernel` use `bytes` of dynamic shared memory, once per device.
template <class K>
int allow_smem(t2sc_ctx *ctx, K kernel, int bytes, std::atomic<uint64_t> &done, std::string &err) {
  const uint64_t bit = ctx->device < 64 ? uint64_t(1) << ctx->device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return T2SC_OK;
  T2SC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "shared memory size");
  done.fetch_or(bit, std::memory_order_relaxed);
  return T2SC_OK;
}

inline bool dtype_known(int dtype) { return dtype == T2SC_DT_F32 || dtype == T2SC_DT_F16 || dtype == T2SC_DT_BF16; }
inline int dtype_size(int dtype) { return dtype == T2SC_DT_F32 ? 4 : 2; }

// `rows` rows of `width` elements, `stride` elements apart.
struct Rows {
  const void *p = nullptr;
  int64_t stride = 0, rows = 0, width = 0;
  int elem = 2;
  int64_t bytes() const { return rows > 0 ? ((rows - 1) * stride + width) * elem : 0; }
};

constexpr int64_t kMaxStride = int64_t(1) << 28;  // elements; (2^31 rows) x (2^28) x 4 bytes stays below 2^63

inline bool stride_ok(const Rows &r) { return r.rows <= 1 || (r.stride >= r.width && r.stride <= kMaxStride); }

inline bool aligned_to_elem(const Rows &r) { return reinterpret_cast<uintptr_t>(r.p) % r.elem == 0; }

// Whether any element of `a` can also be one of `b`. Rows interleaved in one
// packed buffer (equal strides, column windows that do not meet) are apart;
// buffers of different strides are apart only if their address ranges are.
inline bool overlaps(const Rows &a, const Rows &b) {
  if (a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa + a.bytes() <= pb || pb + b.bytes() <= pa) return false;
  if (a.stride != b.stride || a.elem != b.elem) return true;
  const int64_t step = a.stride * a.elem;
  if (step <= 0) return true;
  int64_t d = (int64_t)(pb - pa) % step;  // where b's window starts inside a's row
  if (d < 0) d += step;
  return d < a.width * a.elem || d + b.width * b.elem > step;
}

inline bool same_rows(const Rows &a, const Rows &b) { return a.p == b.p && (a.rows <= 1 || a.stride == b.stride); }

}  // namespace t2sc
