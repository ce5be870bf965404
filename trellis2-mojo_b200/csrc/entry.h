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

// Clusters of 1 to MAX CTAs, one CTA an SM, that a device runs at once; 0: not
// known. Asked for once per device and kernel (the query counts one CTA of a
// kernel with tensor memory an SM, where two run).
template <int MAX>
struct Clusters {
  std::atomic<int> known{0};
  int at_once[MAX + 1] = {};
};

template <int MAX, class K>
int clusters_at_once(t2sc_ctx *ctx, K kernel, int threads, size_t smem, Clusters<MAX> (&table)[64], const int **out, std::string &err) {
  Clusters<MAX> &t = table[ctx->device & 63];
  if (!t.known.load(std::memory_order_acquire)) {
    T2SC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "shared memory size");
    if (MAX > 8) T2SC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cluster size");
    for (int n = 1; n <= MAX; n++) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(n * 1024), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = n, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at, cfg.numAttrs = 1;
      int count = 0;
      if (cudaOccupancyMaxActiveClusters(&count, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        count = 0;
      }
      t.at_once[n] = count;
    }
    t.known.store(1, std::memory_order_release);
  }
  *out = t.at_once;
  return T2SC_OK;
}

// Launches a kernel that begins while the one before it on the stream ends
// (see next_kernel_may_start), in clusters of `cluster` CTAs.
template <class A, class... Args>
cudaError_t launch_overlapped(void (*kernel)(A, Args...), int64_t grid, int threads, size_t smem, cudaStream_t stream, int cluster,
                              const A &first, Args... rest) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid), cfg.blockDim = dim3((unsigned)threads), cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cudaLaunchAttribute at[2] = {};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, first, rest...);
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
