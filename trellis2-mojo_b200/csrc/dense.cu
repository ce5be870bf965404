// Dense linear over token rows with its epilogue in the product:
//   y[r, o] = act(sum_i x[r, i] * w[o, i] + bias[o]) + residual[r, o]
// act: none, SiLU or the tanh form of GELU. Sums and the epilogue are in f32;
// the result is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dense.h"
#include "entry.h"
#include "internal.h"

namespace t2sc {
namespace {

template <int DT>
__device__ __forceinline__ float ld1(const char *p, int64_t i) {
  if (DT == T2SC_DT_F32) return reinterpret_cast<const float *>(p)[i];
  if (DT == T2SC_DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
  return __half2float(reinterpret_cast<const __half *>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void st1(char *p, int64_t i, float v) {
  if (DT == T2SC_DT_F32)
    reinterpret_cast<float *>(p)[i] = v;
  else if (DT == T2SC_DT_BF16)
    reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half *>(p)[i] = __float2half_rn(v);
}

// CUDA-core product for every type, size, stride and alignment: 64 x 64
// outputs a CTA, 4 x 4 a thread, the K axis in steps of 16 through shared
// memory. f32 runs here (exact f32 products); the 16-bit types only where
// rows are not 16-byte aligned, which the TMA loads of the tensor-core kernel
// need.
constexpr int kBM = 64, kBN = 64, kBK = 16;

template <int DT>
__global__ void __launch_bounds__(256) dense_simt_kernel(const DenseArgs a) {
  __shared__ float xs[kBK][kBM + 4], ws[kBK][kBN + 4];
  const int tid = threadIdx.x, tr = tid / 16 * 4, tc = tid % 16 * 4;
  const unsigned row_tiles = (unsigned)((a.rows + kBM - 1) / kBM);  // fastest
  const int64_t row0 = (int64_t)(blockIdx.x % row_tiles) * kBM;
  const int col0 = (int)(blockIdx.x / row_tiles) * kBN;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < a.ci; k0 += kBK) {
    for (int i = tid; i < kBM * kBK; i += 256) {
      const int r = i / kBK, k = i % kBK;
      xs[k][r] = (row0 + r < a.rows && k0 + k < a.ci) ? ld1<DT>(a.x, (row0 + r) * a.ldx + k0 + k) : 0.f;
      ws[k][r] = (col0 + r < a.co && k0 + k < a.ci) ? ld1<DT>(a.w, (col0 + r) * a.ldw + k0 + k) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kBK; k++) {
      float xv[4], wv[4];
#pragma unroll
      for (int i = 0; i < 4; i++) xv[i] = xs[k][tr + i], wv[i] = ws[k][tc + i];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] += xv[i] * wv[j];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t r = row0 + tr + i;
      const int o = col0 + tc + j;
      if (r >= a.rows || o >= a.co) continue;
      float v = acc[i][j] + (a.bias ? __ldg(a.bias + o) : 0.f);
      v = DT == T2SC_DT_F32 ? activate_f32(v, a.act) : activate(v, a.act);
      if (a.res) v += ld1<DT>(a.res, r * a.ldr + o);
      st1<DT>(a.y, r * a.ldy + o, v);
    }
}

}  // namespace

int dense_simt(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err) {
  const int64_t tiles = ((a.rows + kBM - 1) / kBM) * ((a.co + kBN - 1) / kBN);
  if (tiles > INT32_MAX) return fail(ctx, T2SC_ERR_UNSUPPORTED, "dense_linear: too many outputs in one call");
  const unsigned grid = (unsigned)tiles;
  if (dtype == T2SC_DT_F32)
    dense_simt_kernel<T2SC_DT_F32><<<grid, 256, 0, ctx->stream>>>(a);
  else if (dtype == T2SC_DT_BF16)
    dense_simt_kernel<T2SC_DT_BF16><<<grid, 256, 0, ctx->stream>>>(a);
  else
    dense_simt_kernel<T2SC_DT_F16><<<grid, 256, 0, ctx->stream>>>(a);
  T2SC_LAUNCHED(ctx, "dense_linear");
  return T2SC_OK;
}

}  // namespace t2sc

using namespace t2sc;

extern "C" int t2sc_dense_linear_device(t2sc_ctx *ctx, const void *x, int64_t x_stride, const void *w, int64_t w_stride,
                                        const float *bias, const void *residual, int64_t residual_stride, void *y,
                                        int64_t y_stride, int64_t rows, int co, int ci, int flags, int dtype) {
  if (!ctx) return T2SC_ERR_INVALID;
  return guarded(ctx, [&]() -> int {
    if (rows < 0 || rows > INT32_MAX) return fail(ctx, T2SC_ERR_INVALID, "dense_linear: rows must be in [0, 2^31)");
    if (co < 1 || ci < 1 || co > kMaxStride || ci > kMaxStride)
      return fail(ctx, T2SC_ERR_INVALID, "dense_linear: co and ci must be in [1, 2^28]");
    if (!dtype_known(dtype)) return fail(ctx, T2SC_ERR_INVALID, "dense_linear: unknown dtype");
    if (flags & ~(T2SC_SILU | T2SC_GELU | T2SC_RESIDUAL)) return fail(ctx, T2SC_ERR_INVALID, "dense_linear: unknown flags");
    if ((flags & T2SC_SILU) && (flags & T2SC_GELU)) return fail(ctx, T2SC_ERR_INVALID, "dense_linear: SILU and GELU exclude each other");
    if (((flags & T2SC_RESIDUAL) != 0) != (residual != nullptr))
      return fail(ctx, T2SC_ERR_INVALID, "dense_linear: the RESIDUAL flag and residual go together");
    if (rows == 0) return T2SC_OK;
    if (!x || !w || !y) return fail(ctx, T2SC_ERR_INVALID, "dense_linear: null buffer");
    const int es = dtype_size(dtype);
    const Rows rx{x, x_stride, rows, ci, es}, rw{w, w_stride, co, ci, es}, ry{y, y_stride, rows, co, es},
        rb{bias, co, bias ? 1 : 0, co, 4}, rr{residual, residual_stride, residual ? rows : 0, co, es};
    for (const Rows *r : {&rx, &rw, &ry, &rr}) {
      if (!stride_ok(*r)) return fail(ctx, T2SC_ERR_INVALID, "dense_linear: a row stride must be in [row width, 2^28]");
      if (!aligned_to_elem(*r)) return fail(ctx, T2SC_ERR_INVALID, "dense_linear: a buffer is not aligned to its element type");
    }
    if (!aligned_to_elem(rb)) return fail(ctx, T2SC_ERR_INVALID, "dense_linear: bias is not aligned to 4 bytes");
    if (overlaps(ry, rx) || overlaps(ry, rw) || overlaps(ry, rb))
      return fail(ctx, T2SC_ERR_INVALID, "dense_linear: y overlaps x, w or bias");
    if (residual && !same_rows(ry, rr) && overlaps(ry, rr))
      return fail(ctx, T2SC_ERR_INVALID, "dense_linear: y overlaps residual without being residual");
    DenseArgs a;
    a.x = static_cast<const char *>(x), a.w = static_cast<const char *>(w), a.bias = bias;
    a.res = static_cast<const char *>(residual), a.y = static_cast<char *>(y);
    a.ldx = x_stride, a.ldw = w_stride, a.ldr = residual_stride, a.ldy = y_stride;
    a.rows = rows, a.co = co, a.ci = ci;
    a.act = flags & (T2SC_SILU | T2SC_GELU);
    T2SC_TRY(earlier_failure(ctx));
    DeviceGuard g(ctx->device);
    if (dense_rows_takes(a, dtype)) return dense_rows(ctx, a, dtype, ctx->last_error);
    if (dense_skinny_takes(ctx, a, dtype)) return dense_skinny(ctx, a, dtype, ctx->last_error);
    return dense_tc_takes(a, dtype) ? dense_tc(ctx, a, dtype, ctx->last_error) : dense_simt(ctx, a, dtype, ctx->last_error);
  });
}
