// Dense linear of a few rows: y = act(x @ w^T + bias) + residual for at most
// kMaxRows rows of a 16-bit type.
//
// The weight is read once, 2 co ci bytes against 2 rows co ci operations: HBM
// bounds it (L2 where the weight is still there), so the kernel's work is to
// keep loads in flight. A warp takes kOut outputs and a slice of the K axis;
// its lanes read 16-byte chunks of the kOut weight rows, kUnroll K blocks of
// 256 elements at a time, all loads issued before the first product. The
// CTA's 8 warps split into output groups x K slices (as many slices as it
// takes to fill the SMs) and add their f32 sums through shared memory in a
// fixed order. x comes from L1 as packed 16-bit chunks.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dense.h"
#include "entry.h"
#include "internal.h"
#include "sm100.cuh"

namespace t2sc {
namespace {

constexpr int kMaxRows = 2, kWarps = 8, kOut = 4;

template <int DT>
__device__ __forceinline__ float ld16(const char *p, int64_t i) {
  if (DT == T2SC_DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
  return __half2float(reinterpret_cast<const __half *>(p)[i]);
}

// R: rows held (>= a.rows). slices: K slices, a divisor of 8.
template <int DT, int R, int UNROLL>
__global__ void __launch_bounds__(32 * kWarps) dense_rows_kernel(const DenseArgs a, int slices) {
  __shared__ float sums[kWarps][R][kOut];
  sm100::previous_kernel_done();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = warp % slices, groups = kWarps / slices;
  const int o0 = ((int)blockIdx.x * groups + warp / slices) * kOut;
  const int blocks = (a.ci + 255) / 256;                     // K blocks of 32 lanes x 8 elements
  const int per = (blocks + slices - 1) / slices, k_first = slice * per, k_last = min(blocks, k_first + per);
  const uint4 *w[kOut], *x[R];
#pragma unroll
  for (int o = 0; o < kOut; o++) w[o] = reinterpret_cast<const uint4 *>(a.w + (int64_t)min(o0 + o, a.co - 1) * a.ldw * 2) + lane;
#pragma unroll
  for (int r = 0; r < R; r++) x[r] = reinterpret_cast<const uint4 *>(a.x + min((int64_t)r, a.rows - 1) * a.ldx * 2) + lane;
  float acc[R][kOut] = {};
  const int chunks = a.ci / 8;  // ci % 8 == 0
  for (int kb = k_first; kb < k_last; kb += UNROLL) {
    uint4 wr[UNROLL][kOut];
#pragma unroll
    for (int i = 0; i < UNROLL; i++) {
      const bool in = kb + i < k_last && (kb + i) * 32 + lane < chunks;
#pragma unroll
      for (int o = 0; o < kOut; o++) wr[i][o] = in ? w[o][(kb + i) * 32] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < UNROLL; i++) {
      const bool in = kb + i < k_last && (kb + i) * 32 + lane < chunks;
      float wf[kOut][8];
#pragma unroll
      for (int o = 0; o < kOut; o++) unpack8<DT>(wr[i][o], wf[o]);
#pragma unroll
      for (int r = 0; r < R; r++) {
        float xf[8];
        unpack8<DT>(in ? x[r][(kb + i) * 32] : make_uint4(0, 0, 0, 0), xf);
#pragma unroll
        for (int o = 0; o < kOut; o++)
#pragma unroll
          for (int j = 0; j < 8; j++) acc[r][o] += xf[j] * wf[o][j];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int o = 0; o < kOut; o++) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) acc[r][o] += __shfl_xor_sync(0xffffffffu, acc[r][o], d);
    }
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int o = 0; o < kOut; o++) sums[warp][r][o] = acc[r][o];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < groups * R * kOut; i += 32 * kWarps) {
    const int o = i % kOut, g = i / kOut % groups, r = i / (kOut * groups);
    const int col = ((int)blockIdx.x * groups + g) * kOut + o;
    if (r >= a.rows || col >= a.co) continue;
    float v = 0.f;
    for (int s = 0; s < slices; s++) v += sums[g * slices + s][r][o];
    if (a.bias) v += a.bias[col];
    v = activate(v, a.act);
    if (a.res) v += ld16<DT>(a.res, r * a.ldr + col);
    if (DT == T2SC_DT_BF16)
      reinterpret_cast<__nv_bfloat16 *>(a.y)[r * a.ldy + col] = __float2bfloat16_rn(v);
    else
      reinterpret_cast<__half *>(a.y)[r * a.ldy + col] = __float2half_rn(v);
  }
}

template <int DT>
int launch(t2sc_ctx *ctx, const DenseArgs &a, std::string &err) {
  const int out_groups = (a.co + kOut - 1) / kOut, blocks = (a.ci + 255) / 256;
  // K slices until there are 16 warps an SM, at least two K blocks a slice
  int slices = 1;
  while (slices < kWarps && out_groups * slices < 16 * ctx->num_sms && blocks >= 4 * slices) slices *= 2;
  const int grid = (out_groups + kWarps / slices - 1) / (kWarps / slices);
  auto kernel = a.rows == 1 ? dense_rows_kernel<DT, 1, 3> : dense_rows_kernel<DT, 2, 2>;
  T2SC_CUDA(launch_overlapped(kernel, grid, 32 * kWarps, 0, ctx->stream, 1, a, slices), "dense_linear");
  T2SC_LAUNCHED(ctx, "dense_linear");
  return T2SC_OK;
}

}  // namespace

bool dense_rows_takes(const DenseArgs &a, int dtype) { return dense_tc_takes(a, dtype) && a.rows <= kMaxRows && a.ci % 8 == 0; }

int dense_rows(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err) {
  return dtype == T2SC_DT_BF16 ? launch<T2SC_DT_BF16>(ctx, a, err) : launch<T2SC_DT_F16>(ctx, a, err);
}

}  // namespace t2sc
