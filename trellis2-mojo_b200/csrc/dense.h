// Launch arguments and epilogue arithmetic of the dense linear kernels.
#pragma once
#include <stdint.h>

#include <string>

#include "../../include/t2sc.h"
#include "epilogue.cuh"

struct t2sc_ctx;

namespace t2sc {

struct DenseArgs {
  const char *x = nullptr, *w = nullptr, *res = nullptr;
  const float *bias = nullptr;
  char *y = nullptr;
  int64_t ldx = 0, ldw = 0, ldr = 0, ldy = 0;  // elements
  int64_t rows = 0;
  int co = 0, ci = 0, act = 0;
};

// v / (1 + e^-v) and 0.5 v (1 + tanh(u)) = v / (1 + e^(-2u)), u = sqrt(2/pi)
// (v + 0.044715 v^3): one exponential, and no cancellation in the negative
// tail. The exponential may become infinite: any finite v over it is 0, the
// limit of both, however large v is. In f32 for results of 16 bits, whose half
// step of 2^-8 or 2^-11 the quick exponential and division (2^-17 together) stay
// far below; f32 results take activate_f32.
__device__ __forceinline__ float silu_any(float v) { return __fdividef(v, 1.0f + __expf(-v)); }
__device__ __forceinline__ float gelu_tanh(float v) {
  const float u2 = v * (1.5957691216057308f + 0.07135481627f * v * v);
  return __fdividef(v, 1.0f + __expf(-u2));
}

__device__ __forceinline__ float activate(float v, int act) {
  if (act & T2SC_SILU) return silu_any(v);
  if (act & T2SC_GELU) return gelu_tanh(v);
  return v;
}

__device__ __forceinline__ float activate_f32(float v, int act) {
  if (act & T2SC_SILU) return v / (1.0f + expf(-v));
  if (act & T2SC_GELU) return v / (1.0f + expf(-v * (1.5957691216057308f + 0.07135481627f * v * v)));
  return v;
}

// 16-bit rows that start on 16 bytes (what TMA needs of x and w).
bool dense_tc_takes(const DenseArgs &a, int dtype);
int dense_tc(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err);
// What its best tile shape (*best) is expected to take.
double dense_tc_us(t2sc_ctx *ctx, const DenseArgs &a, int *best);
// Such rows, few of them, or few tiles of outputs over a long K axis.
bool dense_skinny_takes(t2sc_ctx *ctx, const DenseArgs &a, int dtype);
int dense_skinny(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err);
// At most 2 such rows, ci a multiple of 8.
bool dense_rows_takes(const DenseArgs &a, int dtype);
int dense_rows(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err);
int dense_simt(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err);

}  // namespace t2sc
