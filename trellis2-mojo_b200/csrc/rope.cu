// Rotary positions over the voxel axes, alone or behind an RMS norm of every
// head: z = x / sqrt(mean(x^2) + eps) * gain, then every pair (u, v) of a
// head turns by its angle, (u cos - v sin, u sin + v cos).
//
// Pair j of axis a turns by coords[row, 1 + a] * theta^(-j / n_a). The angle
// is formed in turns (2 pi = 1) and in 64 bits and reduced to half a turn
// before it is rounded: a 32-bit angle of a position of 10^3 would already be
// off by 3e-5, and any int32 position is allowed here. With theta >= 1 a
// position turns by at most 2^31 / (2 pi) turns, whose product and frequency
// are each off by 2^-53 relative: 2^-23 turns at the farthest positions, and
// less than the rounding to f32 below 2^26.
//
// The operators move their rows once in and once out and do ~10 operations a
// value, so HBM bounds them if enough bytes are in flight and the
// instructions stay few. A CTA takes T rows; a group of lanes (a power of
// two) takes up to R heads of one row, every lane two 16-byte chunks at the
// same place of a head's two halves, which hold whole pairs in either layout.
// All loads are issued before the CTA's T x pairs sines and cosines are
// computed into shared memory, so that their latency hides behind them; a
// lane reads its pairs' once for its R heads. The arithmetic is in packed
// pairs of f32, one instruction for two values.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "entry.h"
#include "internal.h"
#include "sm100.cuh"

struct t2sc_rope {
  t2sc_ctx *ctx = nullptr;
  int device = 0;  // the context's, which may be gone when the handle is destroyed
  int head_dim = 0, layout = 0, rotated = 0;  // rotated: pairs that turn; the others stay
  double *d_turns = nullptr;                  // [rotated] turns per unit of position
  int n_axis[3] = {0, 0, 0};
};

namespace t2sc {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxHeadDim = 256;

struct RopeArgs {
  const int32_t *coords = nullptr;   // [rows, 4]
  const double *turns = nullptr;     // [rotated]
  int n0 = 0, n01 = 0, rotated = 0;  // pairs of axis 0, of axes 0 and 1, of all
  const char *in[2] = {nullptr, nullptr};
  char *out[2] = {nullptr, nullptr};
  int64_t in_stride[2] = {0, 0}, out_stride[2] = {0, 0};  // bytes
  const float *gain[2] = {nullptr, nullptr};              // [heads, head_dim]
  int64_t rows = 0;
  int heads = 0, head_dim = 0, per_row = 0;  // per_row: heads of one row, of q and k together
  float eps = 0.f, inv_dim = 0.f;
};

// cos and sin of pair p at the coordinates of one row.
__device__ __forceinline__ float2 turn_of(const RopeArgs &a, int64_t row, int p) {
  const int axis = p < a.n0 ? 0 : (p < a.n01 ? 1 : 2);
  double t = (double)a.coords[row * 4 + 1 + axis] * __ldg(a.turns + p);
  t -= rint(t);
  float s, c;
  sincospif((float)(2.0 * t), &s, &c);
  return make_float2(c, s);
}

// 16 bytes <-> packed pairs of f32.
template <int DT>
struct Chunk {
  static constexpr int kElems = DT == T2SC_DT_F32 ? 4 : 8;
  __device__ __forceinline__ static void unpack(const uint4 &u, uint64_t *f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if (DT == T2SC_DT_F32) {
      f[0] = sm100::pack_f32x2(__uint_as_float(w[0]), __uint_as_float(w[1]));
      f[1] = sm100::pack_f32x2(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (DT == T2SC_DT_BF16) {
          f[j % (kElems / 2)] = sm100::pack_f32x2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
        } else {
          const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
          f[j % (kElems / 2)] = sm100::pack_f32x2(h.x, h.y);
        }
      }
    }
  }
  __device__ __forceinline__ static uint4 pack(const uint64_t *f) {
    float v[kElems];
#pragma unroll
    for (int j = 0; j < kElems / 2; j++) sm100::unpack_f32x2(f[j], v[2 * j], v[2 * j + 1]);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (DT == T2SC_DT_F32) {
        w[j] = __float_as_uint(v[j]);
      } else if (DT == T2SC_DT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j % kElems], v[(2 * j + 1) % kElems]);
        w[j] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * j % kElems], v[(2 * j + 1) % kElems]);
        w[j] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// NORM: RMS norm and gains first. PAIRS: adjacent channels are a pair, else
// channels j and j + head_dim / 2. R: heads of a row that a group holds at
// once; `slots` groups share a row.
template <int DT, bool NORM, bool PAIRS, int R>
__global__ void __launch_bounds__(kThreads) rope_vec_kernel(const RopeArgs a, int t_rows, int lanes, int chunks, int slots) {
  constexpr int E = Chunk<DT>::kElems, H = E / 2;  // values of a chunk, packed pairs of them
  extern __shared__ float2 turn[];                 // [t_rows][pairs]
  sm100::previous_kernel_done();
  const int groups = (int)blockDim.x / lanes, gid = (int)threadIdx.x / lanes, sub = (int)threadIdx.x % lanes;
  const int64_t row0 = (int64_t)blockIdx.x * t_rows;
  const int here = (int)min((int64_t)t_rows, a.rows - row0);
  const int total = here * slots, pairs = a.head_dim / 2, half = pairs * (16 / E);
  const bool lane_live = sub < chunks;
  // the lane's pairs: H in each half of the head where adjacent channels are pairs, else E
  const int p0 = PAIRS ? sub * H : sub * E, p1 = PAIRS ? pairs / 2 + p0 : p0 + H;
  for (int base = 0; base < total; base += groups) {
    const int w = base + gid, row = w / slots, h0 = (w - row * slots) * R;
    const bool live = w < total && lane_live;
    uint4 raw[R][2];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int t = h0 + r >= a.heads, h = h0 + r - t * a.heads;
      raw[r][0] = raw[r][1] = make_uint4(0, 0, 0, 0);
      if (live && h0 + r < a.per_row) {
        const char *p = a.in[t] + (row0 + row) * a.in_stride[t] + h * 2 * half + sub * 16;
        raw[r][0] = sm100::ld_streaming(p);
        raw[r][1] = sm100::ld_streaming(p + half);
      }
    }
    if (base == 0) {
      for (int i = threadIdx.x; i < here * a.rotated; i += blockDim.x)
        turn[i / a.rotated * pairs + i % a.rotated] = turn_of(a, row0 + i / a.rotated, i % a.rotated);
      __syncthreads();
    }
    // Factors of the lane's pairs. PAIRS: (u, v) (c, c) + (v, u) (-s, s), a
    // pair to a packed value; else u (c) + v (-s) and u (s) + v (c), two pairs
    // to a packed value. Pairs that do not turn are selected away below.
    uint64_t f0[E], f1[E];
    {
      const float2 *t0 = turn + (live ? row * pairs : 0);
      float2 cs[E];
#pragma unroll
      for (int p = 0; p < E; p++) {
        const int at = p < H ? p0 + p : p1 + p - H;
        cs[p] = live && at < a.rotated ? t0[at] : make_float2(1.f, 0.f);
      }
      if (PAIRS) {
#pragma unroll
        for (int p = 0; p < E; p++) f0[p] = sm100::pack_f32x2(cs[p].x, cs[p].x), f1[p] = sm100::pack_f32x2(-cs[p].y, cs[p].y);
      } else {
#pragma unroll
        for (int p = 0; p < H; p++) {
          f0[p] = sm100::pack_f32x2(cs[2 * p].x, cs[2 * p + 1].x);
          f1[p] = sm100::pack_f32x2(cs[2 * p].y, cs[2 * p + 1].y);
          f1[H + p] = sm100::pack_f32x2(-cs[2 * p].y, -cs[2 * p + 1].y);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int t = h0 + r >= a.heads, h = h0 + r - t * a.heads;
      const bool there = live && h0 + r < a.per_row;
      uint64_t x[E];  // H of the first chunk, H of the second
      Chunk<DT>::unpack(raw[r][0], x);
      Chunk<DT>::unpack(raw[r][1], x + H);
      if (NORM) {
        uint64_t ss2 = 0;
#pragma unroll
        for (int e = 0; e < E; e++) ss2 = sm100::fma_f32x2(x[e], x[e], ss2);
        float ss, s1;
        sm100::unpack_f32x2(ss2, ss, s1);
        ss += s1;
        for (int d = lanes >> 1; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float inv = rsqrtf(ss * a.inv_dim + a.eps);
        const uint64_t inv2 = sm100::pack_f32x2(inv, inv);
        if (there) {
          const float *g = a.gain[t] + h * a.head_dim + sub * E;
#pragma unroll
          for (int q = 0; q < 2; q++)
#pragma unroll
            for (int e4 = 0; e4 < E / 4; e4++) {
              const ulonglong2 m = reinterpret_cast<const ulonglong2 *>(g + q * pairs)[e4];
              uint64_t *z = x + q * H + e4 * 2;
              z[0] = sm100::mul_f32x2(z[0], sm100::mul_f32x2(m.x, inv2));
              z[1] = sm100::mul_f32x2(z[1], sm100::mul_f32x2(m.y, inv2));
            }
        }
      }
      if (!there) continue;
      // pairs that do not turn pass through untouched, infinities and NaN too
      if (PAIRS) {
#pragma unroll
        for (int p = 0; p < E; p++) {
          float u, v;
          sm100::unpack_f32x2(x[p], u, v);
          const uint64_t y = sm100::fma_f32x2(x[p], f0[p], sm100::mul_f32x2(sm100::pack_f32x2(v, u), f1[p]));
          x[p] = (p < H ? p0 + p : p1 + p - H) < a.rotated ? y : x[p];
        }
      } else {
#pragma unroll
        for (int p = 0; p < H; p++) {
          const uint64_t u = sm100::fma_f32x2(x[p], f0[p], sm100::mul_f32x2(x[H + p], f1[H + p]));
          const uint64_t v = sm100::fma_f32x2(x[p], f1[p], sm100::mul_f32x2(x[H + p], f0[p]));
          float u0, u1, v0, v1, k0, k1, m0, m1;
          sm100::unpack_f32x2(u, u0, u1), sm100::unpack_f32x2(v, v0, v1);
          sm100::unpack_f32x2(x[p], k0, k1), sm100::unpack_f32x2(x[H + p], m0, m1);
          const bool a0 = p0 + 2 * p < a.rotated, a1 = p0 + 2 * p + 1 < a.rotated;
          x[p] = sm100::pack_f32x2(a0 ? u0 : k0, a1 ? u1 : k1);
          x[H + p] = sm100::pack_f32x2(a0 ? v0 : m0, a1 ? v1 : m1);
        }
      }
      char *p = a.out[t] + (row0 + row) * a.out_stride[t] + h * 2 * half + sub * 16;
      __stcs(reinterpret_cast<uint4 *>(p), Chunk<DT>::pack(x));
      __stcs(reinterpret_cast<uint4 *>(p + half), Chunk<DT>::pack(x + H));
    }
  }
}

template <int DT>
__device__ __forceinline__ float ld1(const char *p, int i) {
  if (DT == T2SC_DT_F32) return reinterpret_cast<const float *>(p)[i];
  if (DT == T2SC_DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
  return __half2float(reinterpret_cast<const __half *>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void st1(char *p, int i, float v) {
  if (DT == T2SC_DT_F32)
    reinterpret_cast<float *>(p)[i] = v;
  else if (DT == T2SC_DT_BF16)
    reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half *>(p)[i] = __float2half_rn(v);
}

// Any even head_dim and any element alignment: one warp a head, one pair a
// lane at a time, the whole head read before any of it is written.
template <int DT, bool NORM, bool PAIRS>
__global__ void __launch_bounds__(kThreads) rope_scalar_kernel(const RopeArgs a) {
  constexpr int P = kMaxHeadDim / 2 / 32;
  const int lane = threadIdx.x & 31;
  const int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (i >= a.rows * a.per_row) return;
  const int64_t row = i / a.per_row;
  int h = (int)(i - row * a.per_row);
  const int t = h >= a.heads;
  h -= t * a.heads;
  const int half = a.head_dim / 2, es = DT == T2SC_DT_F32 ? 4 : 2;
  const char *in = a.in[t] + row * a.in_stride[t] + (int64_t)h * a.head_dim * es;
  char *out = a.out[t] + row * a.out_stride[t] + (int64_t)h * a.head_dim * es;
  float u[P], v[P], ss = 0.f;
#pragma unroll
  for (int q = 0; q < P; q++) {
    const int p = q * 32 + lane;
    u[q] = p < half ? ld1<DT>(in, PAIRS ? 2 * p : p) : 0.f;
    v[q] = p < half ? ld1<DT>(in, PAIRS ? 2 * p + 1 : p + half) : 0.f;
    ss += u[q] * u[q] + v[q] * v[q];
  }
  if (NORM) {
    for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
  }
  const float inv = NORM ? rsqrtf(ss * a.inv_dim + a.eps) : 1.f;
#pragma unroll
  for (int q = 0; q < P; q++) {
    const int p = q * 32 + lane;
    if (p >= half) continue;
    const int iu = PAIRS ? 2 * p : p, iv = PAIRS ? 2 * p + 1 : p + half;
    if (NORM) {
      const float *g = a.gain[t] + h * a.head_dim;
      u[q] *= inv * g[iu], v[q] *= inv * g[iv];
    }
    if (p < a.rotated) {
      const float2 cs = turn_of(a, row, p);
      const float x = u[q], y = v[q];
      u[q] = x * cs.x - y * cs.y, v[q] = x * cs.y + y * cs.x;
    }
    st1<DT>(out, iu, u[q]);
    st1<DT>(out, iv, v[q]);
  }
}

template <int DT, bool NORM, bool PAIRS>
int launch(t2sc_ctx *ctx, const RopeArgs &a, std::string &err) {
  constexpr int E = Chunk<DT>::kElems;
  bool vec = a.head_dim % (2 * E) == 0;
  for (int t = 0; t < (a.per_row > a.heads ? 2 : 1); t++) {
    auto off = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
    if (off(a.in[t]) || off(a.out[t]) || a.in_stride[t] % 16 || a.out_stride[t] % 16 || (NORM && off(a.gain[t]))) vec = false;
  }
  if (vec) {
    const int chunks = a.head_dim / 2 / E;
    int lanes = 1;
    while (lanes < chunks) lanes <<= 1;
    auto go = [&](auto rc) -> int {
      constexpr int R = decltype(rc)::value;
      // Rows a CTA takes: as many as its groups hold at once; fewer when that
      // would leave SMs idle. No more threads than these rows have groups for
      // (12 heads of 128, q and k: 2 rows on 96 threads).
      const int slots = (a.per_row + R - 1) / R, row_threads = slots * lanes;
      int64_t t_rows = std::max(1, std::min(16, kThreads / row_threads));
      while (t_rows > 1 && (a.rows + t_rows - 1) / t_rows < 2 * ctx->num_sms) t_rows--;
      const int threads = (int)std::min<int64_t>(kThreads, (t_rows * row_threads + 31) / 32 * 32);
      const int64_t grid = (a.rows + t_rows - 1) / t_rows;
      const size_t smem = (size_t)t_rows * (a.head_dim / 2) * sizeof(float2);  // <= 16 x 128 x 8 bytes
      T2SC_CUDA(launch_overlapped(rope_vec_kernel<DT, NORM, PAIRS, R>, grid, threads, smem, ctx->stream, 1, a, (int)t_rows, lanes, chunks, slots),
                "rope");
      T2SC_LAUNCHED(ctx, "rope");
      return T2SC_OK;
    };
    // Heads a group holds: four (bf16 [100003, 12, 128] q and k 266 us, with
    // two 282, one 286) while that leaves threads for every SM; with fewer
    // rows fewer ([1941, 12, 128]: 12.4 us with four, 9.9 with two).
    const int64_t enough = (int64_t)1024 * ctx->num_sms;
    auto threads_with = [&](int r) { return a.rows * ((a.per_row + r - 1) / r) * lanes; };
    if (a.per_row >= 4 && threads_with(4) >= enough) return go(std::integral_constant<int, 4>());
    if (a.per_row >= 2 && threads_with(2) >= enough) return go(std::integral_constant<int, 2>());
    return go(std::integral_constant<int, 1>());
  }
  const int64_t warps = a.rows * a.per_row, grid = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (grid > INT32_MAX) return fail(ctx, T2SC_ERR_UNSUPPORTED, "rope: too many heads in one call");
  rope_scalar_kernel<DT, NORM, PAIRS><<<(unsigned)grid, kThreads, 0, ctx->stream>>>(a);
  T2SC_LAUNCHED(ctx, "rope");
  return T2SC_OK;
}

template <int DT>
int launch_dt(t2sc_ctx *ctx, const RopeArgs &a, bool norm, bool pairs, std::string &err) {
  if (norm) return pairs ? launch<DT, true, true>(ctx, a, err) : launch<DT, true, false>(ctx, a, err);
  return pairs ? launch<DT, false, true>(ctx, a, err) : launch<DT, false, false>(ctx, a, err);
}

int launch_any(t2sc_ctx *ctx, const RopeArgs &a, bool norm, bool pairs, int dtype) {
  std::string &err = ctx->last_error;
  if (dtype == T2SC_DT_F32) return launch_dt<T2SC_DT_F32>(ctx, a, norm, pairs, err);
  if (dtype == T2SC_DT_BF16) return launch_dt<T2SC_DT_BF16>(ctx, a, norm, pairs, err);
  return launch_dt<T2SC_DT_F16>(ctx, a, norm, pairs, err);
}

// Checks one input/output pair and enters it into the launch arguments.
int enter(t2sc_ctx *ctx, RopeArgs &a, int t, const void *in, int64_t in_stride, void *out, int64_t out_stride, int dtype,
          const char *what, Rows *ri, Rows *ro) {
  const int64_t width = (int64_t)a.heads * a.head_dim;
  *ri = Rows{in, in_stride, a.rows, width, dtype_size(dtype)};
  *ro = Rows{out, out_stride, a.rows, width, dtype_size(dtype)};
  if (!in || !out) return fail(ctx, T2SC_ERR_INVALID, std::string(what) + ": null buffer");
  if (!stride_ok(*ri) || !stride_ok(*ro))
    return fail(ctx, T2SC_ERR_INVALID, std::string(what) + ": a row stride must be in [heads * head_dim, 2^28]");
  if (!aligned_to_elem(*ri) || !aligned_to_elem(*ro))
    return fail(ctx, T2SC_ERR_INVALID, std::string(what) + ": a buffer is not aligned to its element type");
  if (!same_rows(*ri, *ro) && overlaps(*ri, *ro))
    return fail(ctx, T2SC_ERR_INVALID, std::string(what) + ": the output overlaps the input without being the input");
  a.in[t] = static_cast<const char *>(in), a.out[t] = static_cast<char *>(out);
  a.in_stride[t] = in_stride * dtype_size(dtype), a.out_stride[t] = out_stride * dtype_size(dtype);
  return T2SC_OK;
}

int check_coords(t2sc_ctx *ctx, const int32_t *coords, const char *what) {
  if (!coords) return fail(ctx, T2SC_ERR_INVALID, std::string(what) + ": null coords");
  if (reinterpret_cast<uintptr_t>(coords) % 4)
    return fail(ctx, T2SC_ERR_INVALID, std::string(what) + ": coords are not aligned to 4 bytes");
  return T2SC_OK;
}

void enter_rope(RopeArgs &a, const t2sc_rope *r, const int32_t *coords) {
  a.coords = coords;
  a.turns = r->d_turns;
  a.n0 = r->n_axis[0], a.n01 = r->n_axis[0] + r->n_axis[1], a.rotated = r->rotated;
}

}  // namespace
}  // namespace t2sc

using namespace t2sc;

extern "C" {

int t2sc_rope_create(t2sc_ctx *ctx, int head_dim, int pairs_x, int pairs_y, int pairs_z, double theta, int layout,
                     t2sc_rope **out) {
  if (!ctx || !out) return T2SC_ERR_INVALID;
  *out = nullptr;
  return guarded(ctx, [&]() -> int {
    if (head_dim < 2 || head_dim % 2 || head_dim > kMaxHeadDim)
      return fail(ctx, T2SC_ERR_INVALID, "rope: head_dim must be even and in [2, 256]");
    const int n[3] = {pairs_x, pairs_y, pairs_z};
    for (int i = 0; i < 3; i++)
      if (n[i] < 0 || n[i] > head_dim / 2) return fail(ctx, T2SC_ERR_INVALID, "rope: pairs of an axis must be in [0, head_dim / 2]");
    if (n[0] + n[1] + n[2] > head_dim / 2) return fail(ctx, T2SC_ERR_INVALID, "rope: the axes take more pairs than a head has");
    if (!(theta >= 1.0) || !std::isfinite(theta)) return fail(ctx, T2SC_ERR_INVALID, "rope: theta must be at least 1 and finite");
    if (layout != T2SC_ROPE_PAIRS && layout != T2SC_ROPE_HALVES) return fail(ctx, T2SC_ERR_INVALID, "rope: unknown layout");
    DeviceGuard g(ctx->device);
    CaptureTolerant relaxed;
    std::string &err = ctx->last_error;
    std::unique_ptr<t2sc_rope, int (*)(t2sc_rope *)> r(new t2sc_rope(), t2sc_rope_destroy);
    r->ctx = ctx;
    r->device = ctx->device;
    r->head_dim = head_dim;
    r->layout = layout;
    r->rotated = n[0] + n[1] + n[2];
    std::vector<double> turns;
    for (int i = 0; i < 3; i++) {
      r->n_axis[i] = n[i];
      for (int j = 0; j < n[i]; j++) turns.push_back(std::pow(theta, -(double)j / n[i]) / (2.0 * 3.14159265358979323846));
    }
    // on the context's own stream: nothing else on the device waits
    T2SC_CUDA(cudaMalloc((void **)&r->d_turns, (turns.size() + 1) * sizeof(double)), "rope frequencies");
    if (!turns.empty())
      T2SC_CUDA(cudaMemcpyAsync(r->d_turns, turns.data(), turns.size() * sizeof(double), cudaMemcpyHostToDevice, ctx->own_stream),
                "rope frequencies");
    T2SC_CUDA(cudaStreamSynchronize(ctx->own_stream), "rope frequencies");
    *out = r.release();
    return T2SC_OK;
  });
}

int t2sc_rope_destroy(t2sc_rope *r) {
  if (!r) return T2SC_OK;
  DeviceGuard g(r->device);
  CaptureTolerant relaxed;
  if (r->d_turns) cudaFree(r->d_turns);  // waits for the kernels that read it, on whatever stream
  delete r;
  return T2SC_OK;
}

int t2sc_rope_apply_device(t2sc_rope *rope, const int32_t *coords, const void *x, int64_t x_stride, void *y,
                           int64_t y_stride, int64_t rows, int heads, int dtype) {
  if (!rope) return T2SC_ERR_INVALID;
  t2sc_ctx *ctx = rope->ctx;
  return guarded(ctx, [&]() -> int {
    if (rows < 0 || rows > INT32_MAX) return fail(ctx, T2SC_ERR_INVALID, "rope: rows must be in [0, 2^31)");
    if (heads < 1 || heads > 4096) return fail(ctx, T2SC_ERR_INVALID, "rope: heads must be in [1, 4096]");
    if (!dtype_known(dtype)) return fail(ctx, T2SC_ERR_INVALID, "rope: unknown dtype");
    if (rows == 0) return T2SC_OK;
    RopeArgs a;
    a.rows = rows, a.heads = a.per_row = heads, a.head_dim = rope->head_dim;
    Rows ri, ro;
    T2SC_TRY(check_coords(ctx, coords, "rope"));
    T2SC_TRY(enter(ctx, a, 0, x, x_stride, y, y_stride, dtype, "rope", &ri, &ro));
    if (overlaps(ro, Rows{coords, 4, rows, 4, 4})) return fail(ctx, T2SC_ERR_INVALID, "rope: the output overlaps coords");
    enter_rope(a, rope, coords);
    T2SC_TRY(earlier_failure(ctx));
    DeviceGuard g(ctx->device);
    return launch_any(ctx, a, false, rope->layout == T2SC_ROPE_PAIRS, dtype);
  });
}

int t2sc_qk_norm_rope_device(t2sc_ctx *ctx, t2sc_rope *rope, const int32_t *coords, const void *q, int64_t q_stride,
                             const void *k, int64_t k_stride, const float *gain_q, const float *gain_k, void *q_out,
                             int64_t q_out_stride, void *k_out, int64_t k_out_stride, int64_t rows, int heads,
                             int head_dim, float eps, int dtype) {
  if (!ctx) return T2SC_ERR_INVALID;
  return guarded(ctx, [&]() -> int {
    if (rows < 0 || rows > INT32_MAX) return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: rows must be in [0, 2^31)");
    if (heads < 1 || heads > 4096) return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: heads must be in [1, 4096]");
    if (head_dim < 2 || head_dim % 2 || head_dim > kMaxHeadDim)
      return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: head_dim must be even and in [2, 256]");
    if (!dtype_known(dtype)) return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: unknown dtype");
    if (!(eps > 0.f) || !std::isfinite(eps)) return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: eps must be positive and finite");
    if (rope && (rope->ctx != ctx || rope->head_dim != head_dim))
      return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: rope handle of another context or head_dim");
    if ((k == nullptr) != (k_out == nullptr)) return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: k and k_out must both be set or both NULL");
    if (rows == 0) return T2SC_OK;
    RopeArgs a;
    a.rows = rows, a.heads = heads, a.head_dim = head_dim, a.per_row = k ? 2 * heads : heads;
    a.eps = eps, a.inv_dim = 1.0f / (float)head_dim;
    Rows qi, qo, ki, ko;
    const char *what = "qk_norm_rope";
    T2SC_TRY(enter(ctx, a, 0, q, q_stride, q_out, q_out_stride, dtype, what, &qi, &qo));
    if (k) T2SC_TRY(enter(ctx, a, 1, k, k_stride, k_out, k_out_stride, dtype, what, &ki, &ko));
    if (k && (overlaps(qo, ki) || overlaps(ko, qi) || overlaps(qo, ko)))
      return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: an output overlaps the other input or output");
    const float *gains[2] = {gain_q, gain_k};
    for (int t = 0; t < (k ? 2 : 1); t++) {
      const Rows gr{gains[t], head_dim, heads, head_dim, 4};
      if (!gains[t] || !aligned_to_elem(gr)) return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: null or unaligned gain");
      if (overlaps(qo, gr) || (k && overlaps(ko, gr))) return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: an output overlaps a gain");
      a.gain[t] = gains[t];
    }
    if (rope) {
      T2SC_TRY(check_coords(ctx, coords, what));
      const Rows cr{coords, 4, rows, 4, 4};
      if (overlaps(qo, cr) || (k && overlaps(ko, cr))) return fail(ctx, T2SC_ERR_INVALID, "qk_norm_rope: an output overlaps coords");
      enter_rope(a, rope, coords);
    }
    T2SC_TRY(earlier_failure(ctx));
    DeviceGuard g(ctx->device);
    return launch_any(ctx, a, true, !rope || rope->layout == T2SC_ROPE_PAIRS, dtype);
  });
}

}  // extern "C"
