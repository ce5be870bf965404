// Dense linear of few rows, or of few tiles over a long K axis, on the tensor
// cores, operands swapped: the weight's 128 output channels are the M of an
// MMA, up to 128 rows its N.
//
// With few rows the call streams the weight (HBM, or L2 where it still is
// there), so what counts is how many bytes of it are in flight and that
// nothing is staged that is not there: a tile of 128 x-rows would be mostly
// zeros, here x takes N = 16..128 rows of shared memory. A CTA makes 128
// output channels over a slice of the K axis, one stage of 64 K elements
// after the other through a ring of 220 KB where every CTA has an SM to
// itself ([16, 6144] -> 1536: 8.2 us, 10.6 with 108 KB), else of 108 KB, two
// CTAs an SM. The slices of a cluster are added up through distributed shared
// memory in rank order, four neighbouring channels of a row a thread ([256,
// 1536] -> 6144, one slice: 18.0 us; straight from TMEM, a channel a lane,
// 21.4).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "dense.h"
#include "entry.h"
#include "internal.h"
#include "sm100.cuh"
#include "tensormap.h"

namespace t2sc {
namespace {

constexpr int kMaxSlices = 8, kM = 128, kBK = 64, kThreads = 192;  // warps 0-3 epilogue, 4 TMA, 5 MMA
constexpr int kRingTwo = 108 * 1024, kRingOne = 220 * 1024;  // with two CTAs an SM, with one
constexpr long long kWaitLimit = 4000000000ll;                          // ~2 s of SM clocks

struct SkinnyArgs {
  CUtensorMap map_x, map_w;
  const char *res;
  char *y;
  const float *bias;
  int64_t ldr, ldy;  // elements
  int rows, co, k_iters, act, slices, row_tiles, stages;
  int vec;  // co a multiple of 4, y (and residual) rows start on 8 bytes
  int *err;
};

template <int N>
struct Shape {
  static constexpr int kWBytes = kM * 128, kXBytes = N * 128, kStage = kWBytes + kXBytes;
  static constexpr int stages(int ring) { return ring / kStage; }
  static constexpr size_t smem(int stages) { return 1024 + (size_t)stages * kStage + 256; }
  static constexpr uint32_t kCols = N < 32 ? 32 : N;
  static_assert(N * kM * 4 <= 2 * kStage, "a slice's sums fit the ring");
  static_assert(8 * (2 * stages(kRingOne) + 1) + 8 <= 256, "the barriers fit behind the ring");
};

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort, int *err) {
  const bool ok = sm100::mbar_wait_bounded(bar, parity, abort, err, kDevErrTimeout, kWaitLimit);
  return __all_sync(0xffffffffu, ok);
}

template <int DT>
__device__ __forceinline__ float ld16(const char *p) {
  if (DT == T2SC_DT_BF16) return __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(p));
  return __half2float(*reinterpret_cast<const __half *>(p));
}

template <int DT>
__device__ __forceinline__ void finish(const SkinnyArgs &a, int64_t r, int o, float v, float bias) {
  v = activate(v + bias, a.act);
  if (a.res) v += ld16<DT>(a.res + (r * a.ldr + o) * 2);
  char *p = a.y + (r * a.ldy + o) * 2;
  if (DT == T2SC_DT_BF16)
    *reinterpret_cast<__nv_bfloat16 *>(p) = __float2bfloat16_rn(v);
  else
    *reinterpret_cast<__half *>(p) = __float2half_rn(v);
}

// Four neighbouring channels.
template <int DT>
__device__ __forceinline__ void finish4(const SkinnyArgs &a, int64_t r, int o, const float (&v)[4], const float (&bias)[4]) {
  if (!a.vec) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (o + j < a.co) finish<DT>(a, r, o + j, v[j], bias[j]);
    return;
  }
  if (o >= a.co) return;
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; j++) y[j] = activate(v[j] + bias[j], a.act);
  if (a.res) {
    const uint2 u = *reinterpret_cast<const uint2 *>(a.res + (r * a.ldr + o) * 2);
    const float2 p = unpack2<DT>(u.x), q = unpack2<DT>(u.y);
    y[0] += p.x, y[1] += p.y, y[2] += q.x, y[3] += q.y;
  }
  *reinterpret_cast<uint2 *>(a.y + (r * a.ldy + o) * 2) = make_uint2(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]));
}

__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

template <int DT, int N>
__global__ void __launch_bounds__(kThreads, 2) dense_skinny_kernel(const __grid_constant__ SkinnyArgs a) {
  using S = Shape<N>;
  const int NS = a.stages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (size_t)NS * S::kStage);  // full[NS], empty[NS], done
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * NS + 1);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const uint32_t sbase = sm100::smem_u32(smem), full0 = sm100::smem_u32(bars), empty0 = full0 + 8 * NS, done = empty0 + 8 * NS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = (int)blockIdx.x / a.slices, slice = (int)blockIdx.x % a.slices;
  const int o0 = tile / a.row_tiles * kM, row0 = tile % a.row_tiles * N;  // the row tiles of a piece of w are neighbours
  const int rows = min(N, a.rows - row0);
  const int per = (a.k_iters + a.slices - 1) / a.slices, k0 = min(slice * per, a.k_iters), n = min(k0 + per, a.k_iters) - k0;
  if (warp == 4 && lane == 0) {
    sm100::tma_prefetch(&a.map_x);
    sm100::tma_prefetch(&a.map_w);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; s++) {
      sm100::mbar_init(full0 + 8 * s, 1);
      sm100::mbar_init(empty0 + 8 * s, 1);
    }
    sm100::mbar_init(done, 1);
    *abort = 0;
    sm100::fence_mbar_init();
  }
  if (warp == 5) {
    sm100::tmem_alloc(sm100::smem_u32(tmem_slot), S::kCols);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  sm100::next_kernel_may_start();
  sm100::previous_kernel_done();
  const uint32_t tmem = *tmem_slot;
  if (warp == 4) {
    if (lane == 0) {
      bool ok = true;
      int k = 0;
      uint32_t s = 0, ph = 0;
      for (; k < n && ok; k++) {
        const uint32_t dst = sbase + s * S::kStage;
        ok = sm100::mbar_wait_bounded(empty0 + 8 * s, ph ^ 1, abort, a.err, kDevErrTimeout, kWaitLimit);
        if (!ok) break;
        sm100::mbar_arrive_expect_tx(full0 + 8 * s, S::kStage);
        sm100::tma_load_2d(dst, &a.map_w, (k0 + k) * kBK, o0, full0 + 8 * s);
        sm100::tma_load_2d(dst + S::kWBytes, &a.map_x, (k0 + k) * kBK, row0, full0 + 8 * s);
        if ((int)++s == NS) s = 0, ph ^= 1;
      }
      for (int i = max(0, k - NS); i < k; i++)  // every copy asked for has landed before shared memory is used again or given up
        sm100::mbar_wait_cycles(full0 + 8 * (i % NS), (i / NS) & 1, kWaitLimit / 8);
    }
    __syncwarp();
  } else if (warp == 5) {
    if (sm100::elect_one()) {
      constexpr uint32_t idesc = sm100::instr_desc(DT == T2SC_DT_BF16 ? 1 : 0, N);
      const uint64_t dw = sm100::smem_desc(sbase, 128);
      const uint32_t hi = (uint32_t)(dw >> 32), w_lo = (uint32_t)dw, x_lo = w_lo + (S::kWBytes >> 4);
      bool ok = true;
      uint32_t s = 0, ph = 0;
      for (int k = 0; k < n && ok; k++) {
        const uint32_t at = s * (S::kStage >> 4);
        ok = sm100::mbar_wait_bounded(full0 + 8 * s, ph, abort, a.err, kDevErrTimeout, kWaitLimit);
        if (!ok) break;
        sm100::tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kBK / 16; kk++) sm100::mma_f16_lo(tmem, w_lo + at + kk * 2, x_lo + at + kk * 2, hi, idesc, k + kk > 0);
        sm100::mma_commit(empty0 + 8 * s);
        if ((int)++s == NS) s = 0, ph ^= 1;
      }
      sm100::mma_commit(done);
      // all issued MMAs retire before TMEM and shared memory are given up
      sm100::mbar_wait_cycles(done, 0, kWaitLimit / 8);
    }
    __syncwarp();
  } else {
    const bool ok = warp_wait(done, 0, abort, a.err);
    sm100::tc_fence_after();
    const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
    float *sums = reinterpret_cast<float *>(smem);  // [rows][128] of this slice, over the ring
#pragma unroll 1
    for (int c = 0; c < N; c += 16) {
      if (c >= rows) break;
      uint32_t v[16];
      sm100::tmem_ld16(taddr + c, v);
      sm100::tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; j++) sums[(c + j) * kM + threadIdx.x] = n > 0 ? __uint_as_float(v[j]) : 0.f;
    }
    __syncwarp();
    sm100::cluster_sync();
    // four neighbouring channels of a row a thread; this CTA's share of the rows
    const int c4 = lane * 4;
    const uint32_t at = sm100::smem_u32(sums) + 4 * c4;
    float b4[4];
#pragma unroll
    for (int j = 0; j < 4; j++) b4[j] = a.bias && o0 + c4 + j < a.co ? a.bias[o0 + c4 + j] : 0.f;
    const int step = a.slices * 4;
    for (int r = slice + a.slices * warp; r < rows; r += 2 * step) {  // two rows at a time
      float4 t[2][kMaxSlices];
#pragma unroll
      for (int z = 0; z < kMaxSlices; z++)
        if (z < a.slices) {
#pragma unroll
          for (int i = 0; i < 2; i++)
            if (r + i * step < rows) t[i][z] = ld_cluster(sm100::map_to_rank(at + 4 * kM * (r + i * step), z));
        }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if (r + i * step >= rows) break;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int z = 0; z < kMaxSlices; z++)
          if (z < a.slices) v[0] += t[i][z].x, v[1] += t[i][z].y, v[2] += t[i][z].z, v[3] += t[i][z].w;
        if (ok) finish4<DT>(a, row0 + r + i * step, o0 + c4, v, b4);
      }
    }
    __syncwarp();
    sm100::cluster_sync();  // no CTA leaves before the others have read its sums
  }
  if (warp >= 4) {  // the epilogue's two barriers around the sums' exchange
    sm100::cluster_sync();
    sm100::cluster_sync();
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, S::kCols);
  }
}

// K slices while there are SMs without a CTA, at least four stages a slice
// ([16, 4096] -> 1024: 8.0 us with 8 slices, 18.7 with one; with two CTAs an
// SM the exchange of the sums costs more than it gives: [16, 1536] -> 9216 9.4
// us with two slices, 12.5 with four).
int slices_of(int64_t tiles, int k_iters, int sms) {
  int n = 1;
  while (n < kMaxSlices && tiles * n * 2 <= sms && k_iters >= 8 * n) n *= 2;
  return n;
}

template <int DT, int N>
int launch(t2sc_ctx *ctx, const DenseArgs &a, std::string &err) {
  using S = Shape<N>;
  SkinnyArgs t;
  const uint64_t dx[2] = {(uint64_t)a.ci, (uint64_t)a.rows}, dw[2] = {(uint64_t)a.ci, (uint64_t)a.co};
  const uint64_t one = ((uint64_t)a.ci * 2 + 15) / 16 * 16;  // a stride that a single row never uses
  const uint64_t sx[1] = {a.rows > 1 ? (uint64_t)a.ldx * 2 : one}, sw[1] = {a.co > 1 ? (uint64_t)a.ldw * 2 : one};
  const uint32_t bx[2] = {kBK, N}, bw[2] = {kBK, kM};
  T2SC_TRY(tensormap_16bit(&t.map_x, DT, 2, a.x, dx, sx, bx, err));
  T2SC_TRY(tensormap_16bit(&t.map_w, DT, 2, a.w, dw, sw, bw, err));
  t.res = a.res, t.y = a.y, t.bias = a.bias, t.ldr = a.ldr, t.ldy = a.ldy, t.rows = (int)a.rows, t.co = a.co;
  auto on8 = [&](const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 8 == 0 && (a.rows <= 1 || ld % 4 == 0); };
  t.vec = a.co % 4 == 0 && on8(a.y, a.ldy) && (!a.res || on8(a.res, a.ldr));
  t.row_tiles = ((int)a.rows + N - 1) / N;
  t.k_iters = (a.ci + kBK - 1) / kBK, t.act = a.act, t.err = ctx->d_wait;
  const int64_t tiles = (int64_t)((a.co + kM - 1) / kM) * t.row_tiles;
  t.slices = slices_of(tiles, t.k_iters, ctx->num_sms);
  if (tiles * t.slices > INT32_MAX) return fail(ctx, T2SC_ERR_UNSUPPORTED, "dense_linear: too many outputs");
  auto kernel = dense_skinny_kernel<DT, N>;
  static Clusters<kMaxSlices> table[64];
  const int *at_once = nullptr;
  T2SC_TRY(clusters_at_once(ctx, kernel, kThreads, S::smem(S::stages(kRingOne)), table, &at_once, err));
  // no more stages than a slice has steps: the next kernel's CTAs may wait beside this one's
  const int per = (t.k_iters + t.slices - 1) / t.slices;
  t.stages = std::min(std::max(per, 2), S::stages(tiles <= at_once[t.slices] ? kRingOne : kRingTwo));
  T2SC_CUDA(launch_overlapped(kernel, tiles * t.slices, kThreads, S::smem(t.stages), ctx->stream, t.slices, t), "dense_linear");
  T2SC_LAUNCHED(ctx, "dense_linear");
  return T2SC_OK;
}

template <int DT>
int launch_dt(t2sc_ctx *ctx, const DenseArgs &a, std::string &err) {
  if (a.rows <= 16) return launch<DT, 16>(ctx, a, err);
  if (a.rows <= 32) return launch<DT, 32>(ctx, a, err);
  if (a.rows <= 64) return launch<DT, 64>(ctx, a, err);
  return launch<DT, 128>(ctx, a, err);
}

}  // namespace

// Up to 64 rows. Above, tiles of 128 rows are full enough for the row-major
// kernel, which is the faster one unless it has too few tiles for a long K
// axis, which it does not split: [256, 1536] -> 6144 10.1 us there, 18.1
// here; [256, 6144] -> 1536 24.0 there, 12.8 here. What a call takes here, in
// microseconds: 6, a K step 0.25 on an SM of its own and 0.5 on a shared one,
// and 0.04 a row that a CTA finishes (within 15 % where it is chosen,
// profiles/attention_block_models.txt).
bool dense_skinny_takes(t2sc_ctx *ctx, const DenseArgs &a, int dtype) {
  if (!dense_tc_takes(a, dtype) || a.rows > 65536) return false;
  if (a.rows <= 64) return true;
  const int64_t tiles = ((a.rows + 127) / 128) * ((a.co + kM - 1) / kM);
  const int k_iters = (a.ci + kBK - 1) / kBK, slices = slices_of(tiles, k_iters, ctx->num_sms);
  const int64_t ctas = tiles * slices, at_once = ctas * 8 <= ctx->num_sms * 7 ? ctas : 2 * ctx->num_sms;
  const double steps = (k_iters + slices - 1) / slices, rows = a.rows < 128 ? a.rows : 128;
  const double us = 6 + (double)((ctas + at_once - 1) / at_once) * (steps * (at_once == ctas ? 0.25 : 0.5) + rows / slices * 0.04);
  int best;
  return us < dense_tc_us(ctx, a, &best);
}

int dense_skinny(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err) {
  return dtype == T2SC_DT_BF16 ? launch_dt<T2SC_DT_BF16>(ctx, a, err) : launch_dt<T2SC_DT_F16>(ctx, a, err);
}

}  // namespace t2sc
