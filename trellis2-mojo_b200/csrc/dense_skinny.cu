// Dense linear of a few to 128 rows on the tensor cores, operands swapped: the
// weight's 128 output channels are the M of an MMA, the rows its N.
//
// With few rows the call streams the weight (HBM, or L2 where it still is
// there), so what counts is how many bytes of it are in flight and that
// nothing is staged that is not there: a tile of 128 x-rows would be mostly
// zeros, here x takes N = 16..128 rows of shared memory. A CTA makes 128
// output channels over a slice of the K axis, one stage of 64 K elements
// after the other through a ring that leaves room for a second CTA on the SM;
// the slices of a cluster are added up through distributed shared memory in
// rank order. TMEM lanes are output channels: a warp's stores of one row are
// 32 neighbours.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dense.h"
#include "entry.h"
#include "internal.h"
#include "sm100.cuh"
#include "tensormap.h"

namespace t2sc {
namespace {

constexpr int kMaxSlices = 8, kM = 128, kBK = 64, kThreads = 192, kRing = 108 * 1024;  // warps 0-3 epilogue, 4 TMA, 5 MMA
constexpr long long kWaitLimit = 4000000000ll;                          // ~2 s of SM clocks

struct SkinnyArgs {
  CUtensorMap map_x, map_w;
  const char *res;
  char *y;
  const float *bias;
  int64_t ldr, ldy;  // elements
  int rows, co, k_iters, act, slices;
  int *err;
};

template <int N>
struct Shape {
  static constexpr int kWBytes = kM * 128, kXBytes = N * 128, kStage = kWBytes + kXBytes;
  static constexpr int kStages = kRing / kStage;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + 256;
  static constexpr uint32_t kCols = N < 32 ? 32 : N;
  static_assert(N * kM * 4 <= kStages * kStage, "a slice's sums fit the ring");
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
__device__ __forceinline__ void finish(const SkinnyArgs &a, int r, int o, float v, float bias) {
  v = activate(v + bias, a.act);
  if (a.res) v += ld16<DT>(a.res + (r * a.ldr + o) * 2);
  char *p = a.y + (r * a.ldy + o) * 2;
  if (DT == T2SC_DT_BF16)
    *reinterpret_cast<__nv_bfloat16 *>(p) = __float2bfloat16_rn(v);
  else
    *reinterpret_cast<__half *>(p) = __float2half_rn(v);
}

template <int DT, int N>
__global__ void __launch_bounds__(kThreads, 2) dense_skinny_kernel(const __grid_constant__ SkinnyArgs a) {
  using S = Shape<N>;
  constexpr int NS = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (size_t)NS * S::kStage);  // full[NS], empty[NS], done
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * NS + 1);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const uint32_t sbase = sm100::smem_u32(smem), full0 = sm100::smem_u32(bars), empty0 = full0 + 8 * NS, done = empty0 + 8 * NS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int o0 = (int)blockIdx.x / a.slices * kM, slice = (int)blockIdx.x % a.slices;
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
  const uint32_t tmem = *tmem_slot;
  if (warp == 4) {
    if (lane == 0) {
      bool ok = true;
      int k = 0;
      for (; k < n && ok; k++) {
        const uint32_t s = k % NS, dst = sbase + s * S::kStage;
        ok = sm100::mbar_wait_bounded(empty0 + 8 * s, ((k / NS) & 1) ^ 1, abort, a.err, kDevErrTimeout, kWaitLimit);
        if (!ok) break;
        sm100::mbar_arrive_expect_tx(full0 + 8 * s, S::kStage);
        sm100::tma_load_2d(dst, &a.map_w, (k0 + k) * kBK, o0, full0 + 8 * s);
        sm100::tma_load_2d(dst + S::kWBytes, &a.map_x, (k0 + k) * kBK, 0, full0 + 8 * s);
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
      for (int k = 0; k < n && ok; k++) {
        const uint32_t s = k % NS, at = s * (S::kStage >> 4);
        ok = sm100::mbar_wait_bounded(full0 + 8 * s, (k / NS) & 1, abort, a.err, kDevErrTimeout, kWaitLimit);
        if (!ok) break;
        sm100::tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kBK / 16; kk++) sm100::mma_f16_lo(tmem, w_lo + at + kk * 2, x_lo + at + kk * 2, hi, idesc, k + kk > 0);
        sm100::mma_commit(empty0 + 8 * s);
      }
      sm100::mma_commit(done);
      // all issued MMAs retire before TMEM and shared memory are given up
      sm100::mbar_wait_cycles(done, 0, kWaitLimit / 8);
    }
    __syncwarp();
  } else {
    const int o = o0 + (int)threadIdx.x;
    const float bias = a.bias && o < a.co ? __ldg(a.bias + o) : 0.f;
    const bool ok = warp_wait(done, 0, abort, a.err);
    sm100::tc_fence_after();
    const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
    if (a.slices == 1) {
#pragma unroll 1
      for (int c = 0; c < N; c += 16) {
        if (c >= a.rows) break;
        uint32_t v[16];
        sm100::tmem_ld16(taddr + c, v);
        sm100::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j++)
          if (c + j < a.rows && o < a.co && ok) finish<DT>(a, c + j, o, __uint_as_float(v[j]), bias);
      }
    } else {
      float *sums = reinterpret_cast<float *>(smem);  // [rows][128] of this slice, over the ring
#pragma unroll 1
      for (int c = 0; c < N; c += 16) {
        if (c >= a.rows) break;
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
      for (int j = 0; j < 4; j++) b4[j] = a.bias && o0 + c4 + j < a.co ? __ldg(a.bias + o0 + c4 + j) : 0.f;
      for (int r = slice + a.slices * warp; r < a.rows; r += a.slices * 4) {
        float4 t[kMaxSlices];
#pragma unroll
        for (int z = 0; z < kMaxSlices; z++)
          if (z < a.slices) {
            const uint32_t p = sm100::map_to_rank(at + 4 * kM * r, z);
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(t[z].x), "=f"(t[z].y), "=f"(t[z].z), "=f"(t[z].w) : "r"(p));
          }
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int z = 0; z < kMaxSlices; z++)
          if (z < a.slices) v[0] += t[z].x, v[1] += t[z].y, v[2] += t[z].z, v[3] += t[z].w;
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (o0 + c4 + j < a.co && ok) finish<DT>(a, r, o0 + c4 + j, v[j], b4[j]);
      }
      __syncwarp();
      sm100::cluster_sync();  // no CTA leaves before the others have read its sums
    }
  }
  if (warp >= 4 && a.slices > 1) {  // the epilogue's two barriers around the sums' exchange
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
  t.k_iters = (a.ci + kBK - 1) / kBK, t.act = a.act, t.err = ctx->d_err;
  // K slices while there are SMs without a CTA, at least four stages a slice
  // ([16, 4096] -> 1024: 8.0 us with 8 slices, 18.7 with one; with two CTAs an
  // SM the exchange of the sums costs more than it gives: [16, 1536] -> 9216
  // 9.4 us with two slices, 12.5 with four)
  const int64_t tiles = (a.co + kM - 1) / kM;
  t.slices = 1;
  while (t.slices < kMaxSlices && tiles * t.slices * 2 <= ctx->num_sms && t.k_iters >= 8 * t.slices) t.slices *= 2;
  if (tiles * t.slices > INT32_MAX) return fail(ctx, T2SC_ERR_UNSUPPORTED, "dense_linear: too many outputs");
  auto kernel = dense_skinny_kernel<DT, N>;
  static std::atomic<uint64_t> allowed{0};
  T2SC_TRY(allow_smem(ctx, kernel, (int)S::kSmem, allowed, err));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * t.slices)), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = S::kSmem, cfg.stream = ctx->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = t.slices, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  T2SC_CUDA(cudaLaunchKernelEx(&cfg, kernel, t), "dense_linear");
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

// Up to 64 rows. Above, a tile of 128 rows is full enough for the row-major
// kernel ([128, 1536] -> 9216: 11.2 us there, 18.7 here), unless it has too
// few tiles for a long K axis, which it does not split ([100, 6144] -> 1536:
// 26.9 us there, 12.6 here).
bool dense_skinny_takes(t2sc_ctx *ctx, const DenseArgs &a, int dtype) {
  if (!dense_tc_takes(a, dtype) || a.rows > 128) return false;
  return a.rows <= 64 || (a.ci >= 48 * kBK && (a.co + kM - 1) / kM * 4 <= ctx->num_sms);
}

int dense_skinny(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err) {
  return dtype == T2SC_DT_BF16 ? launch_dt<T2SC_DT_BF16>(ctx, a, err) : launch_dt<T2SC_DT_F16>(ctx, a, err);
}

}  // namespace t2sc
