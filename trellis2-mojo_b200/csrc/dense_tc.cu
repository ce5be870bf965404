// Dense linear on the tensor cores: y = act(x @ w^T + bias) + residual for
// 16-bit rows that start on 16 bytes.
//
// Output tiles of 128 rows x BN columns a CTA, the K axis in 128-byte steps:
// TMA brings the x and w tiles into a ring of shared-memory stages (128-byte
// swizzle, zeros outside the matrices), one warp issues tcgen05.mma into one
// of two TMEM accumulators while eight warps drain the other through the
// epilogue. With a CTA pair (CG = 2) one MMA covers 256 rows and each CTA
// stages only half of the w tile, which halves what shared memory has to
// take in and feed for w. The CTAs are persistent; a CTA's tiles are `slots`
// apart with the columns fastest, so that the tiles in flight share their x
// rows and a band of w in L2.
//
// The epilogue takes 64 columns at a time: a thread owns a row (TMEM lane),
// and the block passes through a swizzled 4 KB of shared memory per warp so
// that the residual is read and y written in whole 128-byte rows. y may be
// the residual: each element is read before the same thread writes it. Rows
// that do not start on 16 bytes, and the last columns, pass two bytes a lane,
// neighbouring columns together ([9813, 616] -> 2143 with residual: 144 us
// with eight neighbours a lane, 84 so).
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

constexpr int kTileM = 128;         // rows of a CTA's tile
constexpr int kBK = 64;             // K elements of a stage: one 128-byte swizzle row
constexpr int kSmemMax = 232448;    // 227 KB: the sm_100 per-block limit
constexpr int kEpiWarps = 8;        // two per TMEM lane quadrant, 64 columns at a time each
constexpr int kTmaWarp = kEpiWarps, kMmaWarp = kEpiWarps + 1, kThreads = 32 * (kEpiWarps + 2);
constexpr int kStageBytes = kEpiWarps * 32 * 128;  // epilogue staging, 4 KB a warp
constexpr long long kWaitLimit = 4000000000ll;  // ~2 s of SM clocks

struct DenseTcArgs {
  CUtensorMap map_x, map_w;
  const char *res;
  char *y;
  const float *bias;
  int64_t ldr, ldy;  // elements
  int64_t rows;
  int co, k_iters, act, m_tiles, n_tiles, band, slots;
  int vec;  // y (and residual) rows start on 16 bytes
  int *err;
};

template <int CG, int BN>
struct Shape {
  static constexpr int kWRows = BN / CG;  // w rows a CTA stages
  static constexpr int kABytes = kTileM * 128, kBBytes = kWRows * 128;
  static constexpr int kBiasBytes = kEpiWarps * 64 * 4;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kStages = (kSmemMax - 1024 - kStageBytes - kBiasBytes - 512) / kStage > 8
                                     ? 8
                                     : (kSmemMax - 1024 - kStageBytes - kBiasBytes - 512) / kStage;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kStageBytes + kBiasBytes + 512;
  static constexpr uint32_t kCols = 2 * BN;  // two accumulators
};

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort, int *err) {
  bool ok = sm100::mbar_test_wait(bar, parity);
  if (__all_sync(0xffffffffu, ok)) return true;
  if (!ok) ok = sm100::mbar_wait_bounded(bar, parity, abort, err, kDevErrTimeout, kWaitLimit);
  return __all_sync(0xffffffffu, ok);
}

template <int DT, int CG, int BN>
__global__ void __launch_bounds__(kThreads, 1) dense_tc_kernel(const __grid_constant__ DenseTcArgs a) {
  using S = Shape<CG, BN>;
  constexpr int NS = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *staging = smem + (size_t)NS * S::kStage;
  uint64_t *bars = reinterpret_cast<uint64_t *>(staging + kStageBytes + S::kBiasBytes);  // full[NS], empty[NS], tfull[2], tempty[2], done
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * NS + 5);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const uint32_t sbase = sm100::smem_u32(smem), full0 = sm100::smem_u32(bars), empty0 = full0 + 8 * NS;
  const uint32_t tfull0 = empty0 + 8 * NS, tempty0 = tfull0 + 16, done = tempty0 + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? sm100::cluster_rank() : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; s++) {
      sm100::mbar_init(full0 + 8 * s, 1);
      sm100::mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; b++) {
      sm100::mbar_init(tfull0 + 8 * b, 1);
      sm100::mbar_init(tempty0 + 8 * b, kEpiWarps * CG);  // every epilogue warp of the pair
    }
    sm100::mbar_init(done, 1);
    *abort = 0;
    sm100::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    if (CG == 2) {
      sm100::tmem_alloc_pair(sm100::smem_u32(tmem_slot), S::kCols);
      sm100::tmem_relinquish_pair();
    } else {
      sm100::tmem_alloc(sm100::smem_u32(tmem_slot), S::kCols);
      sm100::tmem_relinquish();
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (CG == 2) sm100::cluster_sync();  // the other CTA's barriers are ready before anything arrives on them
  sm100::tc_fence_after();
  sm100::next_kernel_may_start();
  sm100::previous_kernel_done();
  const uint32_t tmem = *tmem_slot;
  const int64_t ntiles = (int64_t)a.m_tiles * a.n_tiles;
  const int64_t slot = blockIdx.x / CG;
  // Tile t: blocks of `band` column tiles (what of w stays in L2 beside x),
  // rows by rows inside a band, the columns fastest.
  auto place = [&](int64_t t, int &m, int &n) {
    const int64_t per_band = (int64_t)a.band * a.m_tiles;
    const int first = (int)(t / per_band) * a.band, width = min(a.band, a.n_tiles - first);
    const int64_t i = t % per_band;
    m = (int)(i / width), n = first + (int)(i % width);
  };

  if (warp == kTmaWarp) {
    // ------------------------------- TMA --------------------------------
    if (lane == 0) {
      sm100::tma_prefetch(&a.map_x);
      sm100::tma_prefetch(&a.map_w);
      uint32_t s = 0, ph = 0, it = 0;
      bool ok = true;
      for (int64_t t = slot; t < ntiles && ok; t += a.slots) {
        int m, nt;
        place(t, m, nt);
        const int m0 = m * kTileM * CG + (int)rank * kTileM, n0 = nt * BN + (int)rank * S::kWRows;
        for (int k = 0; k < a.k_iters; k++) {
          ok = sm100::mbar_wait_bounded(empty0 + 8 * s, ph ^ 1, abort, a.err, kDevErrTimeout, kWaitLimit);
          if (!ok) break;
          const uint32_t dst = sbase + s * S::kStage;
          if (CG == 2) {
            const uint32_t bar = sm100::map_to_rank(full0 + 8 * s, 0);  // CTA 0 waits for both CTAs' tiles
            if (rank == 0) sm100::mbar_arrive_expect_tx(full0 + 8 * s, 2 * S::kStage);
            sm100::tma_load_2d_pair(dst, &a.map_x, k * kBK, m0, bar);
            sm100::tma_load_2d_pair(dst + S::kABytes, &a.map_w, k * kBK, n0, bar);
          } else {
            sm100::mbar_arrive_expect_tx(full0 + 8 * s, S::kStage);
            sm100::tma_load_2d(dst, &a.map_x, k * kBK, m0, full0 + 8 * s);
            sm100::tma_load_2d(dst + S::kABytes, &a.map_w, k * kBK, n0, full0 + 8 * s);
          }
          it++;
          if (++s == NS) s = 0, ph ^= 1;
        }
      }
      // every copy asked for has landed before shared memory is given up (a
      // pair's land on CTA 0's barriers, and CTA 1 stays until the cluster's end)
      if (rank == 0)
        for (uint32_t i = it > (uint32_t)NS ? it - NS : 0; i < it; i++)
          sm100::mbar_wait_cycles(full0 + 8 * (i % NS), (i / NS) & 1, kWaitLimit / 8);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ------------------------------- MMA --------------------------------
    if (rank == 0 && sm100::elect_one()) {
      constexpr uint32_t idesc = sm100::instr_desc(DT == T2SC_DT_BF16 ? 1 : 0, BN) + (CG == 2 ? (128u >> 4) << 24 : 0u);
      const uint64_t da0 = sm100::smem_desc(sbase, 128);
      const uint32_t hi = (uint32_t)(da0 >> 32), a_lo = (uint32_t)da0, b_lo = a_lo + (S::kABytes >> 4);
      uint32_t s = 0, ph = 0, acc = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        ok = ok && sm100::mbar_wait_bounded(bar, parity, abort, a.err, kDevErrTimeout, kWaitLimit);
      };
      auto commit = [&](uint32_t bar) {
        if (CG == 2)
          sm100::mma_commit_pair(bar);
        else
          sm100::mma_commit(bar);
      };
      for (int64_t t = slot; t < ntiles && ok; t += a.slots) {
        const uint32_t b = acc & 1;
        wait(tempty0 + 8 * b, ((acc >> 1) & 1) ^ 1);
        if (CG == 2) asm volatile("fence.acq_rel.cluster;" ::: "memory");  // half of the arrivals are the other CTA's
        sm100::tc_fence_after();
        const uint32_t d = tmem + b * BN;
        for (int k = 0; k < a.k_iters && ok; k++) {
          wait(full0 + 8 * s, ph);
          if (!ok) break;
          sm100::tc_fence_after();
          const uint32_t at = s * (S::kStage >> 4);
#pragma unroll
          for (int kk = 0; kk < kBK / 16; kk++) {
            if (CG == 2)
              sm100::mma_f16_pair_lo(d, a_lo + at + kk * 2, b_lo + at + kk * 2, hi, idesc, k + kk > 0);
            else
              sm100::mma_f16_lo(d, a_lo + at + kk * 2, b_lo + at + kk * 2, hi, idesc, k + kk > 0);
          }
          commit(empty0 + 8 * s);
          if (++s == NS) s = 0, ph ^= 1;
        }
        if (!ok) break;
        commit(tfull0 + 8 * b);
        acc++;
      }
      // all issued MMAs retire before TMEM and shared memory are given up
      commit(done);
      sm100::mbar_wait_cycles(done, 0, kWaitLimit / 8);
    }
    __syncwarp();
  } else {
    // ----------------------------- epilogue -----------------------------
    // Warp w reads TMEM lanes 32 (w % 4)..; the two warps of a quadrant take
    // turns at blocks of 64 columns.
    const int quad = warp & 3, half = warp >> 2;
    uint8_t *stage = staging + warp * 4096;
    float *bias = reinterpret_cast<float *>(staging + kStageBytes) + warp * 64;  // of the block at hand
    uint32_t acc = 0;
    const int crow = lane >> 3, cch = lane & 7;  // this lane's place when whole rows move: 4 rows x 8 chunks
    for (int64_t t = slot; t < ntiles; t += a.slots) {
      int m, nt;
      place(t, m, nt);
      const int64_t row0 = (int64_t)m * (kTileM * CG) + (int64_t)rank * kTileM + quad * 32;
      const int n0 = nt * BN;
      const uint32_t b = acc & 1;
      // the first block's bias and residual come in while the tile is still computed
      float bias0, bias1;
      auto load_bias = [&](int col0) {
        const int col = col0 + lane;
        bias0 = a.bias && col < a.co ? a.bias[col] : 0.f;
        bias1 = a.bias && col + 32 < a.co ? a.bias[col + 32] : 0.f;
      };
      uint32_t res[32];  // whole rows: a lane's 8 chunks; else row r's columns lane and lane + 32
      auto load_residual = [&](int col0) {
        if (a.vec && col0 + 64 <= a.co) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int64_t r = row0 + i * 4 + crow;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (r < a.rows) u = *reinterpret_cast<const uint4 *>(a.res + (r * a.ldr + col0 + cch * 8) * 2);
            res[4 * i] = u.x, res[4 * i + 1] = u.y, res[4 * i + 2] = u.z, res[4 * i + 3] = u.w;
          }
        } else {
          // places outside read a neighbour instead, which nothing uses: no branch between the loads
          const uint16_t *p0 = reinterpret_cast<const uint16_t *>(a.res) + min(col0 + lane, a.co - 1);
          const int next = min(col0 + lane + 32, a.co - 1) - min(col0 + lane, a.co - 1);
          const int64_t first = min(row0, a.rows - 1);
          const int last = (int)min((int64_t)31, a.rows - 1 - first);
          p0 += first * a.ldr;
#pragma unroll
          for (int r = 0; r < 32; r++) {
            const uint16_t *p = p0 + min(r, last) * a.ldr;
            res[r] = (uint32_t)p[0] | (uint32_t)p[next] << 16;
          }
        }
      };
      // column c of row r in the staging block
      auto single = [&](int r, int c) { return reinterpret_cast<uint16_t *>(stage + r * 128 + ((c >> 3 ^ (r & 7)) << 4) + (c & 7) * 2); };
      if (half * 64 < BN) {
        load_bias(n0 + half * 64);
        if (a.res) load_residual(n0 + half * 64);
      }
      if (!warp_wait(tfull0 + 8 * b, (acc >> 1) & 1, abort, a.err)) break;
      sm100::tc_fence_after();
      const uint32_t taddr = tmem + b * BN + ((uint32_t)(quad * 32) << 16);
#pragma unroll 1
      for (int c0 = half * 64; c0 < BN; c0 += 128) {
        const int col0 = n0 + c0;
        float v[64];
        sm100::tmem_ld32(taddr + c0, reinterpret_cast<uint32_t *>(v));
        sm100::tmem_ld32(taddr + c0 + 32, reinterpret_cast<uint32_t *>(v) + 32);
        const bool whole = a.vec && col0 + 64 <= a.co;
        if (a.res) {
          if (whole) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int r = i * 4 + crow;
              *reinterpret_cast<uint4 *>(stage + r * 128 + ((cch ^ (r & 7)) << 4)) =
                  make_uint4(res[4 * i], res[4 * i + 1], res[4 * i + 2], res[4 * i + 3]);
            }
          } else {
#pragma unroll
            for (int r = 0; r < 32; r++) *single(r, lane) = (uint16_t)res[r], *single(r, lane + 32) = (uint16_t)(res[r] >> 16);
          }
          if (c0 + 128 < BN) load_residual(col0 + 128);
        }
        bias[lane] = bias0, bias[lane + 32] = bias1;
        if (c0 + 128 < BN) load_bias(col0 + 128);
        __syncwarp();
        sm100::tmem_ld_wait();
        if (c0 + 128 >= BN) {  // this warp's part of the accumulator is read out
          sm100::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2)
              sm100::mbar_arrive_cluster(sm100::map_to_rank(tempty0 + 8 * b, 0));
            else
              sm100::mbar_arrive(tempty0 + 8 * b);
          }
        }
        if (col0 >= a.co || row0 >= a.rows) {
          __syncwarp();
          continue;
        }
#pragma unroll
        for (int c = 0; c < 16; c++) {
          const float4 w = *reinterpret_cast<const float4 *>(bias + c * 4);
          v[4 * c] += w.x, v[4 * c + 1] += w.y, v[4 * c + 2] += w.z, v[4 * c + 3] += w.w;
        }
        if (a.act & T2SC_SILU) {
#pragma unroll
          for (int j = 0; j < 64; j++) v[j] = silu_any(v[j]);
        } else if (a.act & T2SC_GELU) {
#pragma unroll
          for (int j = 0; j < 64; j++) v[j] = gelu_tanh(v[j]);
        }
#pragma unroll
        for (int c = 0; c < 8; c++) {
          float *z = v + c * 8;
          uint4 *sp = reinterpret_cast<uint4 *>(stage + lane * 128 + ((c ^ (lane & 7)) << 4));
          if (a.res) {
            const uint4 u = *sp;
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float2 f = unpack2<DT>(w[j]);
              z[2 * j] += f.x, z[2 * j + 1] += f.y;
            }
          }
          *sp = make_uint4(pack2<DT>(z[0], z[1]), pack2<DT>(z[2], z[3]), pack2<DT>(z[4], z[5]), pack2<DT>(z[6], z[7]));
        }
        __syncwarp();
        if (whole) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int r = i * 4 + crow;
            if (row0 + r < a.rows)
              *reinterpret_cast<uint4 *>(a.y + ((row0 + r) * a.ldy + col0 + cch * 8) * 2) =
                  *reinterpret_cast<const uint4 *>(stage + r * 128 + ((cch ^ (r & 7)) << 4));
          }
        } else {
          uint16_t *p = reinterpret_cast<uint16_t *>(a.y) + row0 * a.ldy + col0 + lane;
          const bool in0 = col0 + lane < a.co, in1 = col0 + 32 + lane < a.co;
          const int rows = (int)min((int64_t)32, a.rows - row0);
#pragma unroll 8
          for (int r = 0; r < rows; r++) {
            if (in0) p[r * a.ldy] = *single(r, lane);
            if (in1) p[r * a.ldy + 32] = *single(r, lane + 32);
          }
        }
        __syncwarp();
      }
      if (half * 64 >= BN) {  // a tile of one block: the second warps have nothing to read
        if (lane == 0) {
          if (CG == 2)
            sm100::mbar_arrive_cluster(sm100::map_to_rank(tempty0 + 8 * b, 0));
          else
            sm100::mbar_arrive(tempty0 + 8 * b);
        }
      }
      acc++;
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (CG == 2) sm100::cluster_sync();  // no CTA leaves while the other may still signal it or read its tiles
  if (warp == kMmaWarp) {
    sm100::tc_fence_after();
    if (CG == 2)
      sm100::tmem_dealloc_pair(tmem, S::kCols);
    else
      sm100::tmem_dealloc(tmem, S::kCols);
  }
}

template <int DT, int CG, int BN>
int launch(t2sc_ctx *ctx, const DenseArgs &a, std::string &err) {
  using S = Shape<CG, BN>;
  DenseTcArgs t;
  const uint64_t dx[2] = {(uint64_t)a.ci, (uint64_t)a.rows}, dw[2] = {(uint64_t)a.ci, (uint64_t)a.co};
  const uint64_t one = ((uint64_t)a.ci * 2 + 15) / 16 * 16;  // a stride that a single row never uses
  const uint64_t sx[1] = {a.rows > 1 ? (uint64_t)a.ldx * 2 : one}, sw[1] = {a.co > 1 ? (uint64_t)a.ldw * 2 : one};
  const uint32_t bx[2] = {kBK, kTileM}, bw[2] = {kBK, (uint32_t)S::kWRows};
  T2SC_TRY(tensormap_16bit(&t.map_x, DT, 2, a.x, dx, sx, bx, err));
  T2SC_TRY(tensormap_16bit(&t.map_w, DT, 2, a.w, dw, sw, bw, err));
  t.res = a.res, t.y = a.y, t.bias = a.bias, t.ldr = a.ldr, t.ldy = a.ldy, t.rows = a.rows, t.co = a.co;
  t.k_iters = (a.ci + kBK - 1) / kBK, t.act = a.act, t.err = ctx->d_wait;
  t.m_tiles = (int)((a.rows + kTileM * CG - 1) / (kTileM * CG)), t.n_tiles = (a.co + BN - 1) / BN;
  auto on16 = [&](const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a.rows <= 1 || ld % 8 == 0); };
  t.vec = on16(a.y, a.ldy) && (!a.res || on16(a.res, a.ldr));
  // 32 MB of w a band
  const int64_t column_tile = (int64_t)BN * a.ci * 2;
  t.band = (int)std::min<int64_t>(t.n_tiles, std::max<int64_t>(1, ((int64_t)32 << 20) / column_tile));
  const int64_t tiles = (int64_t)t.m_tiles * t.n_tiles, most = ctx->num_sms / CG;
  t.slots = (int)(tiles < most ? tiles : most);
  auto kernel = dense_tc_kernel<DT, CG, BN>;
  static std::atomic<uint64_t> allowed{0};
  T2SC_TRY(allow_smem(ctx, kernel, (int)S::kSmem, allowed, err));
  T2SC_CUDA(launch_overlapped(kernel, (int64_t)t.slots * CG, kThreads, S::kSmem, ctx->stream, CG, t), "dense_linear");
  T2SC_LAUNCHED(ctx, "dense_linear");
  return T2SC_OK;
}

// The tile shapes: rounds of tiles x (a K step x K steps + the tile's own) + the
// launch, the first tiles' way in and the last one's epilogue, in microseconds
// as measured with weights out of L2 (128..4736 rows, 1024..8192 -> 512..6144:
// within 8 %; few tiles over a long K axis, where the K-split kernel is the
// faster one, up to 29 %: profiles/attention_block_models.txt). A step is bound by what an SM takes in, 55 of its 64 bytes a
// clock from L2, but for the pair's 256 columns, where the products are close.
struct Option {
  int cg, bn;
  double step, rest;
};
constexpr Option kOptions[] = {{2, 256, 0.31, 5.5}, {2, 128, 0.24, 3.7}, {1, 128, 0.25, 2.9}, {1, 64, 0.218, 3.1}};
constexpr double kTile = 0.6;

template <int DT>
int launch_dt(t2sc_ctx *ctx, const DenseArgs &a, std::string &err) {
  int best = 0;
  dense_tc_us(ctx, a, &best);
  switch (best) {
    case 0: return launch<DT, 2, 256>(ctx, a, err);
    case 1: return launch<DT, 2, 128>(ctx, a, err);
    case 2: return launch<DT, 1, 128>(ctx, a, err);
    default: return launch<DT, 1, 64>(ctx, a, err);
  }
}

}  // namespace

double dense_tc_us(t2sc_ctx *ctx, const DenseArgs &a, int *best) {
  const double k_iters = (a.ci + kBK - 1) / kBK;
  double least = 1e300;
  for (int i = 0; i < 4; i++) {
    const Option &o = kOptions[i];
    const int64_t tiles = ((a.rows + kTileM * o.cg - 1) / (kTileM * o.cg)) * ((a.co + o.bn - 1) / o.bn), slots = ctx->num_sms / o.cg;
    const double us = (double)((tiles + slots - 1) / slots) * (k_iters * o.step + kTile) + o.rest;
    if (us < least) least = us, *best = i;
  }
  return least;
}

bool dense_tc_takes(const DenseArgs &a, int dtype) {
  auto on16 = [](const void *p, int64_t ld, int64_t rows) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || ld % 8 == 0);
  };
  return dtype != T2SC_DT_F32 && on16(a.x, a.ldx, a.rows) && on16(a.w, a.ldw, a.co);
}

int dense_tc(t2sc_ctx *ctx, const DenseArgs &a, int dtype, std::string &err) {
  return dtype == T2SC_DT_BF16 ? launch_dt<T2SC_DT_BF16>(ctx, a, err) : launch_dt<T2SC_DT_F16>(ctx, a, err);
}

}  // namespace t2sc
