// Ragged softmax attention for sequences of at most kMaxRows queries: a few
// queries over many keys read K and V once and compute next to nothing, so
// HBM bounds the call and tensor-core tiles of 128 queries would be empty
// but for a row.
//
// One warp brings blocks of keys, K and V, into a ring of shared-memory
// stages by TMA: 192 KB of an SM in flight (held in registers instead, a
// third of that, the call ran at half the speed), in one CTA, or in two where
// there are more sequences and heads than SMs. Its 16 or 8 warps take a few
// keys of a block each: 8 channels a lane, G lanes a key, 32 / G keys a step.
// Every group of G lanes keeps its own running maximum, sum and f32 output of
// each query; they are merged over the warp by shuffles, over the CTA's warps
// through shared memory and over the cluster's CTAs, which split the keys,
// through distributed shared memory, in a fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "attention.h"
#include "entry.h"
#include "epilogue.cuh"
#include "sm100.cuh"
#include "tensormap.h"

namespace t2sc {
namespace {

constexpr int kMaxRows = 4, kMaxSplits = 16, kStages = 6;

// W: warps that compute, 16 with one CTA an SM, 8 with two.
template <int W>
struct Shape {
  static constexpr int kWarps = W, kThreads = 32 * (W + 1);
  static constexpr int kStageBytes = W * 2048;  // K block, then V block
  static constexpr size_t kSmem = 1024 + kStages * kStageBytes;
};
constexpr long long kWaitLimit = 4000000000ll;  // ~2 s of SM clocks

struct RowsArgs {
  CUtensorMap map_k, map_v;
  AttnArgs a;
  int splits = 1;
  float c = 0.f;  // scale * log2(e)
  int *err = nullptr;
};

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// Weight of a partial sum with maximum m in one with maximum `to` (>= m):
// partial sums without keys have m = -inf and l = 0.
__device__ __forceinline__ float weight(float m, float to, float c) { return m == to ? 1.f : ex2((m - to) * c); }

// Maxima are of q . k; differences of them are scaled (attention.cu says why).
template <int DT, int G, int R, int W>
__global__ void __launch_bounds__(Shape<W>::kThreads, 16 / W) attention_rows_kernel(const __grid_constant__ RowsArgs x) {
  constexpr int kWarps = W, kThreads = Shape<W>::kThreads, kStageBytes = Shape<W>::kStageBytes;
  constexpr int kKeys = 32 / G, kSteps = 2;              // keys a warp and step, steps a block
  constexpr int kBlock = kWarps * kKeys * kSteps;        // keys a stage: with 16 warps 128 of 64 channels, 64 of 128
  constexpr int kSub = G / 8;                            // 64-channel halves, each rows of 128 bytes
  static_assert(kBlock * 128 * kSub == kStageBytes / 2, "a block fills half a stage");
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bars[2 * kStages];
  __shared__ int abort_flag;
  volatile int *abort = &abort_flag;
  // partial sums, over the ring once it is done with
  struct Partial {
    float o[kWarps][R][G * 8], m[kWarps][R], l[kWarps][R];
    float cta_o[R][G * 8], cta_m[R], cta_l[R];
  };
  static_assert(sizeof(Partial) <= kStages * kStageBytes, "the partial sums fit the ring");
  Partial &part = *reinterpret_cast<Partial *>(ring);
  const AttnArgs &a = x.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % G, group = lane / G;
  const int id = blockIdx.x / x.splits, split = blockIdx.x % x.splits;
  const int head = id % a.heads;
  const int4 seq = __ldg(a.seqs + id / a.heads);
  const int rows = seq.y, keys = seq.w;
  sm100::next_kernel_may_start();
  if (rows == 0) {  // the whole cluster
    sm100::previous_kernel_done();
    return;
  }
  const int all = (keys + kBlock - 1) / kBlock, per = (all + x.splits - 1) / x.splits;
  const int b0 = min(split * per, all), n = min(b0 + per, all) - b0;  // this CTA's blocks
  const uint32_t full0 = sm100::smem_u32(bars), empty0 = full0 + 8 * kStages, ring0 = sm100::smem_u32(ring);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; s++) {
      sm100::mbar_init(full0 + 8 * s, 1);
      sm100::mbar_init(empty0 + 8 * s, kWarps);
    }
    *abort = 0;
    sm100::fence_mbar_init();
  }
  __syncthreads();
  sm100::previous_kernel_done();
  float q[R][8], o[R][8], m[R], l[R];
  if (warp == kWarps) {
    // -------------------------------- TMA --------------------------------
    if (lane == 0) {
      bool ok = true;
      int j = 0;
      for (; j < n && ok; j++) {
        const uint32_t s = j % kStages;
        ok = sm100::mbar_wait_bounded(empty0 + 8 * s, ((j / kStages) & 1) ^ 1, abort, x.err, kDevErrTimeout, kWaitLimit);
        if (!ok) break;
        sm100::mbar_arrive_expect_tx(full0 + 8 * s, kStageBytes);
        const int row = seq.z + (b0 + j) * kBlock;
        const uint32_t dst = ring0 + s * kStageBytes;
        for (int h = 0; h < kSub; h++) {
          sm100::tma_load_3d(dst + h * (kBlock * 128), &x.map_k, h * 64, head, row, full0 + 8 * s);
          sm100::tma_load_3d(dst + kStageBytes / 2 + h * (kBlock * 128), &x.map_v, h * 64, head, row, full0 + 8 * s);
        }
      }
      for (int i = max(0, j - kStages); i < j; i++)  // every copy asked for has landed before shared memory is given up
        sm100::mbar_wait_cycles(full0 + 8 * (i % kStages), (i / kStages) & 1, kWaitLimit / 8);
    }
    __syncwarp();
  } else {
    const bool in = sub * 8 < a.head_dim;  // head_dim % 8 == 0
    const int64_t at = (int64_t)head * a.head_dim + sub * 8;
#pragma unroll
    for (int r = 0; r < R; r++) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (r < rows && in) u = *reinterpret_cast<const uint4 *>(a.q + ((int64_t)(seq.x + r) * a.ldq + at) * 2);
      unpack8<DT>(u, q[r]);
      m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) o[r][j] = 0.f;
    }
    // this lane's chunk of key i of a block: rows of 128 bytes, their 16-byte chunks swizzled by row
    auto chunk = [&](int i) {
      const int row = warp * (kKeys * kSteps) + i * kKeys + group;
      return (sub >> 3) * (kBlock * 128) + row * 128 + (((sub & 7) ^ (row & 7)) << 4);
    };
    for (int j = 0; j < n; j++) {
      const uint32_t s0 = j % kStages;
      const bool ok = sm100::mbar_wait_bounded(full0 + 8 * s0, (j / kStages) & 1, abort, x.err, kDevErrTimeout, kWaitLimit);
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint8_t *kb = ring + s0 * kStageBytes, *vb = kb + kStageBytes / 2;
      const int key0 = (b0 + j) * kBlock + warp * (kKeys * kSteps) + group;
      uint4 kr[kSteps], vr[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        kr[i] = *reinterpret_cast<const uint4 *>(kb + chunk(i));
        vr[i] = *reinterpret_cast<const uint4 *>(vb + chunk(i));
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(empty0 + 8 * s0);  // the block is in registers
      float s[kSteps][R];
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        const bool there = key0 + i * kKeys < keys;
        if (!there) vr[i] = make_uint4(0, 0, 0, 0);  // what lies behind the last key may be anything
        float kf[8];
        unpack8<DT>(kr[i], kf);
#pragma unroll
        for (int r = 0; r < R; r++) {
          s[i][r] = 0.f;
#pragma unroll
          for (int c = 0; c < 8; c++) s[i][r] += q[r][c] * kf[c];
#pragma unroll
          for (int d = G / 2; d > 0; d >>= 1) s[i][r] += __shfl_xor_sync(0xffffffffu, s[i][r], d);
          if (!there) s[i][r] = -INFINITY;
        }
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        float top = m[r];
#pragma unroll
        for (int i = 0; i < kSteps; i++) top = fmaxf(top, s[i][r]);
        const float from = top == -INFINITY ? 0.f : top;
        if (top > m[r]) {
          const float keep = ex2((m[r] - top) * x.c);
          m[r] = top;
          l[r] *= keep;
#pragma unroll
          for (int c = 0; c < 8; c++) o[r][c] *= keep;
        }
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
          s[i][r] = ex2((s[i][r] - from) * x.c);
          l[r] += s[i][r];
        }
      }
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        float vf[8];
        unpack8<DT>(vr[i], vf);
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int c = 0; c < 8; c++) o[r][c] += s[i][r] * vf[c];
      }
    }
  }
  __syncthreads();
  if (warp < kWarps) {
    // the warp's groups
#pragma unroll
    for (int r = 0; r < R; r++) {
      float top = m[r];
#pragma unroll
      for (int d = G; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float w = weight(m[r], top, x.c);
      m[r] = top;
      l[r] *= w;
#pragma unroll
      for (int d = G; d < 32; d <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        o[r][j] *= w;
#pragma unroll
        for (int d = G; d < 32; d <<= 1) o[r][j] += __shfl_xor_sync(0xffffffffu, o[r][j], d);
      }
      if (group == 0) {
#pragma unroll
        for (int j = 0; j < 8; j++) part.o[warp][r][sub * 8 + j] = o[r][j];
      }
      if (lane == 0) part.m[warp][r] = m[r], part.l[warp][r] = l[r];
    }
  }
  __syncthreads();
  // the CTA's warps
  for (int i = threadIdx.x; i < R * G * 8; i += kThreads) {
    const int r = i / (G * 8), c = i % (G * 8);
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; w++) top = fmaxf(top, part.m[w][r]);
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const float f = weight(part.m[w][r], top, x.c);
      sum += f * part.l[w][r], v += f * part.o[w][r][c];
    }
    part.cta_o[r][c] = v;
    if (c == 0) part.cta_m[r] = top, part.cta_l[r] = sum;
  }
  // the cluster's CTAs: each writes a part of the output
  __syncthreads();
  sm100::cluster_sync();
  const uint32_t m0 = sm100::smem_u32(part.cta_m), l0 = sm100::smem_u32(part.cta_l), o0 = sm100::smem_u32(part.cta_o);
  for (int i = split * kThreads + (int)threadIdx.x; i < rows * a.head_dim; i += x.splits * kThreads) {
    const int r = i / a.head_dim, c = i % a.head_dim;
    float top = -INFINITY, sum = 0.f, v = 0.f;
    for (int z = 0; z < x.splits; z++) top = fmaxf(top, ld_cluster(sm100::map_to_rank(m0 + 4 * r, z)));
    for (int z = 0; z < x.splits; z++) {
      const float f = weight(ld_cluster(sm100::map_to_rank(m0 + 4 * r, z)), top, x.c);
      sum += f * ld_cluster(sm100::map_to_rank(l0 + 4 * r, z));
      v += f * ld_cluster(sm100::map_to_rank(o0 + 4 * (r * G * 8 + c), z));
    }
    const float y = sum == 0.f ? 0.f : v / sum;
    char *p = a.out + ((int64_t)(seq.x + r) * a.ldo + (int64_t)head * a.head_dim + c) * 2;
    if (DT == T2SC_DT_BF16)
      *reinterpret_cast<__nv_bfloat16 *>(p) = __float2bfloat16_rn(y);
    else
      *reinterpret_cast<__half *>(p) = __float2half_rn(y);
  }
  __syncwarp();
  sm100::cluster_sync();  // no CTA leaves before the others have read its sums
}

template <int DT, int G, int R, int W>
int launch(t2sc_seqs *s, const AttnArgs &a, std::string &err) {
  constexpr int kThreads = Shape<W>::kThreads;
  constexpr size_t kSmem = Shape<W>::kSmem;
  t2sc_ctx *ctx = s->ctx;
  auto kernel = attention_rows_kernel<DT, G, R, W>;
  static Clusters<kMaxSplits> table[64];
  const int *at_once = nullptr;
  T2SC_TRY(clusters_at_once(ctx, kernel, kThreads, kSmem, table, &at_once, err));
  RowsArgs x;
  x.a = a;
  x.c = a.scale * 1.4426950408889634f;
  x.err = ctx->d_wait;
  constexpr int block = W * (32 / G) * 2;
  // The number of key splits that ends first: rounds of clusters x blocks of
  // the longest sequence a CTA takes (+ 2 of 32 KB for what it costs to begin
  // and end).
  const int64_t ctas = s->batch * a.heads, blocks = (s->max_kv + block - 1) / block;
  int64_t least = INT64_MAX;
  for (int n = 1; n <= kMaxSplits; n++) {
    if (at_once[n] < 1 || (n > 1 && n > blocks)) continue;
    const int64_t cost = ((ctas + at_once[n] - 1) / at_once[n]) * ((blocks + n - 1) / n + 32 / W);
    if (cost < least) least = cost, x.splits = n;
  }
  if (ctas * x.splits > INT32_MAX) return fail(ctx, T2SC_ERR_UNSUPPORTED, "attention: too many sequences and heads in one call");
  const bool any = s->kv_off[s->batch] > s->kv_off[0];
  auto encode = [&](CUtensorMap *map, const char *p, int64_t ld) -> int {
    const uint64_t D = a.head_dim, H = a.heads, rows = any ? s->kv_rows : 1;
    const uint64_t dims[3] = {D, H, rows}, strides[2] = {D * 2, rows > 1 ? (uint64_t)ld * 2 : D * H * 2};
    const uint32_t box[3] = {64, 1, block};
    return tensormap_16bit(map, DT, 3, any ? p : a.q, dims, strides, box, err);  // without keys never read
  };
  T2SC_TRY(encode(&x.map_k, a.k, a.ldk));
  T2SC_TRY(encode(&x.map_v, a.v, a.ldv));
  T2SC_CUDA(launch_overlapped(kernel, ctas * x.splits, kThreads, kSmem, ctx->stream, x.splits, x), "attention");
  T2SC_LAUNCHED(ctx, "attention");
  return T2SC_OK;
}

template <int DT, int G, int R>
int launch_warps(t2sc_seqs *s, const AttnArgs &a, std::string &err) {
  // More sequences and heads than SMs: two CTAs of half the size an SM, one's
  // begin and end beside the other's keys (12 sequences of 600 keys, 16 x 64:
  // 9.5 us, 13.8 with one; 32 of 6000 122 and 130). Fewer, whose keys are
  // split: one (6 of 6000, 12 x 128: 38 us, 43 with two).
  if (s->batch * a.heads > s->ctx->num_sms) return launch<DT, G, R, 8>(s, a, err);
  return launch<DT, G, R, 16>(s, a, err);
}

template <int DT, int G>
int launch_rows(t2sc_seqs *s, const AttnArgs &a, std::string &err) {
  if (s->max_q == 1) return launch_warps<DT, G, 1>(s, a, err);
  if (s->max_q == 2) return launch_warps<DT, G, 2>(s, a, err);
  return launch_warps<DT, G, 4>(s, a, err);
}

template <int DT>
int launch_dim(t2sc_seqs *s, const AttnArgs &a, std::string &err) {
  if (a.head_dim <= 64) return launch_rows<DT, 8>(s, a, err);
  return launch_rows<DT, 16>(s, a, err);
}

}  // namespace

bool attention_rows_takes(const t2sc_seqs *s, const AttnArgs &a, int dtype) {
  return attention_tc_takes(s, a, dtype) && s->max_q <= kMaxRows;
}

int attention_rows(t2sc_seqs *s, const AttnArgs &a, int dtype, std::string &err) {
  return dtype == T2SC_DT_BF16 ? launch_dim<T2SC_DT_BF16>(s, a, err) : launch_dim<T2SC_DT_F16>(s, a, err);
}

}  // namespace t2sc
