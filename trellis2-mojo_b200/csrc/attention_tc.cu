// Ragged softmax attention on the tensor cores, for 16-bit rows that start on
// 16 bytes and head dims that are multiples of 8 up to 128.
//
// A CTA owns NT blocks of 128 queries of one head and walks its sequence's
// keys. TMA brings the query blocks once and blocks of 128 K and V rows
// through a ring of shared-memory slots (heads are a dimension of the tensor
// map: channels past head_dim read as zero). One thread issues the
// products, for a unit of 64 keys at a time:
//   S = Q K^T   tcgen05.mma, both operands from shared memory, f32 S in TMEM
//   O += P V    A = P from TMEM, B = V as it lies (channels contiguous:
//               MN-major), f32 O in TMEM
// and a warpgroup per query block, one thread a row, turns S into P in
// between: p = 2^(s c - m c), c = scale log2(e), m the running maximum, P
// rounded to the 16-bit type and written over S. The rounding is what the
// tensor cores ask of an operand: half a step of the type, 2^-8 in bf16 and
// 2^-11 in f16, beside the result's own rounding (0.0023 and 0.00029 off 64 bits
// where weights in f32 would be 0.0017 and 0.00021 off). l sums the weights as
// they were before it.
//
// A query block has two S buffers of 64 columns, so that the scores of the
// next unit are there when the softmax of this one is done: O takes up to 128
// columns, two blocks fill the 512 of an SM. (With one buffer of 128 keys a
// block waits for P V and the next Q K^T after every softmax: 3650 clocks a
// block of 128 keys and two query blocks at head_dim 128, of which the
// softmax takes 1850.) With two blocks (NT = 2) one's softmax also runs under
// the other's products, and K and V are read for 256 queries; with one, two
// CTAs share an SM to the same end.
//
// The running maximum that P is relative to is only raised when a row's
// maximum has grown by more than a factor 2^kSlack (then l and O are
// rescaled by the row's thread): before that, weights are up to 2^kSlack and
// the division by l at the end takes the factor out. In f16 the weights also
// carry a factor 2^8, so that small ones stay clear of its subnormals. One
// multiply-add makes an exponent, s c - m c with m c rounded once for the row:
// a factor that all its weights and l share. Above |m c| = 2^kFar that factor
// approaches 2 (f16 overflows), then m c itself overflows; such rows, whose
// scores f32 hardly tells apart, are computed once more at the end by their
// warp, row by row, from differences (s - m) c. (Differences for every row, an
// addition more, took 1203 + 738 tokens, 12 x 128, from 22.4 to 23.5 us and 23024
// from 2470 to 2665; a second loop for such warps 24.4 and 2540.)
//
// Few query blocks: a cluster of up to 8 CTAs splits the keys of one block
// and adds up its partial (m, l, O) through distributed shared memory, in
// rank order: one launch, no workspace, no atomics.
//
// What a block reads past its sequence belongs to another one: scores there
// become -inf, and V's rows there are zeroed in shared memory, since 0 times
// an infinity or a NaN would reach O.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "attention.h"
#include "entry.h"
#include "epilogue.cuh"
#include "sm100.cuh"
#include "tensormap.h"

namespace t2sc {
namespace {

constexpr int kBQ = 128, kBK = 128, kUnit = 64, kFew = 8, kMaxSplits = 8, kFar = 23;
constexpr long long kWaitLimit = 4000000000ll;  // ~2 s of SM clocks

struct TcArgs {
  CUtensorMap map_q, map_k, map_v;
  const char *q, *k, *v;  // for the far rows alone
  char *out;
  int64_t ldq, ldk, ldv, ldo;  // elements
  const int4 *seqs;       // sequences, most keys first: first query row, query rows, first key row, key rows
  const int64_t *blocks;  // [batch + 1] query blocks (of NT * 128) before each sequence
  int batch, heads, head_dim, splits;
  float c;  // scale * log2(e)
  int *err;
  // seqs and blocks of a batch of up to kFew sequences: no memory read away
  int4 few_seqs[kFew];
  int few_blocks[kFew + 1];
};

template <int DP, int NT>
struct Shape {
  static constexpr int kTile = 128 * DP * 2;  // bytes of a 128-row block
  static constexpr int kSlots = NT == 2 ? (DP == 128 ? 5 : 8) : (DP == 128 ? 2 : 4);
  static constexpr int kExtra = 2048;         // barriers, m and l of the rows
  static constexpr size_t kSmem = 1024 + (size_t)(NT + kSlots) * kTile + kExtra;
  static constexpr int kThreads = 128 * (NT + 1);
  static constexpr uint32_t kCols = NT == 2 ? 512 : 256;
};

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort, int *err) {
  bool ok = sm100::mbar_test_wait(bar, parity);
  if (__all_sync(0xffffffffu, ok)) return true;
  if (!ok) ok = sm100::mbar_wait_bounded(bar, parity, abort, err, kDevErrTimeout, kWaitLimit);
  return __all_sync(0xffffffffu, ok);
}

template <class T>
__device__ __forceinline__ T uniform(T v) {
  return __shfl_sync(0xffffffffu, v, 0);
}

__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ float ld_cluster1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// The rows of a warp in `rows` over `keys` keys from differences (s - m) c, one
// after the other: 8 channels a lane, G lanes a key, as in attention_rows.cu. A
// row's values go to `out`, divided by their sum, or with its maximum and sum to
// the partial sums. q, out and the sums are those of the warp's first row,
// `row0` of the block.
template <int DT, int DP>
__device__ __noinline__ void far_rows(uint32_t rows, const char *q, int64_t ldq, const char *k, int64_t ldk, const char *v, int64_t ldv,
                                      int keys, int head_dim, float c, char *out, int64_t ldo, float4 *part, int row0, float *row_m,
                                      float *row_l) {
  constexpr int G = DP / 8, kKeys = 32 / G, kSteps = 4;
  const int lane = threadIdx.x & 31, sub = lane % G, group = lane / G;
  const bool in = sub * 8 < head_dim;
  auto load8 = [&](const char *p, bool there) {
    return there && in ? *(reinterpret_cast<const uint4 *>(p) + sub) : make_uint4(0, 0, 0, 0);
  };
#pragma unroll 1
  for (; rows; rows &= rows - 1) {
    const int r = __ffs(rows) - 1;
    float m = -INFINITY, l = 0.f, o[8], a[8], b[8];
    unpack8<DT>(load8(q + r * ldq * 2, true), a);
#pragma unroll
    for (int z = 0; z < 8; z++) o[z] = 0.f;
#pragma unroll 1
    for (int64_t j0 = group; j0 - group < keys; j0 += kKeys * kSteps) {
      uint4 kr[kSteps], vr[kSteps];
      float s[kSteps], top = m;
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        const int64_t j = j0 + i * kKeys;
        kr[i] = load8(k + j * ldk * 2, j < keys), vr[i] = load8(v + j * ldv * 2, j < keys);
      }
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        unpack8<DT>(kr[i], b);
        s[i] = 0.f;
#pragma unroll
        for (int z = 0; z < 8; z++) s[i] += a[z] * b[z];
#pragma unroll
        for (int d = G / 2; d > 0; d >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
        if (j0 + i * kKeys >= keys) s[i] = -INFINITY;
        top = fmaxf(top, s[i]);
      }
      const float from = top == -INFINITY ? 0.f : top;
      if (top > m) {
        const float f = ex2((m - top) * c);
        m = top, l *= f;
#pragma unroll
        for (int z = 0; z < 8; z++) o[z] *= f;
      }
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        const float p = ex2((s[i] - from) * c);
        unpack8<DT>(vr[i], b);
        l += p;
#pragma unroll
        for (int z = 0; z < 8; z++) o[z] += p * b[z];
      }
    }
    float top = m;
#pragma unroll
    for (int d = G; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float f = m == top ? 1.f : ex2((m - top) * c);
    l *= f;
#pragma unroll
    for (int d = G; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
    for (int z = 0; z < 8; z++) {
      o[z] *= f;
#pragma unroll
      for (int d = G; d < 32; d <<= 1) o[z] += __shfl_xor_sync(0xffffffffu, o[z], d);
    }
    if (group == 0 && in) {
      if (out) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int z = 0; z < 8; z++) o[z] *= inv;
        *(reinterpret_cast<uint4 *>(out + r * ldo * 2) + sub) =
            make_uint4(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]), pack2<DT>(o[4], o[5]), pack2<DT>(o[6], o[7]));
      } else {
        const int row = row0 + r, swizzle = row & (DP / 4 - 1);
        part[row * (DP / 4) + ((sub * 2) ^ swizzle)] = make_float4(o[0], o[1], o[2], o[3]);
        part[row * (DP / 4) + ((sub * 2 + 1) ^ swizzle)] = make_float4(o[4], o[5], o[6], o[7]);
      }
    }
    if (!out && lane == 0) row_m[r] = top, row_l[r] = l;
  }
}

template <int DT, int DP, int NT>
__global__ void __launch_bounds__(Shape<DP, NT>::kThreads, NT == 2 ? 1 : 2) attention_tc_kernel(const __grid_constant__ TcArgs a) {
  using S = Shape<DP, NT>;
  constexpr int NS = S::kSlots, kSub = DP / 64;
  constexpr float kSlack = DT == T2SC_DT_F16 ? 7.f : 8.f, kLift = DT == T2SC_DT_F16 ? 8.f : 0.f;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *ring = smem + NT * S::kTile;
  float *row_m = reinterpret_cast<float *>(ring + NS * S::kTile), *row_l = row_m + 128;  // split sums
  uint64_t *bars = reinterpret_cast<uint64_t *>(row_l + 128);
  // bars: q_full[NT], s_full[NT][2], o_prev[NT], o_full[NT], ready[2], full[NS], empty[NS]
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 5 * NT + 2 + 2 * NS);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *where = reinterpret_cast<int *>(tmem_slot + 2);  // the CTA's work
  const uint32_t qsm = sm100::smem_u32(smem), rsm = sm100::smem_u32(ring), bar0 = sm100::smem_u32(bars);
  const uint32_t q_full = bar0, s_full = q_full + 8 * NT, o_prev = s_full + 16 * NT, o_full = o_prev + 8 * NT;
  const uint32_t ready = o_full + 8 * NT, full0 = ready + 16, empty0 = full0 + 8 * NS;
  // lane 0's value is every lane's: the compiler may keep it in uniform registers
  const int warp = uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31, wg = warp >> 2;
  constexpr int kTmaWarp = 4 * NT, kMmaWarp = 4 * NT + 1, kFeedWarp = 4 * NT + 2;

  if (warp == kTmaWarp && lane == 0) {
    sm100::tma_prefetch(&a.map_q);
    sm100::tma_prefetch(&a.map_k);
    sm100::tma_prefetch(&a.map_v);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < NT; i++) {
      sm100::mbar_init(q_full + 8 * i, 1);
      for (int b = 0; b < 2; b++) sm100::mbar_init(s_full + 16 * i + 8 * b, 1);
      sm100::mbar_init(o_prev + 8 * i, 1);
      sm100::mbar_init(o_full + 8 * i, 1);
    }
    // the CTA's sequence, head and query block: blocks of a head are neighbours, heads of a sequence follow
    const int id = (int)blockIdx.x / a.splits;
    int4 seq;
    int first, n;
    if (a.batch <= kFew) {
      int lo = 0;
      while (lo + 1 < a.batch && a.few_blocks[lo + 1] * a.heads <= id) lo++;
      seq = a.few_seqs[lo];
      first = a.few_blocks[lo], n = a.few_blocks[lo + 1] - first;
    } else {
      int lo = 0, hi = a.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(a.blocks + mid) * a.heads <= id)
          lo = mid;
        else
          hi = mid - 1;
      }
      seq = __ldg(a.seqs + lo);
      first = (int)__ldg(a.blocks + lo), n = (int)__ldg(a.blocks + lo + 1) - first;
    }
    const int local = id - first * a.heads, head = local / n, block = local - head * n;
    where[0] = head;
    where[1] = seq.x + block * (NT * kBQ);          // first query row
    where[2] = seq.y - block * (NT * kBQ);          // query rows left
    where[3] = seq.z;
    where[4] = seq.w;
    for (int s = 0; s < NS; s++) {
      sm100::mbar_init(full0 + 8 * s, 1);
      sm100::mbar_init(empty0 + 8 * s, 1);
    }
    // a unit's P of every query block (4 warps each), and its V and the next K
    for (int b = 0; b < 2; b++) sm100::mbar_init(ready + 8 * b, (NT == 2 && where[2] > kBQ ? 8 : 4) + 1);
    *abort = 0;
    sm100::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    sm100::tmem_alloc(sm100::smem_u32(tmem_slot), S::kCols);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  sm100::next_kernel_may_start();
  sm100::previous_kernel_done();
  const uint32_t tmem = uniform(*tmem_slot);
  const int head = uniform(where[0]), q0 = uniform(where[1]), here = min(uniform(where[2]), NT * kBQ), kv0 = uniform(where[3]),
            kv_len = uniform(where[4]);
  const int split = a.splits > 1 ? uniform((int)sm100::cluster_rank()) : 0;
  const int all_tiles = (kv_len + kBK - 1) / kBK, per = (all_tiles + a.splits - 1) / a.splits;
  const int t0 = min(split * per, all_tiles), n = min(t0 + per, all_tiles) - t0;  // this CTA's key blocks
  const int keys = min(kv_len - t0 * kBK, n * kBK), units = (keys + kUnit - 1) / kUnit;
  const int nt = NT == 2 && here > kBQ ? 2 : 1;                                     // query blocks with rows
  const uint32_t s_tmem = tmem, o_tmem = tmem + NT * 128;
  const int ksteps = (a.head_dim + 15) / 16;

  if (wg == NT) {
    if (warp == kTmaWarp && n > 0) {
      // ------------------------------- TMA --------------------------------
      bool ok = true;
      uint32_t it = 0;
      if (lane == 0) {
        for (int i = 0; i < nt; i++) {
          sm100::mbar_arrive_expect_tx(q_full + 8 * i, S::kTile);
          for (int h = 0; h < kSub; h++)
            sm100::tma_load_3d(qsm + i * S::kTile + h * 16384, &a.map_q, h * 64, head, q0 + i * kBQ, q_full + 8 * i);
        }
      }
      for (int j = 0; j < 2 * n && ok; j++) {  // K and V blocks in turn
        const uint32_t s = it % NS;
        if (!warp_wait(empty0 + 8 * s, ((it / NS) & 1) ^ 1, abort, a.err)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          sm100::mbar_arrive_expect_tx(full0 + 8 * s, S::kTile);
          const void *map = j & 1 ? &a.map_v : &a.map_k;
          for (int h = 0; h < kSub; h++)
            sm100::tma_load_3d(rsm + s * S::kTile + h * 16384, map, h * 64, head, kv0 + (t0 + (j >> 1)) * kBK, full0 + 8 * s);
        }
        __syncwarp();
        it++;
      }
      if (lane == 0) {  // every copy asked for has landed before shared memory is used again or given up
        for (int i = 0; i < nt; i++) sm100::mbar_wait_cycles(q_full + 8 * i, 0, kWaitLimit / 8);
        for (uint32_t i = it > NS ? it - NS : 0; i < it; i++)
          sm100::mbar_wait_cycles(full0 + 8 * (i % NS), (i / NS) & 1, kWaitLimit / 8);
      }
      __syncwarp();
    } else if (warp == kMmaWarp && n > 0) {
      // ------------------------------- MMA --------------------------------
      // One thread waits and issues. A wait, even on a phase that has
      // completed, stands behind the thread's own products in the queue (~150
      // clocks), so there is one a unit: the barrier that counts the warps
      // that have written P and the feeding warp that has seen the loads. (A
      // thread for each query block hides its waits under the other's
      // products, but the exponentials of the softmax warps on its part of
      // the SM wait behind the products in the same queue: 1250 clocks later
      // than the others.)
      if (sm100::elect_one()) {
        constexpr uint32_t fmt = DT == T2SC_DT_BF16 ? 1 : 0;
        const uint32_t idesc_s = sm100::instr_desc(fmt, kUnit);
        const uint32_t idesc_o = sm100::instr_desc(fmt, ksteps * 16) | sm100::kInstrBMnMajor;
        // descriptors: both operands' high words are the same (1024 bytes between 8-row atoms, 128-byte swizzle)
        const uint64_t dq0 = sm100::smem_desc(qsm, 128);
        const uint32_t hi = (uint32_t)(dq0 >> 32), q_lo = (uint32_t)dq0, k_lo = (uint32_t)sm100::smem_desc(rsm, 128),
                       v_lo = (uint32_t)sm100::smem_desc_mn(rsm, 16384);
        constexpr uint32_t kTile16 = S::kTile >> 4, kUnit16 = kUnit * 128 >> 4;
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
          ok = ok && sm100::mbar_wait_bounded(bar, parity, abort, a.err, kDevErrTimeout, kWaitLimit);
          sm100::tc_fence_after();
        };
        auto scores = [&](int i, int b, uint32_t kslot, bool done) {  // S into buffer b = the unit's half of its block
          const uint32_t dq = q_lo + i * kTile16, dk = k_lo + kslot * kTile16 + b * kUnit16, d = s_tmem + i * 128 + b * kUnit;
          if (ksteps == DP / 16) {
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk++)
              sm100::mma_f16_lo(d, dq + (kk >> 2) * 1024 + (kk & 3) * 2, dk + (kk >> 2) * 1024 + (kk & 3) * 2, hi, idesc_s, kk > 0);
          } else {
#pragma unroll 1
            for (int kk = 0; kk < ksteps; kk++)
              sm100::mma_f16_lo(d, dq + (kk >> 2) * 1024 + (kk & 3) * 2, dk + (kk >> 2) * 1024 + (kk & 3) * 2, hi, idesc_s, kk > 0);
          }
          sm100::mma_commit(s_full + 16 * i + 8 * b);
          if (done && i == nt - 1) sm100::mma_commit(empty0 + 8 * kslot);  // the block's last unit, for the last query block
        };
        // ring position of the V block at hand, and of the K block behind it
        uint32_t vslot = 1 % NS, kslot = 2 % NS;
        auto unit = [&](int u, int b, bool last) {
          const uint32_t dv = v_lo + vslot * kTile16 + b * kUnit16;
          wait(ready + 8 * b, (u >> 1) & 1);
          if (!ok) return;
#pragma unroll
          for (int i = 0; i < NT; i++) {
            if (i >= nt) break;
            const uint32_t o = o_tmem + i * DP, p = s_tmem + i * 128 + b * kUnit;
            if (!last) {
#pragma unroll
              for (int kk = 0; kk < kUnit / 16; kk++) sm100::mma_f16_ts_lo(o, p + kk * 8, dv + kk * 128, hi, idesc_o, u + kk > 0);
            } else {
              const int steps = (keys - u * kUnit + 15) / 16;
#pragma unroll 1
              for (int kk = 0; kk < steps; kk++) sm100::mma_f16_ts_lo(o, p + kk * 8, dv + kk * 128, hi, idesc_o, u + kk > 0);
            }
            if (i == nt - 1 && (b == 1 || last)) sm100::mma_commit(empty0 + 8 * vslot);
            if (u + 2 < units)
              scores(i, b, kslot, b == 1 || u + 2 == units - 1);
            else
              sm100::mma_commit((last ? o_full : o_prev) + 8 * i);
          }
        };
        wait(full0, 0);
        for (int u = 0; u < min(units, 2); u++)
          for (int i = 0; i < nt; i++) {
            if (u == 0) wait(q_full + 8 * i, 0);
            if (ok) scores(i, u, 0, u == 1 || units == 1);
          }
#pragma unroll 1
        for (int u = 0; u < units && ok; u += 2) {
          unit(u, 0, u + 1 >= units);
          if (u + 1 < units && ok) unit(u + 1, 1, u + 2 >= units);
          vslot = kslot + 1 == NS ? 0 : kslot + 1;
          kslot = vslot + 1 == NS ? 0 : vslot + 1;
        }
        // all issued MMAs retire before TMEM and shared memory are given up: in
        // the regular case o_full told so; after an abort wait for a last commit
        if (!ok) {
          sm100::mma_commit(o_full);
          sm100::mbar_wait_cycles(o_full, 0, kWaitLimit / 8);
        }
      }
    } else if (warp == kFeedWarp && n > 0) {
      // ------------------------------- feed -------------------------------
      // Joins a unit's barrier once its V block and the K block of two units
      // on are there, and zeros the V rows behind the last key, up to the 16
      // that a product step takes.
      // Every load is waited for in turn, the first K too: a wait for a slot's
      // next phase is only good once the one before it has completed.
      const bool first = warp_wait(full0, 0, abort, a.err);
      for (int u = 0; u < units && first; u++) {
        if (u > 1 && !warp_wait(ready + 8 * (u & 1), ((u - 2) >> 1) & 1, abort, a.err)) break;  // its last use is over
        if (!(u & 1)) {
          const uint32_t v = u + 1, k = u + 2;  // loads: block j's K is number 2 j, its V 2 j + 1
          if (!warp_wait(full0 + 8 * (v % NS), (v / NS) & 1, abort, a.err)) break;
          if (u + 2 < units && !warp_wait(full0 + 8 * (k % NS), (k / NS) & 1, abort, a.err)) break;
          const int valid = keys - u * kUnit;  // of this block's
          if (valid < kBK && valid % 16) {
            uint8_t *rows = ring + v % NS * S::kTile + valid * 128;
            for (int x = lane; x < (16 - valid % 16) * 8 * kSub; x += 32)
              *reinterpret_cast<uint4 *>(rows + x % kSub * 16384 + x / kSub * 16) = make_uint4(0, 0, 0, 0);
            sm100::fence_proxy_async_smem();
          }
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(ready + 8 * (u & 1));
      }
    }
    __syncwarp();
    if (NT == 1 && a.splits > 1) {  // the softmax warps' two barriers around the sums' exchange
      sm100::cluster_sync();
      sm100::cluster_sync();
    }
  } else {
    // ----------------------------- softmax ------------------------------
    const int i = wg, quad = warp & 3;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t st = s_tmem + i * 128 + lanes, ot = o_tmem + i * DP + lanes;
    const bool live = i < nt && i * kBQ + quad * 32 < here;  // a warp without rows leaves P as it is
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    if (i < nt) {
      for (int u = 0; u < units; u++) {
        const uint32_t b = u & 1, su = st + b * kUnit;
        if (!warp_wait(s_full + 16 * i + 8 * b, (u >> 1) & 1, abort, a.err)) {
          ok = false;
          break;
        }
        sm100::tc_fence_after();
        if (live) {
          float s[kUnit];
          sm100::tmem_ld32(su, reinterpret_cast<uint32_t *>(s));
          sm100::tmem_ld32(su + 32, reinterpret_cast<uint32_t *>(s) + 32);
          sm100::tmem_ld_wait();
          const int valid = keys - u * kUnit;
          if (valid < kUnit) {
#pragma unroll
            for (int q = 0; q < kUnit; q++) s[q] = q < valid ? s[q] : -INFINITY;
          }
          // P is computed relative to the maximum so far while this unit's is
          // still being found, and once more if that turns out to be too low
          // (always in the first unit, hardly ever later).
          float l0, l1;
          for (;;) {
            const float base = kLift - (m == -INFINITY ? 0.f : m * a.c);
            const uint64_t c2 = sm100::pack_f32x2(a.c, a.c), base2 = sm100::pack_f32x2(base, base);
            uint64_t sum[2] = {0, 0};
            float top[4] = {m, m, m, m};
#pragma unroll
            for (int q = 0; q < kUnit; q += 32) {
              uint32_t p[16];
#pragma unroll
              for (int z = 0; z < 32; z += 2) {
                float p0, p1;
                sm100::unpack_f32x2(sm100::fma_f32x2(sm100::pack_f32x2(s[q + z], s[q + z + 1]), c2, base2), p0, p1);
                p0 = ex2(p0), p1 = ex2(p1);
                sum[z >> 1 & 1] = sm100::add_f32x2(sum[z >> 1 & 1], sm100::pack_f32x2(p0, p1));
                p[z / 2] = pack2<DT>(p0, p1);
                top[z >> 1 & 3] = fmaxf(fmaxf(top[z >> 1 & 3], s[q + z]), s[q + z + 1]);
              }
              sm100::tmem_st16(su + q / 2, p);
            }
            sm100::unpack_f32x2(sm100::add_f32x2(sum[0], sum[1]), l0, l1);
            const float mn = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            if (!__any_sync(0xffffffffu, (mn - m) * a.c > kSlack)) break;
            const float f = mn > m ? ex2((m - mn) * a.c) : 1.f;
            m = mn;
            l *= f;
            if (u > 0) {
              // O is complete once P V of the last unit is: the next unit's scores were issued behind it
              if (u + 1 < units)
                ok = warp_wait(s_full + 16 * i + 8 * (b ^ 1), ((u + 1) >> 1) & 1, abort, a.err);
              else
                ok = warp_wait(o_prev + 8 * i, 0, abort, a.err);
              if (!ok) break;
              sm100::tc_fence_after();
#pragma unroll 1
              for (int q = 0; q < DP; q += 32) {
                uint32_t o[32];
                sm100::tmem_ld32(ot + q, o);
                sm100::tmem_ld_wait();
#pragma unroll
                for (int z = 0; z < 32; z++) o[z] = __float_as_uint(__uint_as_float(o[z]) * f);
                sm100::tmem_st16(ot + q, o);
                sm100::tmem_st16(ot + q + 16, o + 16);
              }
            }
          }
          if (!ok) break;
          l += l0 + l1;
          sm100::tmem_st_wait();
        }
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(ready + 8 * b);
      }
      if (n > 0 && ok) ok = warp_wait(o_full + 8 * i, 0, abort, a.err);
      sm100::tc_fence_after();
    }
    const bool have = n > 0 && ok;  // O holds sums
    const int row = quad * 32 + lane;
    const uint32_t far = __ballot_sync(
        0xffffffffu, have && live && i * kBQ + row < here && m != -INFINITY && !(fabsf(m * a.c) < (float)(1 << kFar)));
    auto redo = [&](char *out, float4 *part) {
      const int64_t at = (int64_t)head * a.head_dim, key = (int64_t)kv0 + (int64_t)t0 * kBK, first = (int64_t)q0 + i * kBQ + quad * 32;
      far_rows<DT, DP>(far, a.q + (first * a.ldq + at) * 2, a.ldq, a.k + (key * a.ldk + at) * 2, a.ldk, a.v + (key * a.ldv + at) * 2, a.ldv,
                       keys, a.head_dim, a.c, out, a.ldo, part, quad * 32, row_m + quad * 32, row_l + quad * 32);
    };
    if (a.splits == 1) {
      if (live && ok) {
        // the query block's shared memory is free now: 32 rows x 64 channels at a time through it
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint8_t *stage = smem + i * S::kTile + quad * 4096;
        const int crow = lane >> 3, cch = lane & 7;
        const int64_t row0 = (int64_t)q0 + i * kBQ + quad * 32;
        const int rows_here = here - i * kBQ - quad * 32;
#pragma unroll 1
        for (int c0 = 0; c0 < a.head_dim; c0 += 64) {
          float v[64];
          if (have) {
            sm100::tmem_ld32(ot + c0, reinterpret_cast<uint32_t *>(v));
            sm100::tmem_ld32(ot + c0 + 32, reinterpret_cast<uint32_t *>(v) + 32);
            sm100::tmem_ld_wait();
          }
#pragma unroll
          for (int c = 0; c < 8; c++) {
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; e++) z[e] = have ? v[c * 8 + e] * inv : 0.f;
            *reinterpret_cast<uint4 *>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) =
                make_uint4(pack2<DT>(z[0], z[1]), pack2<DT>(z[2], z[3]), pack2<DT>(z[4], z[5]), pack2<DT>(z[6], z[7]));
          }
          __syncwarp();
#pragma unroll
          for (int z = 0; z < 8; z++) {
            const int r = z * 4 + crow, col = c0 + cch * 8;
            if (r < rows_here && col < a.head_dim)
              *reinterpret_cast<uint4 *>(a.out + ((row0 + r) * a.ldo + (int64_t)head * a.head_dim + col) * 2) =
                  *reinterpret_cast<const uint4 *>(stage + r * 128 + ((cch ^ (r & 7)) << 4));
          }
          __syncwarp();
        }
        if (far) redo(a.out + (row0 * a.ldo + (int64_t)head * a.head_dim) * 2, nullptr);
      }
    } else if (NT == 1) {
      // partial sums for the cluster: rows of f32 over the ring, 16-byte chunks swizzled by row
      row_m[row] = m, row_l[row] = l;
      if (live && have) {
        float4 *part = reinterpret_cast<float4 *>(ring) + row * (DP / 4);
#pragma unroll 1
        for (int c0 = 0; c0 < a.head_dim; c0 += 32) {
          float v[32];
          sm100::tmem_ld32(ot + c0, reinterpret_cast<uint32_t *>(v));
          sm100::tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 8; c++)
            part[(c0 / 4 + c) ^ (row & (DP / 4 - 1))] = make_float4(v[c * 4], v[c * 4 + 1], v[c * 4 + 2], v[c * 4 + 3]);
        }
        __syncwarp();
        if (far) redo(nullptr, reinterpret_cast<float4 *>(ring));
      }
      __syncwarp();
      sm100::cluster_sync();
      const uint32_t m0 = sm100::smem_u32(row_m), l0 = sm100::smem_u32(row_l);
      const int chunks = a.head_dim / 4, items = here * chunks;
      for (int x = split * 128 + (int)threadIdx.x; x < items; x += a.splits * 128) {
        const int r = x / chunks, c = x % chunks;
        float top = -INFINITY;
        for (int z = 0; z < a.splits; z++) top = fmaxf(top, ld_cluster1(sm100::map_to_rank(m0 + 4 * r, z)));
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
        const uint32_t at = rsm + (uint32_t)(r * (DP / 4) + (c ^ (r & (DP / 4 - 1)))) * 16;
        for (int z = 0; z < a.splits; z++) {
          const float lz = ld_cluster1(sm100::map_to_rank(l0 + 4 * r, z));
          if (lz == 0.f) continue;  // no keys there, or every score -inf
          const float w = ex2((ld_cluster1(sm100::map_to_rank(m0 + 4 * r, z)) - top) * a.c);
          const float4 v = ld_cluster(sm100::map_to_rank(at, z));
          sum += w * lz;
          o.x += w * v.x, o.y += w * v.y, o.z += w * v.z, o.w += w * v.w;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2 *>(a.out + (((int64_t)q0 + r) * a.ldo + (int64_t)head * a.head_dim + c * 4) * 2) =
            make_uint2(pack2<DT>(o.x * inv, o.y * inv), pack2<DT>(o.z * inv, o.w * inv));
      }
      __syncwarp();
      sm100::cluster_sync();  // no CTA leaves before the others have read its sums
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, S::kCols);
  }
}

template <int DT, int DP, int NT>
int launch(t2sc_seqs *s, const AttnArgs &a, int splits, std::string &err) {
  using S = Shape<DP, NT>;
  t2sc_ctx *ctx = s->ctx;
  auto kernel = attention_tc_kernel<DT, DP, NT>;
  TcArgs t;
  const uint64_t D = a.head_dim, H = a.heads;
  auto encode = [&](CUtensorMap *m, const char *p, int64_t ld, int64_t rows) -> int {
    const uint64_t dims[3] = {D, H, (uint64_t)std::max<int64_t>(rows, 1)};
    const uint64_t strides[2] = {D * 2, rows > 1 ? (uint64_t)ld * 2 : D * H * 2};
    const uint32_t box[3] = {64, 1, 128};
    return tensormap_16bit(m, DT, 3, p, dims, strides, box, err);
  };
  T2SC_TRY(encode(&t.map_q, a.q, a.ldq, s->q_rows));
  const bool keys = s->kv_off[s->batch] > s->kv_off[0];
  T2SC_TRY(encode(&t.map_k, keys ? a.k : a.q, keys ? a.ldk : a.ldq, keys ? s->kv_rows : 1));  // never read without keys
  T2SC_TRY(encode(&t.map_v, keys ? a.v : a.q, keys ? a.ldv : a.ldq, keys ? s->kv_rows : 1));
  t.q = a.q, t.k = a.k, t.v = a.v, t.out = a.out;
  t.ldq = a.ldq, t.ldk = a.ldk, t.ldv = a.ldv, t.ldo = a.ldo;
  t.seqs = s->d_sorted;
  t.blocks = s->d_blocks + (NT == 2 ? 0 : s->batch + 1);
  t.batch = (int)s->batch, t.heads = a.heads, t.head_dim = a.head_dim, t.splits = splits;
  t.c = a.scale * 1.4426950408889634f, t.err = ctx->d_wait;
  const int64_t grid = (NT == 2 ? s->blocks256 : s->blocks128) * a.heads * splits;
  if (grid > INT32_MAX) return fail(ctx, T2SC_ERR_UNSUPPORTED, "attention: too many query blocks in one call");
  for (int b = 0; b <= kFew && b <= s->batch; b++) {
    t.few_blocks[b] = (int)(NT == 2 ? s->few_blocks256[b] : s->few_blocks128[b]);
    if (b < kFew && b < s->batch) t.few_seqs[b] = s->few_seqs[b];
  }
  static std::atomic<uint64_t> allowed{0};
  T2SC_TRY(allow_smem(ctx, kernel, (int)S::kSmem, allowed, err));
  T2SC_CUDA(launch_overlapped(kernel, grid, S::kThreads, S::kSmem, ctx->stream, splits, t), "attention");
  T2SC_LAUNCHED(ctx, "attention");
  return T2SC_OK;
}

template <int DT, int DP>
int launch_dp(t2sc_seqs *s, const AttnArgs &a, std::string &err) {
  // What ends first, in the time that one query block alone on an SM takes
  // for a unit (0.67 us at head_dim 128). A CTA takes its units x what one
  // takes + kFixed to begin and end: with two query blocks a CTA a pair of
  // units takes kPair (0.83 us); with one, and its keys in n parts, two CTAs
  // that share an SM take kShared for a unit of both, and kExchange goes to
  // the parts' exchange. The end is that of the longest sequences' rounds of
  // CTAs, or, where others follow them, of all CTAs' time spread over the SMs
  // and half a CTA, and not before the rounds that they would take with a unit
  // each. 300 queries over 20000 keys, 12 x 128: 71 us with the 6
  // parts this finds, 97 with 8 (two rounds), 95 with 4, 247 with two blocks a
  // CTA; 20 x 300 tokens, 16 x 64: 34 us with one part, 42 with two blocks a
  // CTA; 21888 queries over 1029 keys, 16 x 64: 177 us with one block, 187
  // with two, 12 x 128 163 and 147 (profiles/attention_block_models.txt).
  constexpr double kFixed = 8, kPair = 1.25, kShared = DP == 64 ? 1.25 : 1.6, kExchange = 3;
  const double units = (double)((s->max_kv + kUnit - 1) / kUnit), heads = a.heads, sms = s->ctx->num_sms;
  auto rounds = [&](int64_t blocks, int64_t slots) { return (blocks * a.heads + slots - 1) / slots; };
  double least = (double)rounds(s->long256, s->ctx->num_sms) * (units * (s->long_q > kBQ ? kPair : 1) + kFixed);
  if (s->long256 < s->blocks256) {
    const double all = s->work256 * kPair + s->blocks256 * kFixed;
    least = std::max({least, all * heads / sms + all / s->blocks256 / 2, (double)rounds(s->blocks256, s->ctx->num_sms) * (kPair + kFixed)});
  }
  int best = 0;
  static Clusters<kMaxSplits> table[64];
  const int *at_once = nullptr;
  T2SC_TRY(clusters_at_once(s->ctx, attention_tc_kernel<DT, DP, 1>, Shape<DP, 1>::kThreads, Shape<DP, 1>::kSmem, table, &at_once, err));
  for (int n = 1; n <= kMaxSplits; n++) {
    if (at_once[n] < 1 || (n > 1 && units < 4 * n)) continue;
    const int64_t r = rounds(s->long128, at_once[n]);
    const double part = (double)((int64_t)(units + n - 1) / n), fixed = n > 1 ? kFixed + kExchange : kFixed;
    double cost = (double)(r / 2) * (part * kShared + fixed) + (double)(r % 2) * (part + fixed);
    if (s->long128 < s->blocks128) {
      const double all = s->work128 / n * kShared + s->blocks128 * fixed;  // of two CTAs that share an SM
      cost = std::max({cost, all * heads / (2 * at_once[n]) + all / s->blocks128 / 2,
                       (double)rounds(s->blocks128, 2 * at_once[n]) * (kShared + fixed)});
    }
    if (cost < least) least = cost, best = n;
  }
  return best == 0 ? launch<DT, DP, 2>(s, a, 1, err) : launch<DT, DP, 1>(s, a, best, err);
}

}  // namespace

bool attention_tc_takes(const t2sc_seqs *s, const AttnArgs &a, int dtype) {
  auto on16 = [](const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
  const bool keys = s->kv_off[s->batch] > s->kv_off[0];
  // scores are compared before they are scaled: the scale has to keep their order; scale * log2(e) has to be finite
  return dtype != T2SC_DT_F32 && a.head_dim % 8 == 0 && a.head_dim <= 128 && a.scale > 0.f && a.scale < 1e38f && on16(a.q, a.ldq) &&
         on16(a.out, a.ldo) && (!keys || (on16(a.k, a.ldk) && on16(a.v, a.ldv)));
}

int attention_tc(t2sc_seqs *s, const AttnArgs &a, int dtype, std::string &err) {
  if (dtype == T2SC_DT_BF16)
    return a.head_dim <= 64 ? launch_dp<T2SC_DT_BF16, 64>(s, a, err) : launch_dp<T2SC_DT_BF16, 128>(s, a, err);
  return a.head_dim <= 64 ? launch_dp<T2SC_DT_F16, 64>(s, a, err) : launch_dp<T2SC_DT_F16, 128>(s, a, err);
}

}  // namespace t2sc
