// Ragged softmax attention on the tensor cores, for 16-bit rows that start on
// 16 bytes and head dims that are multiples of 8 up to 128.
//
// A CTA owns NT blocks of 128 queries of one head and walks its sequence's
// keys 128 at a time. TMA brings the query blocks once and the K and V blocks
// through a ring of shared-memory slots (heads are a dimension of the tensor
// map: channels past head_dim read as zero). One warp issues the products:
//   S = Q K^T   tcgen05.mma, both operands from shared memory, f32 S in TMEM
//   O += P V    A = P from TMEM, B = V as it lies (channels contiguous:
//               MN-major), f32 O in TMEM
// and a warpgroup per query block, one thread a row, turns S into P in
// between: p = 2^(s c - m c), c = scale log2(e), m the running maximum, P
// rounded to the 16-bit type and written over S. With two blocks (NT = 2) one
// block's softmax runs under the other's products, and K and V are read for
// 256 queries; with one, two CTAs share an SM to the same end.
//
// The running maximum that P is relative to is only raised when a row's
// maximum has grown by more than a factor 2^kSlack (then l and O are
// rescaled by the row's thread): before that, weights are up to 2^kSlack and
// the division by l at the end takes the factor out. In f16 the weights also
// carry a factor 2^8, so that small ones stay clear of its subnormals.
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

constexpr int kBQ = 128, kBK = 128;
constexpr long long kWaitLimit = 4000000000ll;  // ~2 s of SM clocks

struct TcArgs {
  CUtensorMap map_q, map_k, map_v;
  char *out;
  int64_t ldo;            // elements
  const int4 *seqs;       // sequences, most keys first: first query row, query rows, first key row, key rows
  const int64_t *blocks;  // [batch + 1] query blocks (of NT * 128) before each sequence
  int batch, heads, head_dim, splits;
  float c;  // scale * log2(e)
  int *err;
};

template <int DP, int NT>
struct Shape {
  static constexpr int kTile = 128 * DP * 2;  // bytes of a 128-row block
  static constexpr int kSlots = NT == 2 ? (DP == 128 ? 5 : 8) : (DP == 128 ? 2 : 4);
  static constexpr int kExtra = 2048;         // barriers, m and l of the rows
  static constexpr size_t kSmem = 1024 + (size_t)(NT + kSlots) * kTile + kExtra;
  static constexpr int kThreads = 128 * (NT + 1);
  // registers a thread of the softmax warpgroups and of the other one; launched with their mean
  static constexpr int kSoftmaxRegs = NT == 2 ? 224 : 192, kOtherRegs = NT == 2 ? 56 : 64;
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
  // bars: q_full[NT], s_full[NT], p_full[NT], o_full[NT], full[NS], empty[NS], v_dirty, v_clean
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 4 * NT + 2 * NS + 2);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *where = reinterpret_cast<int *>(tmem_slot + 2);  // the CTA's work
  const uint32_t qsm = sm100::smem_u32(smem), rsm = sm100::smem_u32(ring), bar0 = sm100::smem_u32(bars);
  const uint32_t q_full = bar0, s_full = q_full + 8 * NT, p_full = s_full + 8 * NT, o_full = p_full + 8 * NT;
  const uint32_t full0 = o_full + 8 * NT, empty0 = full0 + 8 * NS, v_dirty = empty0 + 8 * NS, v_clean = v_dirty + 8;
  // lane 0's value is every lane's: the compiler may keep it in uniform registers
  const int warp = uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31, wg = warp >> 2;
  constexpr int kTmaWarp = 4 * NT, kMmaWarp = 4 * NT + 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NT; i++) {
      sm100::mbar_init(q_full + 8 * i, 1);
      sm100::mbar_init(s_full + 8 * i, 1);
      sm100::mbar_init(p_full + 8 * i, 4);
      sm100::mbar_init(o_full + 8 * i, 1);
    }
    for (int s = 0; s < NS; s++) {
      sm100::mbar_init(full0 + 8 * s, 1);
      sm100::mbar_init(empty0 + 8 * s, 1);
    }
    sm100::mbar_init(v_dirty, 1);
    sm100::mbar_init(v_clean, 1);
    *abort = 0;
    sm100::fence_mbar_init();
    // the CTA's sequence, head and query block: blocks of a head are neighbours, heads of a sequence follow
    const int64_t id = blockIdx.x / a.splits;
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(a.blocks + mid) * a.heads <= id)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int64_t first = __ldg(a.blocks + lo), n = __ldg(a.blocks + lo + 1) - first, local = id - first * a.heads;
    const int4 seq = __ldg(a.seqs + lo);
    const int head = (int)(local / n), block = (int)(local % n);
    where[0] = head;
    where[1] = seq.x + block * (NT * kBQ);          // first query row
    where[2] = seq.y - block * (NT * kBQ);          // query rows left
    where[3] = seq.z;
    where[4] = seq.w;
  }
  if (warp == kMmaWarp) {
    sm100::tmem_alloc(sm100::smem_u32(tmem_slot), S::kCols);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const int head = uniform(where[0]), q0 = uniform(where[1]), here = min(uniform(where[2]), NT * kBQ), kv0 = uniform(where[3]),
            kv_len = uniform(where[4]);
  const int split = a.splits > 1 ? uniform((int)sm100::cluster_rank()) : 0;
  const int all_tiles = (kv_len + kBK - 1) / kBK, per = (all_tiles + a.splits - 1) / a.splits;
  const int t0 = min(split * per, all_tiles), n = min(t0 + per, all_tiles) - t0;  // this CTA's key blocks
  const int nt = NT == 2 && here > kBQ ? 2 : 1;                                     // query blocks with rows
  const uint32_t s_tmem = tmem, o_tmem = tmem + NT * 128;
  const int ksteps = (a.head_dim + 15) / 16;
  const bool tail = n > 0 && t0 + n == all_tiles && kv_len % 16 != 0;  // the last block's keys end inside a product step

  if (wg == NT) {
    sm100::regs_down<S::kOtherRegs>();
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
      // One thread waits and issues: this role is what everything waits for,
      // and a whole warp's waits and votes, or an election at every
      // instruction, cost it ~100 clocks each (measured per block of keys and
      // two query blocks, head_dim 128: 5000 clocks with elections, 4000
      // with one issuing lane between warp-wide waits).
      if (sm100::elect_one()) {
        constexpr uint32_t fmt = DT == T2SC_DT_BF16 ? 1 : 0;
        const uint32_t idesc_s = sm100::instr_desc(fmt, kBK);
        const uint32_t idesc_o = sm100::instr_desc(fmt, ksteps * 16) | sm100::kInstrBMnMajor;
        const uint64_t dq0 = sm100::smem_desc(qsm, 128), dk0 = sm100::smem_desc(rsm, 128), dv0 = sm100::smem_desc_mn(rsm, 16384);
        uint32_t slot = 0, phase = 0;  // ring position of the next block to consume
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
          ok = ok && sm100::mbar_wait_bounded(bar, parity, abort, a.err, kDevErrTimeout, kWaitLimit);
          sm100::tc_fence_after();
        };
        auto next = [&]() {
          if (++slot == NS) slot = 0, phase ^= 1;
        };
        auto scores = [&](int i, uint32_t at) {
          const uint64_t dq = dq0 + (uint64_t)(i * S::kTile >> 4), dk = dk0 + (uint64_t)(at * S::kTile >> 4);
#pragma unroll 1
          for (int kk = 0; kk < ksteps; kk++) {
            const uint64_t off = (uint64_t)((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
            sm100::mma_f16(s_tmem + i * 128, dq + off, dk + off, idesc_s, kk > 0);
          }
          sm100::mma_commit(s_full + 8 * i);
        };
        wait(full0, 0);
        for (int i = 0; i < nt && ok; i++) {
          wait(q_full + 8 * i, 0);
          if (ok) scores(i, 0);
        }
        if (ok) sm100::mma_commit(empty0);
        next();
        for (int j = 0; j < n && ok; j++) {
          const uint32_t vslot = slot;
          wait(full0 + 8 * vslot, phase);
          if (tail && j == n - 1) sm100::mbar_arrive(v_dirty);
          next();
          const uint32_t kslot = slot;
          const int steps = min((kv_len - (t0 + j) * kBK + 15) / 16, kBK / 16);
          const uint64_t dv = dv0 + (uint64_t)(vslot * S::kTile >> 4);
          for (int i = 0; i < nt && ok; i++) {
            wait(p_full + 8 * i, j & 1);
            if (i == 0 && tail && j == n - 1) wait(v_clean, 0);
            if (!ok) break;
#pragma unroll 1
            for (int kk = 0; kk < steps; kk++)
              sm100::mma_f16_ts(o_tmem + i * DP, s_tmem + i * 128 + kk * 8, dv + (uint64_t)(kk * 2048 >> 4), idesc_o, j + kk > 0);
            if (i == nt - 1) sm100::mma_commit(empty0 + 8 * vslot);
            if (j + 1 < n) {
              if (i == 0) wait(full0 + 8 * kslot, phase);  // K of block j + 1
              if (!ok) break;
              scores(i, kslot);
              if (i == nt - 1) sm100::mma_commit(empty0 + 8 * kslot);
            } else {
              sm100::mma_commit(o_full + 8 * i);
            }
          }
          next();
        }
        // all issued MMAs retire before TMEM and shared memory are given up: in
        // the regular case o_full told so; after an abort wait for a last commit
        if (!ok) {
          sm100::mma_commit(o_full);
          sm100::mbar_wait_cycles(o_full, 0, kWaitLimit / 8);
        }
      }
    } else if (warp == kMmaWarp + 1 && tail) {
      // zeros the V rows behind the last key, up to the 16 that a product step takes, once the MMA thread has seen the block
      const int valid = kv_len % kBK;
      if (warp_wait(v_dirty, 0, abort, a.err)) {
        uint8_t *v = ring + (2 * n - 1) % NS * S::kTile + valid * 128;
        for (int x = lane; x < ((valid + 15) / 16 * 16 - valid) * 8 * kSub; x += 32)
          *reinterpret_cast<uint4 *>(v + x % kSub * 16384 + x / kSub * 16) = make_uint4(0, 0, 0, 0);
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(v_clean);
      }
    }
    __syncwarp();
    if (NT == 1 && a.splits > 1) {  // the softmax warps' two barriers around the sums' exchange
      sm100::cluster_sync();
      sm100::cluster_sync();
    }
  } else {
    // ----------------------------- softmax ------------------------------
    sm100::regs_up<S::kSoftmaxRegs>();
    const int i = wg, quad = warp & 3;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t st = s_tmem + i * 128 + lanes, ot = o_tmem + i * DP + lanes;
    const bool live = i < nt && i * kBQ + quad * 32 < here;  // a warp without rows leaves P as it is
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    if (i < nt) {
      for (int j = 0; j < n; j++) {
        if (!warp_wait(s_full + 8 * i, j & 1, abort, a.err)) {
          ok = false;
          break;
        }
        sm100::tc_fence_after();
        if (live) {
          float s[128];
#pragma unroll
          for (int q = 0; q < 4; q++) sm100::tmem_ld32(st + q * 32, reinterpret_cast<uint32_t *>(s) + q * 32);
          sm100::tmem_ld_wait();
          const int valid = kv_len - (t0 + j) * kBK;
          if (valid < kBK) {
#pragma unroll
            for (int q = 0; q < 128; q++) s[q] = q < valid ? s[q] : -INFINITY;
          }
          float top[4];
#pragma unroll
          for (int q = 0; q < 4; q++) top[q] = fmaxf(s[q], s[q + 4]);
#pragma unroll
          for (int q = 8; q < 128; q += 4)
#pragma unroll
            for (int z = 0; z < 4; z++) top[z] = fmaxf(top[z], s[q + z]);
          const float mn = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), m);
          if (__any_sync(0xffffffffu, (mn - m) * a.c > kSlack)) {
            const float f = mn > m ? ex2((m - mn) * a.c) : 1.f;
            m = mn;
            l *= f;
            if (j > 0) {  // S of this block was committed after the last P V: O is complete
#pragma unroll
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
          const float base = kLift - (m == -INFINITY ? 0.f : m * a.c);
          const uint64_t c2 = sm100::pack_f32x2(a.c, a.c), base2 = sm100::pack_f32x2(base, base);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int q = 0; q < 128; q += 32) {
            uint32_t p[16];
#pragma unroll
            for (int z = 0; z < 32; z += 2) {
              const uint64_t x = sm100::fma_f32x2(sm100::pack_f32x2(s[q + z], s[q + z + 1]), c2, base2);
              float p0, p1;
              sm100::unpack_f32x2(x, p0, p1);
              p0 = ex2(p0), p1 = ex2(p1);
              sum[z >> 1 & 1] = sm100::add_f32x2(sum[z >> 1 & 1], sm100::pack_f32x2(p0, p1));
              p[z / 2] = pack2<DT>(p0, p1);
            }
            sm100::tmem_st16(st + q / 2, p);
          }
          float l0, l1;
          sm100::unpack_f32x2(sm100::add_f32x2(sum[0], sum[1]), l0, l1);
          l += l0 + l1;
          sm100::tmem_st_wait();
        }
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(p_full + 8 * i);
      }
      if (n > 0 && ok) ok = warp_wait(o_full + 8 * i, 0, abort, a.err);
      sm100::tc_fence_after();
    }
    const bool have = n > 0 && ok;  // O holds sums
    const int row = quad * 32 + lane;
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
  static int regs = 0;  // registers a thread the kernel is launched with: what its warpgroups share
  if (!regs) {
    cudaFuncAttributes fa;
    T2SC_CUDA(cudaFuncGetAttributes(&fa, kernel), "attention");
    regs = fa.numRegs;
  }
  if (regs * (NT + 1) < NT * S::kSoftmaxRegs + S::kOtherRegs) {
    err = "attention: the kernel was built with fewer registers than its warpgroups share";
    return T2SC_ERR_UNSUPPORTED;
  }
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
  t.out = a.out, t.ldo = a.ldo;
  t.seqs = s->d_sorted;
  t.blocks = s->d_blocks + (NT == 2 ? 0 : s->batch + 1);
  t.batch = (int)s->batch, t.heads = a.heads, t.head_dim = a.head_dim, t.splits = splits;
  t.c = a.scale * 1.4426950408889634f, t.err = ctx->d_err;
  const int64_t grid = (NT == 2 ? s->blocks256 : s->blocks128) * a.heads * splits;
  if (grid > INT32_MAX) return fail(ctx, T2SC_ERR_UNSUPPORTED, "attention: too many query blocks in one call");
  T2SC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem), "attention");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid), cfg.blockDim = dim3(S::kThreads), cfg.dynamicSmemBytes = S::kSmem, cfg.stream = ctx->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  T2SC_CUDA(cudaLaunchKernelEx(&cfg, kernel, t), "attention");
  T2SC_LAUNCHED(ctx, "attention");
  return T2SC_OK;
}

template <int DT, int DP>
int launch_dp(t2sc_seqs *s, const AttnArgs &a, std::string &err) {
  const int64_t sms = s->ctx->num_sms, pairs = s->blocks256 * a.heads, singles = s->blocks128 * a.heads;
  // Two query blocks a CTA once they fill the SMs; below that one block a
  // CTA (two CTAs an SM), its keys split while CTA places stay free and every
  // part keeps at least two key blocks.
  if (pairs >= sms) return launch<DT, DP, 2>(s, a, 1, err);
  int splits = 1;
  while (splits < 8 && singles * splits * 2 <= 2 * sms && s->max_kv >= (int64_t)4 * splits * kBK) splits *= 2;
  return launch<DT, DP, 1>(s, a, splits, err);
}

}  // namespace

bool attention_tc_takes(const t2sc_seqs *s, const AttnArgs &a, int dtype) {
  auto on16 = [](const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
  const bool keys = s->kv_off[s->batch] > s->kv_off[0];
  // scores are compared before they are scaled: the scale has to keep their order
  return dtype != T2SC_DT_F32 && a.head_dim % 8 == 0 && a.head_dim <= 128 && a.scale > 0.f && on16(a.q, a.ldq) &&
         on16(a.out, a.ldo) && (!keys || (on16(a.k, a.ldk) && on16(a.v, a.ldv)));
}

int attention_tc(t2sc_seqs *s, const AttnArgs &a, int dtype, std::string &err) {
  if (dtype == T2SC_DT_BF16)
    return a.head_dim <= 64 ? launch_dp<T2SC_DT_BF16, 64>(s, a, err) : launch_dp<T2SC_DT_BF16, 128>(s, a, err);
  return a.head_dim <= 64 ? launch_dp<T2SC_DT_F16, 64>(s, a, err) : launch_dp<T2SC_DT_F16, 128>(s, a, err);
}

}  // namespace t2sc
