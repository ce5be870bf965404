// Softmax attention inside each sequence of a ragged batch:
//   out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j, h]) v[j, h],
// j over the keys of i's sequence; a sequence without keys gives zeros.
//
// One pass over the keys: with m the running maximum of q . k and l the running
// sum of a row, a block of products s updates m' = max(m, s), o = o e^(scale (m
// - m')) + sum e^(scale (s - m')) v and l likewise; out = o / l. m, l and o are
// f32. The difference is taken before the scale: near the maximum it is exact,
// where the difference of two scaled products would keep their roundings, and
// no finite scale makes it an infinity minus an infinity.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string.h>

#include <algorithm>
#include <cmath>

#include "attention.h"
#include "entry.h"

namespace t2sc {
namespace {

constexpr int kMaxHeadDim = 256;
constexpr int64_t kMaxRow = INT32_MAX - 65535;  // block counts and ends of rows stay below 2^31

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

// CUDA-core kernel for every type, head_dim up to 256, stride and alignment:
// 32 queries of one head a CTA, four threads a query, keys in blocks of 32
// through shared memory. Products are f32. f32 runs here; the 16-bit types
// only where the tensor-core kernel's TMA loads do not apply.
constexpr int kBQ = 32, kBKV = 32, kThreads = 128;

template <int DT>
__global__ void __launch_bounds__(kThreads) attention_simt_kernel(const AttnArgs a) {
  extern __shared__ float smem[];
  const int D = a.head_dim, pitch = D + 1;
  float *qs = smem, *kv = qs + kBQ * pitch, *ps = kv + kBKV * pitch;  // ps: [kBQ][kBKV + 1]
  const int tid = threadIdx.x, row = tid >> 2, part = tid & 3;
  const int head = blockIdx.y;
  // the CTA's sequence (the last one that begins at or before this block) and its block of queries inside it
  int lo = 0, hi = a.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(a.blocks32 + mid) <= (int64_t)blockIdx.x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int4 seq = __ldg(a.seqs + lo);
  const int64_t q0 = seq.x + ((int64_t)blockIdx.x - __ldg(a.blocks32 + lo)) * kBQ;
  const int here = (int)min((int64_t)kBQ, seq.x + (int64_t)seq.y - q0);
  const int64_t at = (int64_t)head * D;
  for (int i = tid; i < kBQ * D; i += kThreads) {
    const int r = i / D, c = i % D;
    // a negative scale's sign goes to the query, so that the largest product has the largest weight
    qs[r * pitch + c] = r < here ? copysignf(1.f, a.scale) * ld1<DT>(a.q, (q0 + r) * a.ldq + at + c) : 0.f;
  }
  const float scale = fabsf(a.scale);
  float m = -INFINITY, l = 0.f;
  constexpr int P = kMaxHeadDim / 4;
  float o[P];
#pragma unroll
  for (int i = 0; i < P; i++) o[i] = 0.f;
  for (int64_t k0 = 0; k0 < seq.w; k0 += kBKV) {
    const int keys = (int)min((int64_t)kBKV, seq.w - k0);
    __syncthreads();
    for (int i = tid; i < kBKV * D; i += kThreads) {
      const int r = i / D, c = i % D;
      kv[r * pitch + c] = r < keys ? ld1<DT>(a.k, (seq.z + k0 + r) * a.ldk + at + c) : 0.f;
    }
    __syncthreads();
    float s[kBKV / 4], top = m;
#pragma unroll
    for (int j = 0; j < kBKV / 4; j++) s[j] = 0.f;
    for (int c = 0; c < D; c++) {
      const float qc = qs[row * pitch + c];
#pragma unroll
      for (int j = 0; j < kBKV / 4; j++) s[j] += qc * kv[(j * 4 + part) * pitch + c];
    }
#pragma unroll
    for (int j = 0; j < kBKV / 4; j++) {
      if (j * 4 + part >= keys) s[j] = -INFINITY;
      top = fmaxf(top, s[j]);
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float base = top == -INFINITY ? 0.f : top;  // every score -inf so far: their weights are 0
    const float keep = m == -INFINITY ? 0.f : expf((m - base) * scale);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kBKV / 4; j++) {
      const float p = j * 4 + part < keys ? expf((s[j] - base) * scale) : 0.f;
      ps[row * (kBKV + 1) + j * 4 + part] = p;
      sum += p;
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    l = l * keep + sum, m = top;
    __syncthreads();
    for (int i = tid; i < kBKV * D; i += kThreads) {
      const int r = i / D, c = i % D;
      kv[r * pitch + c] = r < keys ? ld1<DT>(a.v, (seq.z + k0 + r) * a.ldv + at + c) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P; i++) {
      const int c = i * 4 + part;
      if (c >= D) break;
      float t = o[i] * keep;
      for (int j = 0; j < keys; j++) t += ps[row * (kBKV + 1) + j] * kv[j * pitch + c];
      o[i] = t;
    }
  }
  if (row >= here) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no key, or every score -inf: zeros
#pragma unroll
  for (int i = 0; i < P; i++) {
    const int c = i * 4 + part;
    if (c >= D) break;
    st1<DT>(a.out, (q0 + row) * a.ldo + at + c, o[i] * inv);
  }
}

}  // namespace

int attention_simt(t2sc_seqs *s, const AttnArgs &a, int dtype, std::string &err) {
  t2sc_ctx *ctx = s->ctx;
  if (s->blocks32 > INT32_MAX) return fail(ctx, T2SC_ERR_UNSUPPORTED, "attention: too many query blocks in one call");
  auto smem_of = [](int head_dim) { return ((kBQ + kBKV) * (size_t)(head_dim + 1) + kBQ * (kBKV + 1)) * sizeof(float); };
  const size_t smem = smem_of(a.head_dim);
  const dim3 grid((unsigned)s->blocks32, (unsigned)a.heads);
  auto go = [&](auto kernel) -> int {
    // for the largest head: calls of other head dims may be in other threads
    static std::atomic<uint64_t> allowed[3] = {};
    T2SC_TRY(allow_smem(ctx, kernel, (int)smem_of(kMaxHeadDim), allowed[dtype], err));
    kernel<<<grid, kThreads, smem, ctx->stream>>>(a);
    T2SC_LAUNCHED(ctx, "attention");
    return T2SC_OK;
  };
  if (dtype == T2SC_DT_F32) return go(attention_simt_kernel<T2SC_DT_F32>);
  if (dtype == T2SC_DT_BF16) return go(attention_simt_kernel<T2SC_DT_BF16>);
  return go(attention_simt_kernel<T2SC_DT_F16>);
}

}  // namespace t2sc

using namespace t2sc;

extern "C" {

int t2sc_seqs_create(t2sc_ctx *ctx, const int64_t *q_offsets, const int64_t *kv_offsets, int64_t batch, t2sc_seqs **out) {
  if (!ctx || !out) return T2SC_ERR_INVALID;
  *out = nullptr;
  return guarded(ctx, [&]() -> int {
    if (batch < 0 || batch > (1 << 20)) return fail(ctx, T2SC_ERR_INVALID, "seqs: batch must be in [0, 2^20]");
    if (!q_offsets) return fail(ctx, T2SC_ERR_INVALID, "seqs: null offsets");
    if (!kv_offsets) kv_offsets = q_offsets;
    for (const int64_t *off : {q_offsets, kv_offsets}) {
      if (off[0] < 0 || off[batch] > kMaxRow) return fail(ctx, T2SC_ERR_INVALID, "seqs: offsets must be in [0, 2^31 - 2^16]");
      for (int64_t b = 0; b < batch; b++)
        if (off[b + 1] < off[b]) return fail(ctx, T2SC_ERR_INVALID, "seqs: offsets must not fall");
    }
    DeviceGuard g(ctx->device);
    CaptureTolerant relaxed;
    std::string &err = ctx->last_error;
    std::unique_ptr<t2sc_seqs, int (*)(t2sc_seqs *)> s(new t2sc_seqs(), t2sc_seqs_destroy);
    s->ctx = ctx;
    s->device = ctx->device;
    s->batch = batch;
    s->q_off.assign(q_offsets, q_offsets + batch + 1);
    s->kv_off.assign(kv_offsets, kv_offsets + batch + 1);
    s->q_rows = s->q_off[batch], s->kv_rows = s->kv_off[batch];
    s->q_total = s->q_off[batch] - s->q_off[0];
    std::vector<int4> h((size_t)batch + 1);
    for (int64_t b = 0; b < batch; b++)
      h[b] = make_int4((int)s->q_off[b], (int)(s->q_off[b + 1] - s->q_off[b]), (int)s->kv_off[b],
                       (int)(s->kv_off[b + 1] - s->kv_off[b]));
    std::vector<int4> sorted(h.begin(), h.begin() + batch);
    std::stable_sort(sorted.begin(), sorted.end(), [](const int4 &x, const int4 &y) { return x.w > y.w; });
    std::vector<int64_t> blocks(3 * (size_t)(batch + 1), 0);
    for (int64_t b = 0; b < batch; b++) {
      blocks[b + 1] = blocks[b] + ((int64_t)sorted[b].y + 255) / 256;
      blocks[batch + 1 + b + 1] = blocks[batch + 1 + b] + ((int64_t)sorted[b].y + 127) / 128;
      blocks[2 * (batch + 1) + b + 1] = blocks[2 * (batch + 1) + b] + ((int64_t)h[b].y + kBQ - 1) / kBQ;
      s->max_q = std::max<int64_t>(s->max_q, sorted[b].y);
      s->max_kv = std::max<int64_t>(s->max_kv, sorted[b].w);
    }
    for (const int4 &q : sorted) {
      const int64_t b256 = ((int64_t)q.y + 255) / 256, b128 = ((int64_t)q.y + 127) / 128;
      const double units = (double)(((int64_t)q.w + 63) / 64);
      s->work256 += b256 * units, s->work128 += b128 * units;
      if ((int64_t)q.w * 8 >= s->max_kv * 7) s->long256 += b256, s->long128 += b128, s->long_q = std::max<int64_t>(s->long_q, q.y);
    }
    for (int64_t b = 0; b <= 8; b++) {
      s->few_blocks256[b] = b <= batch ? blocks[b] : 0, s->few_blocks128[b] = b <= batch ? blocks[batch + 1 + b] : 0;
      if (b < 8) s->few_seqs[b] = b < batch ? sorted[b] : make_int4(0, 0, 0, 0);
    }
    s->blocks256 = blocks[batch], s->blocks128 = blocks[2 * batch + 1], s->blocks32 = blocks[3 * batch + 2];
    // one allocation: sequences in order, sorted, block counts
    const size_t nb = (size_t)batch + 1, bytes = 2 * nb * sizeof(int4) + blocks.size() * sizeof(int64_t);
    T2SC_CUDA(cudaMalloc((void **)&s->d_seqs, bytes), "seqs");
    s->d_sorted = s->d_seqs + nb;
    s->d_blocks = reinterpret_cast<int64_t *>(s->d_sorted + nb);
    sorted.resize(nb);
    std::vector<char> image(bytes);
    memcpy(image.data(), h.data(), nb * sizeof(int4));
    memcpy(image.data() + nb * sizeof(int4), sorted.data(), nb * sizeof(int4));
    memcpy(image.data() + 2 * nb * sizeof(int4), blocks.data(), blocks.size() * sizeof(int64_t));
    T2SC_CUDA(cudaMemcpyAsync(s->d_seqs, image.data(), bytes, cudaMemcpyHostToDevice, ctx->own_stream), "seqs");
    T2SC_CUDA(cudaStreamSynchronize(ctx->own_stream), "seqs");
    *out = s.release();
    return T2SC_OK;
  });
}

int t2sc_seqs_destroy(t2sc_seqs *s) {
  if (!s) return T2SC_OK;
  DeviceGuard g(s->device);
  CaptureTolerant relaxed;
  if (s->d_seqs) cudaFree(s->d_seqs);  // waits for the kernels that read it, on whatever stream
  delete s;
  return T2SC_OK;
}

int t2sc_attention_device(t2sc_seqs *seqs, const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v,
                          int64_t v_stride, void *out, int64_t out_stride, int heads, int head_dim, float scale, int dtype) {
  if (!seqs) return T2SC_ERR_INVALID;
  t2sc_ctx *ctx = seqs->ctx;
  return guarded(ctx, [&]() -> int {
    if (heads < 1 || heads > 4096) return fail(ctx, T2SC_ERR_INVALID, "attention: heads must be in [1, 4096]");
    if (head_dim < 1 || head_dim > kMaxHeadDim) return fail(ctx, T2SC_ERR_INVALID, "attention: head_dim must be in [1, 256]");
    if (!std::isfinite(scale)) return fail(ctx, T2SC_ERR_INVALID, "attention: scale must be finite");
    if (!dtype_known(dtype)) return fail(ctx, T2SC_ERR_INVALID, "attention: unknown dtype");
    if (seqs->q_total == 0) return T2SC_OK;
    const int64_t width = (int64_t)heads * head_dim;
    const int es = dtype_size(dtype);
    const bool keys = seqs->kv_off[seqs->batch] > seqs->kv_off[0];
    if (!q || !out || (keys && (!k || !v))) return fail(ctx, T2SC_ERR_INVALID, "attention: null buffer");
    // rows [0, last offset) of every buffer
    const Rows rq{q, q_stride, seqs->q_rows, width, es}, ro{out, out_stride, seqs->q_rows, width, es},
        rk{k, k_stride, keys ? seqs->kv_rows : 0, width, es}, rv{v, v_stride, keys ? seqs->kv_rows : 0, width, es};
    for (const Rows *r : {&rq, &rk, &rv, &ro}) {
      if (!stride_ok(*r)) return fail(ctx, T2SC_ERR_INVALID, "attention: a row stride must be in [heads * head_dim, 2^28]");
      if (!aligned_to_elem(*r)) return fail(ctx, T2SC_ERR_INVALID, "attention: a buffer is not aligned to its element type");
    }
    for (const Rows *r : {&rq, &rk, &rv})
      if (overlaps(ro, *r)) return fail(ctx, T2SC_ERR_INVALID, "attention: out overlaps q, k or v");
    AttnArgs a;
    a.q = static_cast<const char *>(q), a.k = static_cast<const char *>(k), a.v = static_cast<const char *>(v);
    a.out = static_cast<char *>(out);
    a.ldq = q_stride, a.ldk = k_stride, a.ldv = v_stride, a.ldo = out_stride;
    a.seqs = seqs->d_seqs, a.blocks32 = seqs->d_blocks + 2 * (seqs->batch + 1), a.batch = (int)seqs->batch, a.heads = heads, a.head_dim = head_dim, a.scale = scale;
    T2SC_TRY(earlier_failure(ctx));
    DeviceGuard g(ctx->device);
    if (attention_rows_takes(seqs, a, dtype)) return attention_rows(seqs, a, dtype, ctx->last_error);
    return attention_tc_takes(seqs, a, dtype) ? attention_tc(seqs, a, dtype, ctx->last_error)
                                              : attention_simt(seqs, a, dtype, ctx->last_error);
  });
}

}  // extern "C"
