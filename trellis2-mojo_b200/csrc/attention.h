// A ragged batch's sequences and the launch arguments of the attention kernels.
#pragma once
#include <stdint.h>

#include <string>
#include <vector>

#include "internal.h"

struct t2sc_seqs {
  t2sc_ctx *ctx = nullptr;
  int device = 0;  // the context's, which may be gone when the handle is destroyed
  int64_t batch = 0;
  std::vector<int64_t> q_off, kv_off;  // [batch + 1]
  int64_t q_rows = 0, kv_rows = 0;     // rows up to the last offset
  int64_t q_total = 0;                 // query rows inside sequences
  int64_t max_q = 0, max_kv = 0;       // queries, keys of the longest sequence
  int64_t blocks32 = 0, blocks128 = 0, blocks256 = 0;  // blocks of 32 / 128 / 256 query rows, sequence by sequence
  int64_t long128 = 0, long256 = 0;    // blocks of 128 / 256 rows of sequences with at least 7/8 of the longest one's keys
  int64_t long_q = 0;                  // most queries of one of these
  double work128 = 0, work256 = 0;     // sum over the blocks of their units of 64 keys
  int4 *d_sorted = nullptr;            // as d_seqs, most keys first
  int64_t *d_blocks = nullptr;         // [3][batch + 1] blocks of 256 / 128 rows before each of d_sorted, of 32 rows before each of d_seqs
  // the first sequences of d_sorted and d_blocks, for kernels to carry in their arguments
  int4 few_seqs[8];
  int64_t few_blocks256[9], few_blocks128[9];
  int4 *d_seqs = nullptr;              // [batch] first query row, query rows, first key row, key rows
};

namespace t2sc {

// 2^x, relative error 2^-22; results below 2^-126 are zero.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct AttnArgs {
  const char *q = nullptr, *k = nullptr, *v = nullptr;
  char *out = nullptr;
  int64_t ldq = 0, ldk = 0, ldv = 0, ldo = 0;  // elements between rows
  const int4 *seqs = nullptr;
  const int64_t *blocks32 = nullptr;  // [batch + 1] blocks of 32 query rows before each sequence
  int batch = 0, heads = 0, head_dim = 0;
  float scale = 0.f;
};

// 16-bit rows that start on 16 bytes, head_dim a multiple of 8 up to 128, scale in (0, 1e38).
bool attention_tc_takes(const t2sc_seqs *s, const AttnArgs &a, int dtype);
int attention_tc(t2sc_seqs *s, const AttnArgs &a, int dtype, std::string &err);
// As attention_tc, for at most 4 queries a sequence.
bool attention_rows_takes(const t2sc_seqs *s, const AttnArgs &a, int dtype);
int attention_rows(t2sc_seqs *s, const AttnArgs &a, int dtype, std::string &err);
int attention_simt(t2sc_seqs *s, const AttnArgs &a, int dtype, std::string &err);

}  // namespace t2sc
