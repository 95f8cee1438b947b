// g4_paged.cuh -- the paged-cache operators' shared definitions (internal to libgemma4_cuda.so).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/g4.h"

namespace g4 {

struct Pool {
  uint8_t *k, *v;
  float *ks, *vs;
  int n_pages, page_size, kv_heads, hd, fmt;
};

// A ragged attention call (g4_op_paged_attention's arguments, checked).
struct PagedAttn {
  Pool pool;
  const void *q;
  void *out;
  float *lse;
  long long q_stride, o_stride;   // elements between rows
  int type, heads, group, rows, batch;
  const int32_t *q_begin, *q_pos, *kv_len, *table;
  int table_stride, max_q, max_kv, window;
  float scale;
  // Set by the launcher: the least tiles of 16 positions a block takes, the tiles that beginning a list
  // item counts for, the row groups per (sequence, KV head); the blocks' partials and the counts of
  // finished ones.
  int split_tiles, begin_tiles, row_groups;
  float *part;
  uint32_t *count;
  int *err;
};

// A verification call (g4_op_verify_drafts' arguments, checked).
struct DraftArgs {
  const void *logits;
  long long ld;
  int type, vocab, rows, batch;
  const int32_t *row_begin, *drafts;
  const float *probs;
  long long ld_probs;
  const float *uniforms, *gumbel;
  long long ld_gumbel;
  const float *temperature;
  int max_drafts;
  int32_t *tokens, *counts;
  float *logprobs;
  // Set by the launcher.
  int splits, chunk;
  struct DraftPart *part;
  uint32_t *count;
  int *err;
};
// One block's share of a row: the greatest x, how many are equal to it, the sum of exp(x - m) over the
// others, the winner of the race.
struct __align__(16) DraftPart {
  float m, n, r, key;
  int idx, pad[3];
};

// Every workspace starts with this many zeroed counters; a kernel that counts its finished blocks
// leaves them zero, and what follows holds nothing between calls.
constexpr int kPagedCounters = 65536;
constexpr size_t kPagedHeader = (size_t)kPagedCounters * 4;

// Device address of the current device's sticky G4_PAGED_* bits (null when it cannot be had).
int *paged_error_flags();

__device__ __forceinline__ void paged_raise(int *flags, int bit) { atomicOr(flags, bit); }

// One sequence's part of a call: its rows of q, the position of the first, the cached length.
struct SeqSpan {
  int row, n, pos, kv;
};
__device__ __forceinline__ SeqSpan seq_span(const PagedAttn &a, int b, bool report = true) {
  const int b0 = a.q_begin[b], b1 = a.q_begin[b + 1], kv = a.kv_len[b], pos = a.q_pos[b];
  SeqSpan s;
  s.row = min(max(b0, 0), a.rows);
  const int end = min(max(b1, s.row), a.rows);
  s.n = min(end - s.row, a.max_q);
  s.kv = min(max(kv, 0), a.max_kv);
  // Positions lie in 0 .. 2^30, so sums with a row index stay in 32 bits.
  s.pos = min(max(pos, -(1 << 30)), 1 << 30);
  if (report && (b0 < 0 || b1 < b0 || b1 > a.rows || end - s.row > a.max_q || kv < 0 || kv > a.max_kv || s.pos != pos))
    paged_raise(a.err, G4_PAGED_BAD_LENGTH);
  return s;
}
// The positions [lo, hi) that the row at position p sees: within 0 .. kv and neither end falling
// as p grows, also where nothing is seen.
__device__ __forceinline__ void row_range(const PagedAttn &a, int p, int kv, int &lo, int &hi) {
  hi = max(0, min(p + 1, kv));
  lo = min(hi, a.window > 0 ? max(0, p - a.window + 1) : 0);
}

cudaError_t launch_paged_attention(const PagedAttn &a, cudaStream_t st);
// Chunks of bf16 rows (g4_paged_chunk.cu).
cudaError_t launch_paged_chunk(const PagedAttn &a, cudaStream_t st);
// Bytes of partials a call of this shape needs past the counters.
size_t paged_attention_partials(const PagedAttn &a);

constexpr int kMaxDrafts = 255;
cudaError_t launch_verify_drafts(const DraftArgs &a, cudaStream_t st);
// Bytes past the counters.
size_t verify_drafts_partials(int vocab, int rows, int batch, int max_drafts);

}  // namespace g4
