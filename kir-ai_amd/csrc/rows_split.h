// The keys of a sequence and their split in the packed-row kernels (rows.hip, weights.hip).
#pragma once

#include "wave_ops.h"

namespace llh {

// The keys of a sequence and their split, the same in every kernel of a call.
struct SeqSplit {
  int c0, chunk, ctx;  // first query row, query rows, context length
  int lo;              // first position any row attends
  int unit0, units;    // units of UK keys
  int per_split, n_splits;
  bool skip;           // nothing to compute (flags: why)
  int flags;
};

template <int UK>
__device__ __forceinline__ SeqSplit seq_split(const RowsArgs &a, int b) {
  SeqSplit s;
  s.flags = 0;
  s.c0 = a.chunk_starts ? a.chunk_starts[b] : b;
  s.chunk = a.chunk_starts ? a.chunk_starts[b + 1] - s.c0 : 1;
  s.ctx = a.context_lens[b];
  const int first = s.ctx - s.chunk;  // position of the first row
  s.lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  const int span = max(0, s.ctx - s.lo);
  if ((a.max_span > 0 && span > a.max_span) || (a.max_len > 0 && s.ctx > a.max_len)) s.flags = kErrTooManySplits;
  else if ((int64_t)span > (int64_t)a.max_blocks * a.pool.block_tokens) s.flags = kErrSpan;
  s.skip = s.flags != 0 || s.chunk <= 0 || (a.chunk_starts && s.ctx < s.chunk);
  s.unit0 = s.lo / UK;
  s.units = span > 0 ? (s.ctx - 1) / UK - s.unit0 + 1 : 0;
  s.per_split = s.units <= a.single_units ? a.single_units
                                          : max(a.split_units, (s.units + a.max_splits - 1) / a.max_splits);
  s.n_splits = (s.units + s.per_split - 1) / s.per_split;
  return s;
}

// 1 / (weight sum).  No weight at all (every key masked, or every score -inf) gives the zero
// row of the tile prefill and the reference-order decode, and the NaN (0 / 0) of the vector
// decode kernels in the calls that are theirs too.
__device__ __forceinline__ float row_inv(const RowsArgs &a, float ll) {
  return ll == 0.0f && (a.chunk_starts || a.zero_bad || a.scores) ? 0.0f : 1.0f / ll;
}

// The weight of a score, given its row's maximum and 1 / sum, and an accumulator's new value: the same
// bits wherever they are computed.
__device__ __forceinline__ float score_weight(float s, float m, float inv) {
  return rounded_product(fast_exp2(s - m), inv);
}
__device__ __forceinline__ float accumulated(const RowsArgs &a, float before, float sum) {
  return a.w_in ? __builtin_fmaf(a.decay, before, sum) : sum;
}

}  // namespace llh
