// The keys of a sequence, their split and the splits' merge in the packed-row kernels (rows.hip,
// weights.hip).
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

// Merge of the n <= N splits of one (query row, head): every partial row in flight at
// once, the (max, sum) pairs one per lane, split weights through v_readlane.
template <int D, int N>
__device__ __forceinline__ void rows_merge_n(const RowsArgs &a, size_t prow, size_t orow, int last, int d) {
  const size_t p0 = prow * a.max_splits;
  float o_sp[N];
#pragma unroll
  for (int i = 0; i < N; i++) o_sp[i] = a.ws_o[(p0 + min(i, last)) * D + d];
  const int li = d & 63;
  const float2 ml = a.ws_ml[p0 + min(li, last)];
  const float mx[1] = {li <= last ? ml.x : -INFINITY}, ly[1] = {ml.y};
  float f[1];
  const float ll = merge_weights<1>(mx, ly, li, f);
  float oo = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++)  // nothing of the places past the last (0 x infinity is NaN)
    oo += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f[0]), i)) * (i <= last ? o_sp[i] : 0.0f);
  const float inv = row_inv(a, ll);
  a.out[orow * D + d] = f32_to_bf16_rne(gated(oo * inv, a.gate, orow * D + d));
}

template <int D>
__device__ __forceinline__ void rows_merge(const RowsArgs &a, size_t prow, size_t orow, int last, int d) {
  if (last < 8) return rows_merge_n<D, 8>(a, prow, orow, last, d);
  if (last < 16) return rows_merge_n<D, 16>(a, prow, orow, last, d);
  if (last < 32) return rows_merge_n<D, 32>(a, prow, orow, last, d);
  return rows_merge_n<D, kRowsMaxSplits>(a, prow, orow, last, d);
}

}  // namespace llh
