// Accumulated attention weights: how much softmax weight each cached token received from the
// query rows of a call, added up over the rows and over the query heads of a kv head.
//
// The weights of a row are known only when all its scores are, and the output needs V at once, so
// a call runs attention first (the packed-row kernel of rows.hip, or the kernel below for other
// shapes) and keeps every score s (f32, log2 units) and each row's (max m, sum l); then one pass
// turns the scores into weights 2^(s - m) / l and adds them to the accumulator:
//   out[p] = decay in[p] + sum_rows 2^(s - m) / l.
// Keeping a score costs 8 bytes a (row, key), written and read; computing it again would read K
// again, 2 head_dim bytes a key: dearer from 16 rows of a kv head down at head_dim 128 in 16 bits.
#include "rows_split.h"
#include "wave_ops.h"

namespace llh {

namespace {

constexpr int kKeysPerThread = 4;
constexpr int kKeysPerWg = 256 * kKeysPerThread;

// One thread per four neighbouring positions of a (sequence, kv head).
__global__ __launch_bounds__(256) void accumulate_weights_kernel(const WeightsArgs w) {
  const RowsArgs &a = w.rows;
  const int b = blockIdx.z;
  const int kvh = blockIdx.y;
  const SeqSplit sq = seq_split<64>(a, b);
  if (sq.flags || (a.chunk_starts && sq.ctx < sq.chunk)) return;  // flagged, or no such call: left alone
  const int p0 = (int)(blockIdx.x * kKeysPerWg + threadIdx.x * kKeysPerThread);
  if (p0 >= sq.ctx) return;
  const int G = a.q_heads / a.pool.kv_heads;
  const int rows = max(0, min(sq.chunk, a.max_rows));
  const int first = sq.ctx - sq.chunk;
  float acc[kKeysPerThread] = {};
  if (p0 + kKeysPerThread > sq.lo) {
    const size_t row0 = (size_t)b * a.max_rows * a.q_heads + kvh * G;
    const float *sc = a.scores + row0 * a.score_stride + (p0 - weights_base(sq.lo));
    for (int t = 0; t < rows; t++) {
      const int pos = first + t;
      if (p0 > pos) continue;
      const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
      if (p0 + kKeysPerThread <= lo) continue;
      for (int g = 0; g < G; g++) {
        const size_t r = (size_t)t * a.q_heads + g;
        const float2 ml = a.row_ml[row0 + r];
        const float m = ml.x == -INFINITY ? 0.0f : ml.x;  // no key left: every score is -inf
        const float inv = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;
        const float4 s = *reinterpret_cast<const float4 *>(sc + r * a.score_stride);
#pragma unroll
        for (int i = 0; i < kKeysPerThread; i++) {
          const int p = p0 + i;
          if (p >= lo && p <= pos) acc[i] += fast_exp2((&s.x)[i] - m) * inv;
        }
      }
    }
  }
  const size_t at = ((size_t)b * a.pool.kv_heads + kvh) * w.stride + p0;
#pragma unroll
  for (int i = 0; i < kKeysPerThread; i++)
    if (p0 + i < sq.ctx) w.w_out[at + i] = (w.w_in ? w.decay * w.w_in[at + i] : 0.0f) + acc[i];
}

// Attention of one (query row, head) per workgroup for the shapes outside the packed-row kernel:
// any head_dim up to 512, block size, pool format and alignment.  Element-wise f32 dot products.
__global__ __launch_bounds__(256) void weights_generic_kernel(const RowsArgs a) {
  const int b = blockIdx.y;
  const int t = blockIdx.x / a.q_heads;
  const int h = blockIdx.x % a.q_heads;
  const int tid = threadIdx.x;
  const SeqSplit sq = seq_split<64>(a, b);
  if (sq.skip) {
    if (sq.flags && tid == 0 && blockIdx.x == 0) atomicOr(a.err, sq.flags);
    return;
  }
  if (t >= min(sq.chunk, a.max_rows)) return;
  const int Dh = a.pool.head_dim;
  const int bt = a.pool.block_tokens;
  const int kvh = h / (a.q_heads / a.pool.kv_heads);
  const int pos = sq.ctx - sq.chunk + t;
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int32_t *table = a.tables + (size_t)b * a.max_blocks;
  const size_t row = ((size_t)(sq.c0 + t) * a.q_heads + h) * Dh;
  const size_t prow = ((size_t)b * a.max_rows + t) * a.q_heads + h;
  float *sc = a.scores + prow * a.score_stride - weights_base(sq.lo);

  __shared__ float qs[kWeightsMaxDim];
  __shared__ float w[256];
  __shared__ float red[256];
  __shared__ int64_t kblk[256];
  __shared__ int s_bad;
  for (int d = tid; d < Dh; d += 256) qs[d] = __uint_as_float((uint32_t)a.q[row + d] << 16);
  if (tid == 0) s_bad = 0;
  __syncthreads();

  auto block_of = [&](int p) -> int64_t {
    const int64_t blk = table[(p / bt) % a.max_blocks];
    return blk >= 0 && blk < a.pool.n_blocks ? blk : -1;
  };
  float m = -INFINITY;
  for (int p = lo + tid; p <= pos; p += 256) {
    const int64_t blk = block_of(p);
    float s = -INFINITY;
    if (blk < 0) {
      atomicOr(&s_bad, kErrBadBlock);
    } else {
      float dot = 0.0f;
      for (int d = 0; d < Dh; d++) dot += pool_elem(a.pool, 0, blk, kvh, p % bt, d) * qs[d];
      if (!(fabsf(dot * a.scale) < INFINITY)) atomicOr(&s_bad, kErrNonFinite);
      s = dot * a.scale_log2e;
    }
    sc[p] = s;
    m = fmaxf(m, s);
  }
  red[tid] = m;
  __syncthreads();
  for (int st = 128; st > 0; st >>= 1) {
    if (tid < st) red[tid] = fmaxf(red[tid], red[tid + st]);
    __syncthreads();
  }
  m = red[0];
  const float mref = m == -INFINITY ? 0.0f : m;
  __syncthreads();
  float l = 0.0f;
  float acc[kWeightsMaxDim / 256] = {};
  for (int k0 = lo; k0 <= pos; k0 += 256) {
    const int n = min(256, pos - k0 + 1);
    float e = 0.0f;
    if (tid < n) {
      e = fast_exp2(sc[k0 + tid] - mref);
      kblk[tid] = block_of(k0 + tid);
    }
    w[tid] = e;
    l += e;
    __syncthreads();
    for (int x = 0; x < kWeightsMaxDim / 256; x++) {
      const int d = tid + 256 * x;
      if (d < Dh)
        for (int k = 0; k < n; k++)
          if (kblk[k] >= 0) acc[x] += w[k] * pool_elem(a.pool, 1, kblk[k], kvh, (k0 + k) % bt, d);
    }
    __syncthreads();
  }
  red[tid] = l;
  __syncthreads();
  for (int st = 128; st > 0; st >>= 1) {
    if (tid < st) red[tid] += red[tid + st];
    __syncthreads();
  }
  l = red[0];
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int x = 0; x < kWeightsMaxDim / 256; x++) {
    const int d = tid + 256 * x;
    if (d < Dh) a.out[row + d] = f32_to_bf16_rne(gated(acc[x] * inv, a.gate, row + d));
  }
  if (tid == 0) {
    a.row_ml[prow] = make_float2(m, l);
    if (s_bad) atomicOr(a.err, s_bad);
  }
}

}  // namespace

hipError_t launch_weights_generic(const RowsArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(weights_generic_kernel, dim3(a.max_rows * a.q_heads, a.num_seqs), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_weights_accumulate(const WeightsArgs &w, int max_len, hipStream_t s) {
  const int tiles = (max_len + kKeysPerWg - 1) / kKeysPerWg;
  if (tiles <= 0) return hipSuccess;
  hipLaunchKernelGGL(accumulate_weights_kernel, dim3(tiles, w.rows.pool.kv_heads, w.rows.num_seqs), dim3(256), 0, s, w);
  return hipGetLastError();
}

}  // namespace llh
