// Accumulated attention weights: how much softmax weight each cached token received from the
// query rows of a call, added up over the rows and over the query heads of a kv head.
//
// The weights of a row are known only when all its scores are, and the output needs V at once, so
// a call runs attention first (the packed-row kernel of rows.hip, or the kernel below for other
// shapes) and keeps every score s (f32, log2 units) and each row's (max m, sum l) per split; a second
// launch merges the splits' outputs and, in other workgroups, turns the scores into weights and
// adds them to the accumulator:
//   out[p] = decay in[p] + sum_rows 2^(s - m) / l.
// Keeping a score costs 8 bytes a (row, key), written and read; computing it again would read K
// again, 2 head_dim bytes a key: dearer up to 16 rows of a kv head at head_dim 128 in 16 bits.
#include "rows_split.h"
#include "wave_ops.h"

namespace llh {

namespace {

constexpr int kWaveKeys = 256;  // positions of a wavefront, four neighbouring ones a lane

// The first `merge_wgs` workgroups of a (kv head, sequence) merge the splits of its rows, the others
// take kWaveKeys / RW * (wavefronts) positions each: wavefront w takes rows w % RW, w % RW + RW, ...
// of the positions w / RW, and the RW sums of a position meet in LDS.  Each wavefront finds
// the (max, sum) of its own rows from the splits' pairs, one a lane; pairs and scores of four rows are
// in flight together.
template <int D, int THREADS, int RW>
__global__ __launch_bounds__(THREADS) void weights_finish_kernel(const WeightsArgs w, int merge_wgs) {
  constexpr int BATCH = 4;
  const RowsArgs &a = w.rows;
  const int b = blockIdx.z;
  const int kvh = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.q_heads / a.pool.kv_heads;
  const SeqSplit sq = seq_split<D == 256 ? 32 : 64>(a, b);
  if ((int)blockIdx.x < merge_wgs) {
    constexpr int ROWS = THREADS / D;
    const int i = blockIdx.x * ROWS + tid / D;
    const int tok = i / G;
    if (sq.skip || sq.n_splits <= 1 || tok >= min(sq.chunk, a.max_rows)) return;
    const size_t head = kvh * G + i % G;
    rows_merge<D>(a, ((size_t)b * a.max_rows + tok) * a.q_heads + head, (size_t)(sq.c0 + tok) * a.q_heads + head,
                  sq.n_splits - 1, tid % D);
    return;
  }
  if (sq.flags || (a.chunk_starts && sq.ctx < sq.chunk)) return;  // flagged, or no such call: left alone
  const int tile0 = ((int)blockIdx.x - merge_wgs) * (THREADS / 64 / RW * kWaveKeys);
  if (tile0 >= sq.ctx) return;
  const int p0 = tile0 + wave / RW * kWaveKeys + 4 * lane;
  const size_t at = ((size_t)b * a.pool.kv_heads + kvh) * w.stride + p0;
  float before[4] = {};
  if (wave % RW == 0 && w.w_in) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (p0 + i < sq.ctx) before[i] = w.w_in[at + i];
  }
  const int rows = max(0, min(sq.chunk, a.max_rows)) * G;
  const int first = sq.ctx - sq.chunk;
  const int base = weights_base(sq.lo);
  const bool here = p0 >= base && p0 < sq.ctx;  // scores of these positions are stored
  const size_t row0 = (size_t)b * a.max_rows * a.q_heads + kvh * G;
  float acc[4] = {};
  if (tile0 + wave / RW * kWaveKeys + kWaveKeys > base) {
    for (int r0 = wave % RW; r0 < rows; r0 += RW * BATCH) {
      float2 ml[BATCH];
      float4 s[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; k++) {
        const int r = min(r0 + k * RW, rows - 1);
        const size_t row = row0 + (size_t)(r / G) * a.q_heads + r % G;
        ml[k] = a.ws_ml[row * a.max_splits + min(lane, sq.n_splits - 1)];
        s[k] = here ? *reinterpret_cast<const float4 *>(a.scores + row * a.score_stride + (p0 - base))
                    : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int k = 0; k < BATCH; k++) {
        const int r = r0 + k * RW;
        if (r >= rows) break;
        const float mx[1] = {lane < sq.n_splits ? ml[k].x : -INFINITY}, l[1] = {ml[k].y};
        float f[1], top;
        const float sum = merge_weights<1>(mx, l, lane, f, &top);
        const float m = top == -INFINITY ? 0.0f : top;  // no key left: every score is -inf
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int pos = first + r / G;
        const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int p = p0 + i;
          acc[i] += (here & (p >= lo) & (p <= pos)) ? fast_exp2((&s[k].x)[i] - m) * inv : 0.0f;
        }
      }
    }
  }
  if constexpr (RW > 1) {
    __shared__ float4 part[THREADS];
    part[tid] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (wave % RW) return;
#pragma unroll
    for (int x = 1; x < RW; x++) {
      const float4 o = part[tid + 64 * x];
#pragma unroll
      for (int i = 0; i < 4; i++) acc[i] += (&o.x)[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (p0 + i < sq.ctx) w.w_out[at + i] = (w.w_in ? w.decay * before[i] : 0.0f) + acc[i];
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
  const size_t prow = ((size_t)b * a.max_rows + t) * a.q_heads + h;  // (one split)
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
    a.ws_ml[prow] = make_float2(m, l);
    if (s_bad) atomicOr(a.err, s_bad);
  }
}

}  // namespace

hipError_t launch_weights_generic(const RowsArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(weights_generic_kernel, dim3(a.max_rows * a.q_heads, a.num_seqs), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int D, int THREADS, int RW>
static hipError_t launch_finish(const WeightsArgs &w, int max_len, hipStream_t s) {
  const RowsArgs &a = w.rows;
  const int G = a.q_heads / a.pool.kv_heads;
  const int tile = THREADS / 64 / RW * kWaveKeys;
  const int merge_wgs = a.max_splits > 1 ? (a.max_rows * G + THREADS / D - 1) / (THREADS / D) : 0;
  const unsigned tiles = ((unsigned)max_len + tile - 1) / tile;
  if (merge_wgs + tiles == 0) return hipSuccess;
  hipLaunchKernelGGL((weights_finish_kernel<D, THREADS, RW>), dim3(merge_wgs + tiles, a.pool.kv_heads, a.num_seqs),
                     dim3(THREADS), 0, s, w, merge_wgs);
  return hipGetLastError();
}

template <int D>
static hipError_t launch_finish_d(const WeightsArgs &w, int max_len, hipStream_t s) {
  const int rows = w.rows.max_rows * (w.rows.q_heads / w.rows.pool.kv_heads);
  if (rows <= 4) return launch_finish<D, 256, 1>(w, max_len, s);
  if (rows <= 16) return launch_finish<D, 256, 4>(w, max_len, s);
  return launch_finish<D, 1024, 16>(w, max_len, s);
}

hipError_t launch_weights_finish(const WeightsArgs &w, int max_len, hipStream_t s) {
  // (other head_dims come in one split: nothing is merged)
  return w.rows.pool.head_dim == 256 ? launch_finish_d<256>(w, max_len, s) : launch_finish_d<128>(w, max_len, s);
}

}  // namespace llh
