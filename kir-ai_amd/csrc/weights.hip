// Accumulated attention weights: how much softmax weight each cached token received from the
// query rows of a call, added up over the rows and over the query heads of a kv head.
//
// The weights of a row are known only when all its scores are, and the output needs V at once, so
// a call runs attention first (the packed-row kernel of rows.hip, or the kernel below for other
// shapes) and keeps every score s (f32, log2 units) and each row's (max m, sum l) per split; a second
// launch merges the splits' outputs and, in other workgroups, turns the scores into weights and
// adds them to the accumulator:
//   out[p] = decay in[p] + sum_rows 2^(s - m) / l.
// The sums' order is fixed.  Keeping a score costs 8 bytes a (row, key), written and read; computing it again would read K
// again, 2 head_dim bytes a key: dearer up to 16 rows of a kv head at head_dim 128 in 16 bits.
//
// Bound: memory, at the rate of a copy, in large steps; the launch and its loads in small ones.
// Measured on MI355X (the second launch, us): 32 x U[256, 4096], Hq16 / Hkv8 6.1; 64 x 8192, Hq32 / Hkv8 20.8 (101
// MB, 4.8 TB/s); one sequence of 512 3.0.
#include "rows_split.h"
#include "wave_ops.h"

namespace llh {

namespace {


// The output of one (query row, head) from the partial rows of its splits, by one wavefront: D / 64
// dims a lane, eight partials in flight, the pairs one a lane.
template <int D>
__device__ __forceinline__ void merge_row(const RowsArgs &a, size_t prow, size_t orow, int n, int lane) {
  constexpr int PER = D / 64, FLIGHT = 8;
  typedef __attribute__((ext_vector_type(PER))) float part_t;
  const float2 ml = a.ws_ml[prow * a.max_splits + min(lane, n - 1)];
  const part_t *src = reinterpret_cast<const part_t *>(a.ws_o + prow * a.max_splits * D) + lane;
  part_t o = {};
  float f[1], sum = 0.0f;
  for (int i0 = 0; i0 < n; i0 += FLIGHT) {
    part_t p[FLIGHT];
#pragma unroll
    for (int i = 0; i < FLIGHT; i++) p[i] = src[(size_t)min(i0 + i, n - 1) * 64];
    if (i0 == 0) {
      const float mx[1] = {lane < n ? ml.x : -INFINITY}, l[1] = {ml.y};
      sum = merge_weights<1>(mx, l, lane, f);
    }
#pragma unroll
    for (int i = 0; i < FLIGHT; i++)
      if (i0 + i < n) o += p[i] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f[0]), i0 + i));
  }
  const float inv = row_inv(a, sum);
  const size_t at = orow * D + PER * lane;
#pragma unroll
  for (int d = 0; d < PER; d++) a.out[at + d] = f32_to_bf16_rne(gated(o[d] * inv, a.gate, at + d));
}

// The first `tiles` workgroups of a (kv head, sequence) take 64 KPL positions for each wavefront but
// for those that share them, the others merge the splits of its rows.  Of a tile, wavefront w takes
// the rows w % RW, w % RW + RW, ... of the positions w / RW, KPL neighbouring ones a lane, BATCH rows in
// flight, and the RW sums of a position meet in LDS.
// A row's (max, sum) come from its splits' pairs.  Few rows: each wavefront finds its own rows',
// a pair a lane.  Many (RW = 16): eight lanes a row, into LDS for the whole workgroup (a wavefront's
// reduction over 64 lanes for each of its rows took 10 us of 23, up to 256 rows over up to 1732
// positions, 4 sequences x 2 kv heads).
template <int D, int THREADS, int RW, int KPL, int BATCH>
__global__ __launch_bounds__(THREADS) void weights_finish_kernel(const RowsArgs a, int tiles) {
  typedef __attribute__((ext_vector_type(KPL))) float keys_t;
  constexpr int WAVE_KEYS = 64 * KPL;
  constexpr bool MANY = RW == 16;
  constexpr int BLOCK = MANY ? 1024 : 1;  // rows whose (max, 1 / sum, position) LDS holds
  const int b = blockIdx.z;
  const int kvh = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.q_heads / a.pool.kv_heads;
  const SeqSplit sq = seq_split<D == 256 ? 32 : 64>(a, b);
  if ((int)blockIdx.x >= tiles) {
    const int i = ((int)blockIdx.x - tiles) * (THREADS / 64) + wave;
    const int tok = i / G;
    if (sq.skip || sq.n_splits <= 1 || tok >= min(sq.chunk, a.max_rows)) return;
    const size_t head = kvh * G + i % G;
    merge_row<D>(a, ((size_t)b * a.max_rows + tok) * a.q_heads + head, (size_t)(sq.c0 + tok) * a.q_heads + head,
                 sq.n_splits, lane);
    return;
  }
  if (sq.flags || (a.chunk_starts && sq.ctx < sq.chunk)) return;  // flagged, or no such call: left alone
  const int tile0 = (int)blockIdx.x * (THREADS / 64 / RW * WAVE_KEYS);
  if (tile0 >= sq.ctx) return;
  const int wave0 = tile0 + wave / RW * WAVE_KEYS;  // this wavefront's first position
  const int p0 = wave0 + KPL * lane;
  const size_t at = ((size_t)b * a.pool.kv_heads + kvh) * a.w_stride + p0;
  float before[KPL] = {};
  if (wave % RW == 0 && a.w_in) {
#pragma unroll
    for (int i = 0; i < KPL; i++)
      if (p0 + i < sq.ctx) before[i] = a.w_in[at + i];
  }
  const int rows = max(0, min(sq.chunk, a.max_rows)) * G;
  const int first = sq.ctx - sq.chunk;
  const int base = weights_base(sq.lo);
  const bool here = p0 >= base && p0 < sq.ctx;  // scores of these positions are stored
  const size_t row0 = (size_t)b * a.max_rows * a.q_heads + kvh * G;
  float acc[KPL] = {};
  // adds row r's weights of this lane's positions, given its scores
  auto add = [&](const keys_t &s, float m, float inv, int pos) __attribute__((always_inline)) {
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
#pragma unroll
    for (int i = 0; i < KPL; i++) {
      const int p = p0 + i;
      acc[i] += (here & (p >= lo) & (p <= pos)) ? score_weight(s[i], m, inv) : 0.0f;
    }
  };
  // the index of row r's scores and pairs
  auto row_of = [&](int r) __attribute__((always_inline)) { return row0 + (size_t)(r / G) * a.q_heads + r % G; };
  auto scores_of = [&](size_t row) __attribute__((always_inline)) {
    return here ? *reinterpret_cast<const keys_t *>(a.scores + row * a.score_stride + (p0 - base)) : keys_t(0.0f);
  };
  if constexpr (MANY) {
    struct Row {
      float m, inv;
      int pos, row;  // (row: of the call's rows and heads, which the host keeps below 2^31)
    };
    __shared__ Row s_row[BLOCK];
    if (tile0 + THREADS / 64 / RW * WAVE_KEYS > base) {
      for (int block = 0; block < rows; block += BLOCK) {
        const int n = min(BLOCK, rows - block);
        for (int x = tid / 8; x < n; x += THREADS / 8) {
          const size_t row = row_of(block + x);
          const float2 *pairs = a.ws_ml + row * a.max_splits;
          float2 ml[kRowsMaxSplits / 8];
          float m = -INFINITY, sum = 0.0f;
#pragma unroll
          for (int i = 0; i < kRowsMaxSplits / 8; i++)
            if (8 * i < sq.n_splits) {
              ml[i] = pairs[min(8 * i + tid % 8, sq.n_splits - 1)];
              m = fmaxf(m, ml[i].x);
            }
          m = fmaxf(m, dpp<0xB1>(m));
          m = fmaxf(m, dpp<0x4E>(m));
          m = fmaxf(m, dpp<0x141>(m));
          m = m == -INFINITY ? 0.0f : m;  // no key left: every score is -inf
#pragma unroll
          for (int i = 0; i < kRowsMaxSplits / 8; i++)
            if (8 * i < sq.n_splits) sum += 8 * i + tid % 8 < sq.n_splits ? ml[i].y * fast_exp2(ml[i].x - m) : 0.0f;
          sum = row_sum8(sum);
          if (tid % 8 == 0)
            s_row[x] = Row{m, sum == 0.0f ? 0.0f : 1.0f / sum, first + (block + x) / G, (int)(row - row0)};
        }
        __syncthreads();
        for (int r0 = wave % RW; r0 < n; r0 += RW * BATCH) {
          keys_t s[BATCH];
#pragma unroll
          for (int k = 0; k < BATCH; k++) s[k] = scores_of(row0 + s_row[min(r0 + k * RW, n - 1)].row);
#pragma unroll
          for (int k = 0; k < BATCH; k++)
            if (r0 + k * RW < n) {
              const Row x = s_row[r0 + k * RW];
              add(s[k], x.m, x.inv, x.pos);
            }
        }
        __syncthreads();
      }
    }
  } else if (wave0 + WAVE_KEYS > base) {
    for (int r0 = wave % RW; r0 < rows; r0 += RW * BATCH) {
      float2 ml[BATCH];
      keys_t s[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; k++) {
        const size_t row = row_of(min(r0 + k * RW, rows - 1));
        ml[k] = a.ws_ml[row * a.max_splits + min(lane, sq.n_splits - 1)];
        s[k] = scores_of(row);
      }
#pragma unroll
      for (int k = 0; k < BATCH; k++) {
        const int r = r0 + k * RW;
        if (r >= rows) break;
        const float mx[1] = {lane < sq.n_splits ? ml[k].x : -INFINITY}, l[1] = {ml[k].y};
        float f[1], top;
        const float sum = merge_weights<1>(mx, l, lane, f, &top);
        add(s[k], top == -INFINITY ? 0.0f : top, sum == 0.0f ? 0.0f : 1.0f / sum, first + r / G);
      }
    }
  }
  if constexpr (RW > 1) {
    __shared__ float part[KPL][THREADS];
#pragma unroll
    for (int i = 0; i < KPL; i++) part[i][tid] = acc[i];
    __syncthreads();
    if (wave % RW) return;
#pragma unroll
    for (int x = 1; x < RW; x++)
#pragma unroll
      for (int i = 0; i < KPL; i++) acc[i] += part[i][tid + 64 * x];
  }
#pragma unroll
  for (int i = 0; i < KPL; i++)
    if (p0 + i < sq.ctx) a.w_out[at + i] = accumulated(a, before[i], acc[i]);
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

template <int D, int THREADS, int RW, int KPL, int BATCH>
static hipError_t launch_finish(const RowsArgs &a, int max_len, hipStream_t s) {
  const int rows = a.max_rows * (a.q_heads / a.pool.kv_heads);
  const int tile = THREADS / 64 / RW * 64 * KPL;
  const int merge_wgs = a.max_splits > 1 ? (rows + THREADS / 64 - 1) / (THREADS / 64) : 0;
  const int tiles = (int)(((unsigned)max_len + tile - 1) / tile);
  if (merge_wgs + tiles == 0) return hipSuccess;
  hipLaunchKernelGGL((weights_finish_kernel<D, THREADS, RW, KPL, BATCH>),
                     dim3(tiles + merge_wgs, a.pool.kv_heads, a.num_seqs), dim3(THREADS), 0, s, a, tiles);
  return hipGetLastError();
}

// Many rows are shared between wavefronts, and their positions, as one compute unit takes some 50 GB/s,
// spread over more workgroups.  Measured on MI355X (us, this launch), up to 256 rows of a kv head
// over up to 1732 positions, 4 x 2 of them: 16 wavefronts sharing 256 positions 11.8, 128 10.0, 64 12.5; 8
// sharing 256 15.8, 128 13.5.
template <int D>
static hipError_t launch_finish_d(const RowsArgs &a, int max_len, hipStream_t s) {
  const int rows = a.max_rows * (a.q_heads / a.pool.kv_heads);
  // few rows, a wavefront's positions each its own / shared by four (both launches, us): Hq32 / Hkv8, 1 x 1000 12.5 /
  // 11.5, 8 x 1000 14.2 / 13.8, 8 x 4000 32.3 / 33.1, 32 x 4000 106.5 / 113.3; eight rows (Hq32 / Hkv4) 1 x 1000
  // 14.7 / 12.4, 8 x 4000 24.5 / 23.3, 32 x 4000 65.5 / 67.3
  const long long wgs = (long long)a.num_seqs * a.pool.kv_heads * (((long long)max_len + 1023) / 1024);
  if (rows <= 4 && wgs >= 128) return launch_finish<D, 256, 1, 4, 4>(a, max_len, s);
  if (rows <= 16) return launch_finish<D, 256, 4, 4, 4>(a, max_len, s);
  return launch_finish<D, 1024, 16, 2, 16>(a, max_len, s);
}

hipError_t launch_weights_finish(const RowsArgs &a, int max_len, hipStream_t s) {
  // (other head_dims come in one split: nothing is merged)
  return a.pool.head_dim == 256 ? launch_finish_d<256>(a, max_len, s) : launch_finish_d<128>(a, max_len, s);
}

}  // namespace llh
