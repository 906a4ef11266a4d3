// Eviction from the paged cache by accumulated attention weight: the choice of the tokens to keep
// (kv_select) and their move to other blocks (kv_compact).
#include "wave_ops.h"

namespace llh {

namespace {

// Order-preserving bits of a weight: NaN below every number, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;

// Exclusive sum of `v` over the threads of the workgroup; *total receives the sum of all.
__device__ __forceinline__ int block_exclusive(int v, int *s_waves, int *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // s_waves may still be read
  if (lane == 63) s_waves[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; w++) {
    if (w < wave) before += s_waves[w];
    all += s_waves[w];
  }
  *total = all;
  return before + x - v;
}

// One workgroup per (sequence, kv head).  The k-th largest key of the positions between the sinks
// and the recent ones is found eight bits at a time; the kept positions are then written in order.
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(const SelectArgs a) {
  const int b = blockIdx.y, h = blockIdx.x;
  const int tid = threadIdx.x;
  const int len = a.seq_lens[b];
  if (len < 0 || len > a.max_seq_len) {
    if (tid == 0 && h == 0) {
      atomicOr(a.err, kErrTooManySplits);
      a.kept_lens[b] = 0;
    }
    return;
  }
  if (tid == 0 && h == 0) a.kept_lens[b] = min(len, a.budget);
  int32_t *keep = a.keep + ((size_t)b * a.kv_heads + h) * a.keep_stride;
  if (len <= a.budget) {
    for (int i = tid; i < len; i += kSelectThreads) keep[i] = i;
    return;
  }
  const float *w = a.weights + ((size_t)b * a.kv_heads + h) * a.weights_stride;
  const int lo = a.sinks, hi = len - a.recent;  // the positions to choose from; lo <= hi as len > budget
  int want = a.budget - a.sinks - a.recent;
  __shared__ int hist[256];
  __shared__ int s_waves[kSelectWaves];
  __shared__ int s_bin, s_above;
  uint32_t prefix = 0, mask = 0;
  int equal_wanted = 0;
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int p = lo + tid; p < hi; p += kSelectThreads) {
        const uint32_t k = order_key(w[p]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      // the bin that holds the want-th largest: sums from the top down
      int total;
      const int mine = tid < 256 ? hist[255 - tid] : 0;
      const int above = block_exclusive(mine, s_waves, &total);
      if (tid < 256 && above < want && above + mine >= want) {
        s_bin = 255 - tid;
        s_above = above;
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      mask |= 255u << shift;
      want -= s_above;
      __syncthreads();
    }
    equal_wanted = want;
  } else {
    prefix = 0xffffffffu;  // nothing of the middle (no key reaches it: a NaN's is 0)
  }
  int n_out = 0, n_equal = 0;
  for (int p0 = 0; p0 < len; p0 += kSelectThreads) {
    const int p = p0 + tid;
    bool on = p < len && (p < lo || p >= hi);
    bool eq = false;
    if (p >= lo && p < hi) {
      const uint32_t k = order_key(w[p]);
      on = k > prefix;
      eq = k == prefix;
    }
    int total;
    const int rank = n_equal + block_exclusive(eq ? 1 : 0, s_waves, &total);
    n_equal += total;
    on = on || (eq && rank < equal_wanted);
    const int at = n_out + block_exclusive(on ? 1 : 0, s_waves, &total);
    n_out += total;
    if (on) keep[at] = p;
  }
}

// One workgroup per (destination block, kv head, sequence), element by element: any block size,
// head_dim and format but int8 rows.
__global__ __launch_bounds__(256) void kv_compact_generic_kernel(const CompactArgs a) {
  const int j = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x;
  const int bt = a.pool.block_tokens, Dh = a.pool.head_dim, Hkv = a.pool.kv_heads;
  const int kept = a.kept_lens[b];
  if (kept > a.max_kept) {
    if (tid == 0 && j == 0 && h == 0) atomicOr(a.err, kErrTooManySplits);
    return;
  }
  if (j * bt >= kept) return;
  const int32_t *keep = a.keep + ((size_t)b * Hkv + h) * a.keep_stride;
  int64_t limit = min((int64_t)a.seq_lens[b], (int64_t)a.src_max_blocks * bt);
  if (a.w_in) limit = min(limit, a.w_in_stride);
  // slot of kept token i, or -1
  auto slot_of = [&](int i) -> int64_t {
    if (i >= kept) return -1;
    const int p = keep[i];
    if (p < 0 || p >= limit) return -1;
    const int64_t blk = a.src_tables[(size_t)b * a.src_max_blocks + p / bt];
    return blk < 0 || blk >= a.pool.n_blocks ? -1 : blk * bt + p % bt;
  };
  for (int t = tid; t < bt; t += 256) {
    const int i = j * bt + t;
    if (i >= kept) break;
    const int64_t s = slot_of(i);
    if (s < 0) atomicOr(a.err, kErrBadBlock);
    if (a.w_out)
      a.w_out[((size_t)b * Hkv + h) * a.w_out_stride + i] =
          s < 0 ? 0.0f : a.w_in[((size_t)b * Hkv + h) * a.w_in_stride + keep[i]];
  }
  const int64_t dst = a.dst_tables[(size_t)b * a.dst_max_blocks + j];
  if (dst < 0 || dst >= a.pool.n_blocks) {
    if (tid == 0) atomicOr(a.err, kErrBadBlock);
    return;
  }
  const size_t dbh = (size_t)dst * Hkv + h;
  const int n = bt * Dh;
  if (a.pool.format != kFp8) {
    for (int tensor = 0; tensor < 2; tensor++) {
      const void *src = tensor ? a.pool.v : a.pool.k;
      void *out = tensor ? a.v_dst : a.k_dst;
      for (int e = tid; e < n; e += 256) {
        const int t = tensor ? e % bt : e / Dh, d = tensor ? e / bt : e % Dh;
        const int64_t s = slot_of(j * bt + t);
        const size_t sbh = (size_t)(s < 0 ? 0 : s / bt) * Hkv + h;
        const int off = (int)(s < 0 ? 0 : s % bt);
        const size_t from = tensor ? (sbh * Dh + d) * bt + off : (sbh * bt + off) * Dh + d;
        const size_t to = dbh * n + e;
        if (is16(a.pool.format))
          static_cast<uint16_t *>(out)[to] = s < 0 ? 0 : static_cast<const uint16_t *>(src)[from];
        else
          static_cast<uint8_t *>(out)[to] = s < 0 ? 0 : static_cast<const uint8_t *>(src)[from];
      }
    }
    if (a.pool.format == kInt8)
      for (int t = tid; t < bt; t += 256) {
        const int64_t s = slot_of(j * bt + t);
        const size_t sbh = (size_t)(s < 0 ? 0 : s / bt) * Hkv + h;
        const size_t from = int8_scale_index(sbh, (int)(s < 0 ? 0 : s % bt), bt);
        const size_t to = int8_scale_index(dbh, t, bt);
        static_cast<uint16_t *>(a.ks_dst)[to] = s < 0 ? 0 : static_cast<const uint16_t *>(a.pool.k_scales)[from];
        static_cast<uint16_t *>(a.vs_dst)[to] = s < 0 ? 0 : static_cast<const uint16_t *>(a.pool.v_scales)[from];
      }
    return;
  }
  __shared__ float red[256];
  for (int tensor = 0; tensor < 2; tensor++) {
    auto elem = [&](int e) {
      const int t = tensor ? e % bt : e / Dh, d = tensor ? e / bt : e % Dh;
      const int64_t s = slot_of(j * bt + t);
      return s < 0 ? 0.0f : pool_elem(a.pool, tensor, s / bt, h, (int)(s % bt), d);
    };
    float mx = 0.0f;
    for (int e = tid; e < n; e += 256) mx = fmaxf(mx, fabsf(elem(e)));
    red[tid] = mx;
    __syncthreads();
    for (int st = 128; st > 0; st >>= 1) {
      if (tid < st) red[tid] = fmaxf(red[tid], red[tid + st]);
      __syncthreads();
    }
    const float sc = red[0] == 0.0f ? 0.0f : __fdiv_rn(red[0], 448.0f);
    __syncthreads();
    for (int e = tid; e < n; e += 256)
      static_cast<uint8_t *>(tensor ? a.v_dst : a.k_dst)[dbh * n + e] =
          sc == 0.0f ? 0 : encode_e4m3(__fdiv_rn(elem(e), sc));
    if (tid == 0) static_cast<float *>(tensor ? a.vs_dst : a.ks_dst)[fp8_scale_index(dbh)] = sc;
  }
}

}  // namespace

hipError_t launch_kv_select(const SelectArgs &a, hipStream_t s) {
  if (a.num_seqs <= 0) return hipSuccess;
  hipLaunchKernelGGL(kv_select_kernel, dim3(a.kv_heads, a.num_seqs), dim3(kSelectThreads), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_kv_compact(const CompactArgs &a, hipStream_t s) {
  const int blocks = (a.max_kept + a.pool.block_tokens - 1) / a.pool.block_tokens;
  if (a.num_seqs <= 0 || blocks <= 0) return hipSuccess;
  hipLaunchKernelGGL(kv_compact_generic_kernel, dim3(blocks, a.pool.kv_heads, a.num_seqs), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace llh
