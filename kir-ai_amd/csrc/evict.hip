// Eviction from the paged cache by accumulated attention weight: the choice of the tokens to keep
// (kv_select) and their move to other blocks (kv_compact).
#include <type_traits>

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

// The same over 16-token blocks at head_dim 128 or 256: one workgroup of D ES lanes per (destination
// block, kv head, sequence), a 16-byte piece of a K row and of a source block's V tile per lane.
// Every wavefront looks the block's 16 tokens up for itself, one per lane, and takes what is
// uniform from there by v_readlane.  K rows go straight through.  V lies dim-major, so a token's
// column cannot be read without its block's tile: the tiles of the kept tokens' blocks (positions
// ascend, so each is met once) are read whole, eight in flight, and the kept columns picked into an LDS tile
// [token][dim], from which every lane writes 16 bytes of one dim row.
template <int D, int FMT>
__global__ __launch_bounds__(D * (is16(FMT) ? 2 : 1)) void kv_compact_kernel(const CompactArgs a) {
  constexpr int BT = kFastBlockTokens;
  constexpr int ES = is16(FMT) ? 2 : 1;
  constexpr int PIECES = D * ES / 16;   // 16-byte pieces of a token's row
  constexpr int FLIGHT = 8;
  constexpr bool FP8 = FMT == kFp8;
  typedef typename std::conditional<ES == 2, uint16_t, uint8_t>::type elem_t;
  // neighbouring destination blocks share a source block: give each XCD (workgroups go round them) a run
  const int nx = gridDim.x, xcd = blockIdx.x % 8;
  const int j = xcd * (nx / 8) + min(xcd, nx % 8) + (int)blockIdx.x / 8;
  const int h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63;
  const int Hkv = a.pool.kv_heads;
  // lane t (mod 16): token t of the block; its position is loaded beside the lengths (the row holds
  // max_kept entries whatever the length is)
  const int mine = j * BT + (lane & 15);
  const size_t row = (size_t)b * Hkv + h;
  const int pos = a.keep[row * a.keep_stride + min(mine, a.max_kept - 1)];
  const int dst = a.dst_tables[(size_t)b * a.dst_max_blocks + j];
  const int kept = a.kept_lens[b];
  if (kept > a.max_kept) {
    if (tid == 0 && j == 0 && h == 0) atomicOr(a.err, kErrTooManySplits);
    return;
  }
  if (j * BT >= kept) return;
  int64_t limit = min((int64_t)a.seq_lens[b], (int64_t)a.src_max_blocks * BT);
  if (a.w_in) limit = min(limit, a.w_in_stride);
  // its source block (-1: none) and offset
  const int p = mine < kept ? pos : -1;
  const bool inside = p >= 0 && p < limit;
  int blk = inside ? a.src_tables[(size_t)b * a.src_max_blocks + p / BT] : -1;
  if (blk < 0 || blk >= a.pool.n_blocks) blk = -1;
  const int off = p & (BT - 1);
  if (tid < BT && mine < kept) {
    if (blk < 0) atomicOr(a.err, kErrBadBlock);
    if (a.w_out) a.w_out[row * a.w_out_stride + mine] = blk < 0 ? 0.0f : a.w_in[row * a.w_in_stride + p];
  }
  if (dst < 0 || dst >= a.pool.n_blocks) {
    if (tid == 0) atomicOr(a.err, kErrBadBlock);
    return;
  }
  const size_t dbh = (size_t)dst * Hkv + h;

  // ---- K: this lane's piece of token kt ----
  const int kt = tid / PIECES, kc = tid % PIECES;
  const int kblk = __shfl(blk, kt), koff = __shfl(off, kt);
  u32x4_t kw = {0, 0, 0, 0};
  if (kblk >= 0)
    kw = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(
        static_cast<const char *>(a.pool.k) + ((((size_t)kblk * Hkv + h) * BT + koff) * D * ES + 16 * kc)));
  // scales: int8 the token's pair, fp8 the source blocks' pairs (lane t: token t's)
  uint32_t pair = 0;
  float ks = 0.0f, vs = 0.0f;
  if constexpr (FMT == kInt8) {
    if (tid < BT && blk >= 0)
      pair = *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(a.pool.k_scales) +
                                                 int8_scale_index((size_t)blk * Hkv + h, off, BT));
  }
  if constexpr (FP8) {
    if (blk >= 0) {
      const float2 t = *reinterpret_cast<const float2 *>(static_cast<const float *>(a.pool.k_scales) +
                                                         fp8_scale_index((size_t)blk * Hkv + h));
      ks = t.x;
      vs = t.y;
    }
  }

  // ---- V: the kept columns into LDS ----
  // a lane's piece of a tile: dim vd, tokens 8 vh .. +7 (16-bit) or all 16 (8-bit)
  constexpr int PAD = ES == 2 ? 8 : 16;
  __shared__ __attribute__((aligned(16))) elem_t lv[BT][D + PAD];
  const int vd = ES == 2 ? tid >> 1 : tid;
  const int vh = ES == 2 ? tid & 1 : 0;
  const int prev = __shfl(blk, max(lane - 1, 0));
  uint32_t starts = (uint32_t)(__ballot(lane < BT && blk >= 0 && (lane == 0 || prev != blk)) & 0xffffu);
  const uint32_t none = (uint32_t)(__ballot(lane < BT && blk < 0) & 0xffffu);
  for (uint32_t m = none; m; m &= m - 1) {
    if (vh == 0) lv[__builtin_ctz(m)][vd] = 0;
  }
  while (starts) {
    u32x4_t w[FLIGHT];
    uint32_t left = starts;
#pragma unroll
    for (int f = 0; f < FLIGHT; f++) {
      if (left) {
        const int t = __builtin_ctz(left);
        left &= left - 1;
        const int sb = __builtin_amdgcn_readlane(blk, t);
        w[f] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(
            static_cast<const char *>(a.pool.v) + ((size_t)sb * Hkv + h) * (BT * D * ES) + 16 * tid));
      }
    }
#pragma unroll
    for (int f = 0; f < FLIGHT; f++) {
      if (!starts) break;
      const int t0 = __builtin_ctz(starts);
      starts &= starts - 1;
      const uint32_t ends = (starts | none | 0x10000u) >> (t0 + 1);
      const int t1 = t0 + 1 + __builtin_ctz(ends);
      for (int t = t0; t < t1; t++) {
        const int o = __builtin_amdgcn_readlane(off, t);
        const int e = ES == 2 ? o & 7 : o;  // element of the piece
        const int x = e >> (ES == 2 ? 1 : 2);
        const uint32_t word = x == 0 ? w[f][0] : x == 1 ? w[f][1] : x == 2 ? w[f][2] : w[f][3];
        const elem_t v = (elem_t)(word >> (8 * ES * (e & (4 / ES - 1))));
        if (ES == 1 || (o >> 3) == vh) lv[t][vd] = v;
      }
    }
  }

  if constexpr (!FP8) {
    *reinterpret_cast<u32x4_t *>(static_cast<char *>(a.k_dst) + dbh * (BT * D * ES) + 16 * tid) = kw;
    if constexpr (FMT == kInt8) {
      if (tid < BT)
        *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.ks_dst) + int8_scale_index(dbh, tid, BT)) = pair;
    }
    __syncthreads();
    u32x4_t out;
    if constexpr (ES == 2) {
#pragma unroll
      for (int x = 0; x < 4; x++)
        out[x] = (uint32_t)lv[8 * vh + 2 * x][vd] | ((uint32_t)lv[8 * vh + 2 * x + 1][vd] << 16);
    } else {
#pragma unroll
      for (int x = 0; x < 4; x++)
        out[x] = (uint32_t)lv[4 * x][vd] | ((uint32_t)lv[4 * x + 1][vd] << 8) | ((uint32_t)lv[4 * x + 2][vd] << 16) |
                 ((uint32_t)lv[4 * x + 3][vd] << 24);
    }
    *reinterpret_cast<u32x4_t *>(static_cast<char *>(a.v_dst) + dbh * (BT * D * ES) + 16 * tid) = out;
    return;
  } else {
    // fp8: the kept rows' values, the block's new scales (the largest magnitudes / 448), new codes
    __shared__ uint32_t s_max[2];
    if (tid < 2) s_max[tid] = 0;
    __syncthreads();
    const float kst = __shfl(ks, kt);
    float x[2][16];
#pragma unroll
    for (int e = 0; e < 16; e++) x[0][e] = decode_e4m3((kw[e >> 2] >> (8 * (e & 3))) & 0xffu) * kst;
#pragma unroll
    for (int t = 0; t < BT; t++)
      x[1][t] = decode_e4m3(lv[t][vd]) * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), t));
#pragma unroll
    for (int tensor = 0; tensor < 2; tensor++) {
      float m = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; e++) m = fmaxf(m, fabsf(x[tensor][e]));
      m = fmaxf(m, dpp<0xB1>(m));
      m = fmaxf(m, dpp<0x4E>(m));
      m = fmaxf(m, dpp<0x141>(m));
      m = fmaxf(m, dpp<0x140>(m));
      m = fmaxf(m, xor16_other(m, lane));
      m = fmaxf(m, xor32_other(m, lane));
      if (lane == 0) atomicMax(&s_max[tensor], __float_as_uint(m));  // magnitudes order as integers
    }
    __syncthreads();
#pragma unroll
    for (int tensor = 0; tensor < 2; tensor++) {
      const float top = __uint_as_float(s_max[tensor]);
      const float sc = top == 0.0f ? 0.0f : __fdiv_rn(top, 448.0f);
      u32x4_t out = {0, 0, 0, 0};
      if (sc != 0.0f) {
#pragma unroll
        for (int e = 0; e < 16; e++) out[e >> 2] |= (uint32_t)encode_e4m3(__fdiv_rn(x[tensor][e], sc)) << (8 * (e & 3));
      }
      *reinterpret_cast<u32x4_t *>(static_cast<char *>(tensor ? a.v_dst : a.k_dst) + dbh * (BT * D) + 16 * tid) = out;
      if (tid == 0) static_cast<float *>(tensor ? a.vs_dst : a.ks_dst)[fp8_scale_index(dbh)] = sc;
    }
  }
}

template <int D>
void launch_compact_d(const CompactArgs &a, dim3 grid, hipStream_t s) {
  switch (a.pool.format) {
    case kInt8:
      hipLaunchKernelGGL((kv_compact_kernel<D, kInt8>), grid, dim3(D), 0, s, a);
      break;
    case kFp8:
      hipLaunchKernelGGL((kv_compact_kernel<D, kFp8>), grid, dim3(D), 0, s, a);
      break;
    default:  // bf16 and fp16 elements move alike
      hipLaunchKernelGGL((kv_compact_kernel<D, kBf16>), grid, dim3(2 * D), 0, s, a);
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
  const dim3 grid(blocks, a.pool.kv_heads, a.num_seqs);
  if (a.pool.block_tokens == kFastBlockTokens && a.pool.head_dim == 128) launch_compact_d<128>(a, grid, s);
  else if (a.pool.block_tokens == kFastBlockTokens && a.pool.head_dim == 256) launch_compact_d<256>(a, grid, s);
  else hipLaunchKernelGGL(kv_compact_generic_kernel, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace llh
