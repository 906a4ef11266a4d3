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

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------
//
// The k-th largest key is found by its digits of 11, 11 and 10 bits from the top: a histogram of
// the next digit over the keys that share the digits so far, and the bin in which the sum from
// the largest digit down passes k.  Eleven bits are the sign, the exponent and two bits of the
// fraction, which spreads weights over tens of bins.  The kept positions are then those of larger
// keys and the first of the equal ones, written in order by ballots.
//
// A wavefront holds 64 KPT neighbouring positions, position i * 64 + lane of them in register i:
// loads are whole whatever the rows' alignment, and order is wavefront, register, lane.
//
// Bound: latency (the load, up to three passes of a histogram, a sum over it and their barriers, the
// write).  Measured on MI355X: 32 x 8 rows of U[1025, 4096] 7.9 us, two rows of 131072 23.0.
constexpr int kBins = 2048;
constexpr int kSelectMaxKpt = 32;  // keys a thread holds of a row that one workgroup selects from

struct RowRange {
  int len, lo, hi;  // tokens; the positions to choose from
  int want;         // how many of those are kept
};
__device__ __forceinline__ RowRange row_range(const SelectArgs &a, int b) {
  const int len = a.seq_lens[b];
  return {len, a.sinks, len - a.recent, a.budget - a.sinks - a.recent};
}
// A row that needs no choice: none of it, or all.
__device__ __forceinline__ bool row_is_plain(const SelectArgs &a, int len) {
  return len < 0 || len > a.max_seq_len || len <= a.budget;
}

// Sum of v over the lanes up to this one (DPP: shifts within a row of 16, then the rows' totals).
__device__ __forceinline__ int wave_inclusive(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15: rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31: rows 2 and 3
  return v;
}

// Largest v of the wavefront, the same way.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Sum of the wavefronts' numbers before this one's.
template <int WAVES>
__device__ __forceinline__ int waves_before(const int *s_waves, int wave) {
  int before = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w += 4) {
    const int4 x = *reinterpret_cast<const int4 *>(s_waves + w);
    before += (w < wave ? x.x : 0) + (w + 1 < wave ? x.y : 0) + (w + 2 < wave ? x.z : 0) + (w + 3 < wave ? x.w : 0);
  }
  return before;
}

// Exclusive sum of v over the threads; s_waves: one int a wavefront, 16-byte aligned.
template <int WAVES>
__device__ __forceinline__ int block_exclusive(int v, int *s_waves) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int x = wave_inclusive(v);
  if (lane == 63) s_waves[wave] = x;
  __syncthreads();
  return waves_before<WAVES>(s_waves, wave) + x - v;
}

// Adds the lanes' digits to a histogram: the first lane's digit once for all lanes that share it
// (most weights may be equal), the others one by one.
__device__ __forceinline__ void count_digit(int *hist, int digit, bool on, int lane) {
  const uint64_t live = __ballot(on);
  if (!live) return;
  const int head = __builtin_amdgcn_readlane(digit, __builtin_ctzll(live));
  const uint64_t same = __ballot(on && digit == head);
  if (lane == __builtin_ctzll(live)) atomicAdd(&hist[head], __builtin_popcountll(same));
  if (on && digit != head) atomicAdd(&hist[digit], 1);
}

// The digit in which the sum of counts from the largest digit down reaches `want`, given each
// thread's counts of its 2048 / THREADS neighbouring bins, largest first from thread 0's; *want
// loses what the larger digits hold, *all: whether every key of the digit is wanted.  Ends with a
// barrier.
template <int THREADS, int PER>
__device__ __forceinline__ int find_digit(const int (&c)[PER], int top, int *want, bool *all, int *s_waves,
                                          int *s_found) {
  int sum = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) sum += c[i];
  int above = block_exclusive<THREADS / 64>(sum, s_waves);
  if (above < *want && above + sum >= *want) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      if (above < *want && above + c[i] >= *want) {
        s_found[0] = top - (int)threadIdx.x * PER - i;
        s_found[1] = above;
        s_found[2] = c[i];
      }
      above += c[i];
    }
  }
  __syncthreads();
  *want -= s_found[1];
  *all = s_found[2] == *want;
  return s_found[0];
}

// Bits of digit `pass` (0, 1, 2) and where it starts.
constexpr int kDigitShift[3] = {21, 10, 0};
constexpr uint32_t kDigitMask[3] = {2047u, 2047u, 1023u};

// Writes the kept ones of this workgroup's positions from p0 on, in order.  threshold: the least key
// kept; of the equal ones the first `equal_wanted` in the row.  n_out, n_equal: kept and
// equal positions of the row before p0.
template <int THREADS, int KPT>
__device__ __forceinline__ void write_kept(const uint32_t (&key)[KPT], const RowRange &r, int p0, uint32_t threshold,
                                           int equal_wanted, int n_out, int n_equal, int32_t *keep, int *s_waves) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t below = (1ull << lane) - 1;
  const int first = p0 + wave * 64 * KPT + lane;
  // equal keys of the wavefronts before this one
  int eq = 0;
#pragma unroll
  for (int i = 0; i < KPT; i++) {
    const int p = first + 64 * i;
    eq += __builtin_popcountll(__ballot(p >= r.lo && p < r.hi && key[i] == threshold));
  }
  __syncthreads();
  if (lane == 0) s_waves[wave] = eq;
  __syncthreads();
  n_equal += waves_before<THREADS / 64>(s_waves, wave);
  uint32_t on = 0;  // bit i: register i is kept
  int count = 0;
#pragma unroll
  for (int i = 0; i < KPT; i++) {
    const int p = first + 64 * i;
    const bool mid = p >= r.lo && p < r.hi;
    const uint64_t e = __ballot(mid && key[i] == threshold);
    const bool k = p < r.len && (!mid || key[i] > threshold ||
                                 (key[i] == threshold && n_equal + __builtin_popcountll(e & below) < equal_wanted));
    n_equal += __builtin_popcountll(e);
    count += __builtin_popcountll(__ballot(k));
    on |= k ? 1u << i : 0u;
  }
  __syncthreads();
  if (lane == 0) s_waves[wave] = count;
  __syncthreads();
  n_out += waves_before<THREADS / 64>(s_waves, wave);
#pragma unroll
  for (int i = 0; i < KPT; i++) {
    const bool k = on >> i & 1;
    const uint64_t m = __ballot(k);
    if (k) keep[n_out + __builtin_popcountll(m & below)] = first + 64 * i;
    n_out += __builtin_popcountll(m);
  }
}

template <int THREADS, int KPT>
__device__ __forceinline__ void load_keys(uint32_t (&key)[KPT], const float *w, const RowRange &r, int p0) {
  const int first = p0 + (threadIdx.x >> 6) * 64 * KPT + (threadIdx.x & 63);
  float x[KPT];
#pragma unroll
  for (int i = 0; i < KPT; i++) {
    const int p = first + 64 * i;
    x[i] = p >= r.lo && p < r.hi ? w[p] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < KPT; i++) key[i] = order_key(x[i]);
}

// What a row's first workgroup says of it: its kept length, and a length that is out of range.
__device__ __forceinline__ void row_lengths(const SelectArgs &a, int b, int len) {
  const bool bad = len < 0 || len > a.max_seq_len;
  if (bad) atomicOr(a.err, kErrTooManySplits);
  a.kept_lens[b] = bad ? 0 : min(len, a.budget);
}

// One workgroup per (sequence, kv head), which holds the row's keys in registers.
template <int THREADS, int KPT>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(const SelectArgs a) {
  constexpr int PER = kBins / THREADS;
  const int b = blockIdx.y, h = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const RowRange r = row_range(a, b);
  if (tid == 0 && h == 0) row_lengths(a, b, r.len);
  const size_t row = (size_t)b * a.kv_heads + h;
  int32_t *keep = a.keep + row * a.keep_stride;
  if (row_is_plain(a, r.len)) {
    if (r.len <= a.max_seq_len)
      for (int i = tid; i < r.len; i += THREADS) keep[i] = i;
    return;
  }
  __shared__ int hist[kBins];
  __shared__ __attribute__((aligned(16))) int s_waves[THREADS / 64];
  __shared__ int s_found[3];
  uint32_t key[KPT];
  load_keys<THREADS, KPT>(key, a.weights + row * a.weights_stride, r, 0);
  const int first = (tid >> 6) * 64 * KPT + lane;
  uint32_t threshold = 0xffffffffu;  // nothing of the middle: no key reaches it
  int want = r.want;
  if (want > 0) {
    uint32_t prefix = 0, mask = 0;
    bool all = false;
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
      if (all) break;
#pragma unroll
      for (int i = 0; i < PER; i++) hist[tid + i * THREADS] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < KPT; i++) {
        const int p = first + 64 * i;
        count_digit(hist, (int)((key[i] >> kDigitShift[pass]) & kDigitMask[pass]),
                    p >= r.lo && p < r.hi && (key[i] & mask) == prefix, lane);
      }
      __syncthreads();
      int c[PER];
#pragma unroll
      for (int i = 0; i < PER; i++) c[i] = hist[kBins - 1 - tid * PER - i];
      const int digit = find_digit<THREADS, PER>(c, kBins - 1, &want, &all, s_waves, s_found);
      prefix |= (uint32_t)digit << kDigitShift[pass];
      mask |= kDigitMask[pass] << kDigitShift[pass];
    }
    threshold = prefix;
    if (all) {  // every key from the digits so far on is kept (not every key of all: prefix > 0)
      threshold = prefix - 1;
      want = 0;
    }
  }
  write_kept<THREADS, KPT>(key, r, 0, threshold, want, 0, 0, keep, s_waves);
}

// Longer rows: tiles of kTileKeys positions and three launches.  The first leaves every tile's
// histogram of the first digit (16-bit counts, two a word) in the workspace; in the second every
// workgroup adds up its row's, finds the digit and leaves the tile's keys of that digit, a few per cent
// of them as a rule; in the third every workgroup finds the threshold among the row's such keys and writes
// its tile's positions.  No counter has to be cleared, and nothing depends on order.  Keys of the
// digit that are all equal (weights that are all zero, say) are recognised by their least and largest;
// where they differ and are yet most of a long row, the third launch reads them all in every workgroup
// (two rows of 1048576 positions: 26 us all equal, 37 spread, 1.3 ms read so).
constexpr int kTileThreads = 1024;
constexpr int kTileWaves = kTileThreads / 64;
constexpr int kTileKpt = 8;
constexpr int kTileKeys = kTileThreads * kTileKpt;
constexpr int kTileWords = kBins / 2;
struct TileCounts {
  int larger;  // keys of a larger first digit
  int cands;   // keys of the digit
  uint32_t not_least, largest;  // of those: ~ the least, the largest (0 and 0: none)
};
struct TileView {
  uint32_t *hist;      // [rows][tiles][kTileWords]
  uint32_t *cand;      // [rows][tiles][kTileKeys]
  TileCounts *counts;  // [rows][tiles]
  int2 *state;         // [rows] the first digit, and how many of its keys are wanted
};
__host__ __device__ inline size_t tile_bytes(size_t rows, size_t tiles) {
  return rows * tiles * ((kTileWords + kTileKeys) * 4 + sizeof(TileCounts)) + rows * sizeof(int2);
}
__host__ __device__ inline TileView tile_view(void *ws, size_t rows, size_t tiles) {
  TileView v;
  v.hist = static_cast<uint32_t *>(ws);
  v.cand = v.hist + rows * tiles * kTileWords;
  v.counts = reinterpret_cast<TileCounts *>(v.cand + rows * tiles * kTileKeys);
  v.state = reinterpret_cast<int2 *>(v.counts + rows * tiles);
  return v;
}

enum { kTileHist, kTileCands, kTileWrite };

template <int STEP>
__global__ __launch_bounds__(kTileThreads) void kv_select_tile_kernel(const SelectArgs a) {
  const int tile = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RowRange r = row_range(a, b);
  const size_t row = (size_t)b * a.kv_heads + h;
  int32_t *keep = a.keep + row * a.keep_stride;
  if (STEP == kTileWrite && tid == 0 && h == 0 && tile == 0) row_lengths(a, b, r.len);
  const int p0 = tile * kTileKeys;
  if (row_is_plain(a, r.len)) {
    if (STEP == kTileWrite && r.len <= a.max_seq_len)
      for (int i = p0 + tid; i < min(r.len, p0 + kTileKeys); i += kTileThreads) keep[i] = i;
    return;
  }
  if (p0 >= r.len || (STEP != kTileWrite && r.want == 0)) return;
  const int tiles = (r.len + kTileKeys - 1) / kTileKeys;
  const TileView v = tile_view(a.scratch, (size_t)a.num_seqs * a.kv_heads, gridDim.x);
  const size_t tile_row = row * gridDim.x;
  __shared__ int hist[kBins];
  __shared__ __attribute__((aligned(16))) int s_waves[kTileWaves];
  __shared__ int s_found[3];
  __shared__ int2 s_before[kTileWaves];
  __shared__ uint2 s_ends[kTileWaves];
  uint32_t key[kTileKpt];
  load_keys<kTileThreads, kTileKpt>(key, a.weights + row * a.weights_stride, r, p0);
  const int first = p0 + wave * 64 * kTileKpt + lane;
  auto clear = [&]() __attribute__((always_inline)) {
    hist[tid] = 0;
    hist[tid + kTileThreads] = 0;
    __syncthreads();
  };

  if constexpr (STEP == kTileHist) {
    clear();
#pragma unroll
    for (int i = 0; i < kTileKpt; i++) {
      const int p = first + 64 * i;
      count_digit(hist, (int)(key[i] >> kDigitShift[0]), p >= r.lo && p < r.hi, lane);
    }
    __syncthreads();
    v.hist[(tile_row + tile) * kTileWords + tid] = (uint32_t)hist[2 * tid] | ((uint32_t)hist[2 * tid + 1] << 16);
  } else if constexpr (STEP == kTileCands) {
    int c[2] = {0, 0};
    const uint32_t *words = v.hist + tile_row * kTileWords + (kTileWords - 1 - tid);
#pragma unroll 8
    for (int t = 0; t < tiles; t++) {
      const uint32_t w = words[(size_t)t * kTileWords];
      c[0] += (int)(w >> 16);
      c[1] += (int)(w & 0xffffu);
    }
    int want = r.want;
    bool all;
    const uint32_t digit = (uint32_t)find_digit<kTileThreads, 2>(c, kBins - 1, &want, &all, s_waves, s_found);
    if (tile == 0 && tid == 0) v.state[row] = make_int2((int)digit, want);
    int larger = 0, n = 0;
    uint32_t mine = 0;
    uint2 ends = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < kTileKpt; i++) {
      const int p = first + 64 * i;
      const uint32_t d = key[i] >> kDigitShift[0];
      const bool mid = p >= r.lo && p < r.hi;
      larger += __builtin_popcountll(__ballot(mid && d > digit));
      n += __builtin_popcountll(__ballot(mid && d == digit));
      mine |= mid && d == digit ? 1u << i : 0u;
      ends.x = max(ends.x, mid && d == digit ? ~key[i] : 0u);
      ends.y = max(ends.y, mid && d == digit ? key[i] : 0u);
    }
    ends = make_uint2(wave_umax(ends.x), wave_umax(ends.y));
    if (lane == 0) {
      s_before[wave] = make_int2(larger, n);
      s_ends[wave] = ends;
    }
    __syncthreads();
    int at = 0, all_larger = 0, all_n = 0;
#pragma unroll
    for (int w = 0; w < kTileWaves; w++) {
      at += w < wave ? s_before[w].y : 0;
      all_larger += s_before[w].x;
      all_n += s_before[w].y;
      ends.x = max(ends.x, s_ends[w].x);
      ends.y = max(ends.y, s_ends[w].y);
    }
    if (tid == 0) v.counts[tile_row + tile] = TileCounts{all_larger, all_n, ends.x, ends.y};
    uint32_t *cand = v.cand + (tile_row + tile) * kTileKeys;
#pragma unroll
    for (int i = 0; i < kTileKpt; i++) {
      const bool k = mine >> i & 1;
      const uint64_t m = __ballot(k);
      if (k) cand[at + __builtin_popcountll(m & ((1ull << lane) - 1))] = key[i];
      at += __builtin_popcountll(m);
    }
  } else {
    uint32_t threshold = 0xffffffffu;  // nothing of the middle: no key reaches it
    int want = 0, n_larger = 0, n_equal = 0;
    if (r.want > 0) {
      const int2 state = v.state[row];
      uint32_t prefix = (uint32_t)state.x << kDigitShift[0], mask = kDigitMask[0] << kDigitShift[0];
      want = state.y;
      // f(key, in the row, tile) for the row's keys of the digit, a tile per wavefront at a time
      auto for_cands = [&](auto f) __attribute__((always_inline)) {
        for (int t = wave; t < tiles; t += kTileWaves) {
          const int n = v.counts[tile_row + t].cands;
          const uint32_t *cand = v.cand + (tile_row + t) * kTileKeys;
          for (int i = lane; i < ((n + 63) & ~63); i += 64) f(cand[min(i, n - 1)], i < n, t);
        }
      };
      // the tiles' counts, a tile a lane (every wavefront for itself: no barrier)
      int larger = 0, equal = 0;  // of the tiles before this one
      uint2 ends = make_uint2(0, 0);
      for (int t = lane; t < tiles; t += 64) {
        const TileCounts c = v.counts[tile_row + t];
        ends.x = max(ends.x, c.not_least);
        ends.y = max(ends.y, c.largest);
        larger += t < tile ? c.larger : 0;
        equal += t < tile ? c.cands : 0;
      }
      larger = __builtin_amdgcn_readlane(wave_inclusive(larger), 63);
      equal = __builtin_amdgcn_readlane(wave_inclusive(equal), 63);
      n_larger = larger;
      ends = make_uint2(wave_umax(ends.x), wave_umax(ends.y));
      if (~ends.x == ends.y) {
        threshold = ends.y;
        n_equal = equal;
      } else {
        bool all = false;
#pragma unroll
        for (int pass = 1; pass < 3; pass++) {
          if (all) break;
          clear();
          for_cands([&](uint32_t k, bool on, int) __attribute__((always_inline)) {
            count_digit(hist, (int)((k >> kDigitShift[pass]) & kDigitMask[pass]), on && (k & mask) == prefix, lane);
          });
          __syncthreads();
          const int c[2] = {hist[kBins - 1 - 2 * tid], hist[kBins - 2 - 2 * tid]};
          const int digit = find_digit<kTileThreads, 2>(c, kBins - 1, &want, &all, s_waves, s_found);
          prefix |= (uint32_t)digit << kDigitShift[pass];
          mask |= kDigitMask[pass] << kDigitShift[pass];
        }
        threshold = prefix;
        if (all) {
          threshold = prefix - 1;
          want = 0;
        }
        larger = equal = 0;
        for_cands([&](uint32_t k, bool on, int t) __attribute__((always_inline)) {
          larger += __builtin_popcountll(__ballot(on && t < tile && k > threshold));
          equal += __builtin_popcountll(__ballot(on && t < tile && k == threshold));
        });
        if (lane == 0) s_before[wave] = make_int2(larger, equal);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kTileWaves; w++) {
          n_larger += s_before[w].x;
          n_equal += s_before[w].y;
        }
      }
    }
    const int n_out = min(p0, r.lo) + max(0, p0 - r.hi) + n_larger + min(n_equal, want);
    write_kept<kTileThreads, kTileKpt>(key, r, p0, threshold, want, n_out, n_equal, keep, s_waves);
  }
}

// ---------------------------------------------------------------------------
// compaction
// ---------------------------------------------------------------------------

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
//
// Bound: memory.  Measured on MI355X: 32 x 4096 tokens to 1024 (random ones), Hkv 8, head_dim 128, bf16: 470 MB of
// rows and tiles in 99.8 us, 4.7 TB/s (element by element 328); five ragged fp8 caches at head_dim 256 6.7
// us, the chain positions -> table -> tiles -> scale -> codes.
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

// Whether rows are selected from in tiles: beyond what a workgroup's registers hold, and somewhat below
// where there are few rows.  Measured on MI355X, a workgroup a row / tiles (us): 8 rows of 16384 18.2 /
// 24.6, 24000 28.7 / 25.3, 32768 33.3 / 24.7; 64 rows of 32768 33.7 / 27.8; 256 rows 37.7 / 99.7.
static bool select_in_tiles(int num_seqs, int kv_heads, int max_seq_len) {
  return max_seq_len > 1024 * kSelectMaxKpt ||
         (max_seq_len > 1024 * kSelectMaxKpt / 2 && (long long)num_seqs * kv_heads <= 64);
}

size_t select_scratch_bytes(int num_seqs, int kv_heads, int max_seq_len) {
  if (!select_in_tiles(num_seqs, kv_heads, max_seq_len)) return 0;
  return tile_bytes((size_t)num_seqs * kv_heads, (max_seq_len + kTileKeys - 1) / kTileKeys);
}

hipError_t launch_kv_select(const SelectArgs &a, hipStream_t s) {
  if (a.num_seqs <= 0) return hipSuccess;
  const int n = a.max_seq_len;
  const dim3 grid(a.kv_heads, a.num_seqs);
  if (!select_in_tiles(a.num_seqs, a.kv_heads, n)) {
    // short rows by fewer threads: 64 x 8 rows of 1000, 1024 threads 9.0 us, 256 6.2; 8 rows 6.1 / 5.2 (and
    // 32 x 8 of up to 4096 by 1024 threads 7.7, 512 8.6, 256 13.0)
    if (n <= 1024) hipLaunchKernelGGL((kv_select_kernel<256, 4>), grid, dim3(256), 0, s, a);
    else if (n <= 4096) hipLaunchKernelGGL((kv_select_kernel<1024, 4>), grid, dim3(1024), 0, s, a);
    else if (n <= 8192) hipLaunchKernelGGL((kv_select_kernel<1024, 8>), grid, dim3(1024), 0, s, a);
    else if (n <= 16384) hipLaunchKernelGGL((kv_select_kernel<1024, 16>), grid, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((kv_select_kernel<1024, kSelectMaxKpt>), grid, dim3(1024), 0, s, a);
    return hipGetLastError();
  }
  const dim3 tiles((n + kTileKeys - 1) / kTileKeys, a.kv_heads, a.num_seqs);
  hipLaunchKernelGGL(kv_select_tile_kernel<kTileHist>, tiles, dim3(kTileThreads), 0, s, a);
  hipLaunchKernelGGL(kv_select_tile_kernel<kTileCands>, tiles, dim3(kTileThreads), 0, s, a);
  hipLaunchKernelGGL(kv_select_tile_kernel<kTileWrite>, tiles, dim3(kTileThreads), 0, s, a);
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
