// Norms of queries and keys for each head, with the position rotation in the same pass, and the
// keys' and values' way into the paged cache.
//
//   y = x / sqrt(mean(x^2) + eps) * (weight + offset)        over a head's elements
//   (y_i, y_j) -> (y_i cos a - y_j sin a, y_j cos a + y_i sin a),  a = position * inv_freq
//
// f32 throughout, one rounding (bf16) at the end; a key bound for an fp16 pool is rounded to bf16
// first, so that the pool holds what a separate append of the bf16 row would have stored.
//
// The angle is wanted modulo one turn only.  position * inv_freq / 2 pi in f64 (24 + 31 bits of
// product, rounded to 53) keeps 2^-22 turns and better at any int32 position; its distance to the
// nearest whole turn then goes to v_sin_f32 / v_cos_f32, which take turns, as f32 (about 2^-20 off at
// most: a bf16 output is rounded by 2^-9 and more).
//
// Bound: memory for prompts, launch and one chain of loads for tokens.  Measured on MI355X with append: 4096
// tokens, Hq32 / Hkv4, head_dim 128 (84 MB) 19.6 us, 4.3 TB/s of the 4.8 of a copy (a wavefront a row: 66);
// one token 3.5 us of the GPU.
#include "wave_ops.h"

namespace llh {

namespace {

__device__ __forceinline__ void turn(int pos, float inv_freq, float &c, float &s) {
  const double t = (double)pos * ((double)inv_freq * 0.15915494309189535);
  const float r = (float)(t - __builtin_rint(t));
  c = __builtin_amdgcn_cosf(r);
  s = __builtin_amdgcn_sinf(r);
}

__device__ __forceinline__ float wave_sum(float v, int lane) {
  v = row_sum16(v);
  v += xor16_other(v, lane);
  return v + xor32_other(v, lane);
}

// One wavefront per (token, head): any head_dim up to 512, stride and alignment.  Heads are the
// queries', the keys', then (with a destination for them) the values'.
__global__ __launch_bounds__(64) void qk_rope_generic_kernel(const QkRopeArgs a) {
  const int i = blockIdx.x;
  const int lane = threadIdx.x;
  const int Dh = a.head_dim;
  int h = blockIdx.y;
  const int which = h < a.q_heads ? 0 : h < a.q_heads + a.kv_heads ? 1 : 2;
  h -= which == 0 ? 0 : which == 1 ? a.q_heads : a.q_heads + a.kv_heads;
  const uint16_t *src = (which == 0 ? a.q + i * a.q_stride : which == 1 ? a.k + i * a.k_stride : a.v + i * a.v_stride) +
                        (size_t)h * Dh;
  const uint16_t *weight = which == 0 ? a.q_weight : which == 1 ? a.k_weight : nullptr;
  __shared__ float y[kRopeMaxDim];
  float sum = 0.0f;
  for (int d = lane; d < Dh; d += 64) {
    const float x = bf16_lo(src[d]);
    y[d] = x;
    sum += x * x;
  }
  sum = wave_sum(sum, lane);
  if (weight) {
    const float inv = 1.0f / sqrtf(sum / (float)Dh + a.eps);
    for (int d = lane; d < Dh; d += 64) y[d] = y[d] * inv * (bf16_lo(weight[d]) + a.offset);
  }
  __syncthreads();
  if (which < 2 && a.rotary_dim > 0) {
    const int half = a.rotary_dim / 2;
    const int pos = a.positions[i];
    for (int p = lane; p < half; p += 64) {
      const int u = a.adjacent ? 2 * p : p, v = a.adjacent ? 2 * p + 1 : p + half;
      float c, s;
      turn(pos, a.inv_freq[p], c, s);
      const float yu = y[u], yv = y[v];
      y[u] = yu * c - yv * s;
      y[v] = yv * c + yu * s;
    }
    __syncthreads();
  }
  uint16_t *out = which == 0   ? a.q_out + ((size_t)i * a.q_heads + h) * Dh
                  : which == 1 ? (a.k_out ? a.k_out + ((size_t)i * a.kv_heads + h) * Dh : nullptr)
                               : (a.v_out ? a.v_out + ((size_t)i * a.kv_heads + h) * Dh : nullptr);
  if (out) {
    for (int d = lane; d < Dh; d += 64) out[d] = f32_to_bf16_rne(y[d]);
    return;
  }
  const int64_t slot = a.slots[i];
  const int bt = a.pool.block_tokens;
  const int64_t blk = slot / bt;
  if (slot < 0 || blk >= a.pool.n_blocks) {
    if (lane == 0) atomicOr(a.err, kErrBadBlock);
    return;
  }
  const size_t bh = (size_t)blk * a.kv_heads + h;
  const int off = (int)(slot % bt);
  uint16_t *dst = reinterpret_cast<uint16_t *>(which == 1 ? a.k_dst : a.v_dst);
  for (int d = lane; d < Dh; d += 64) {
    const uint16_t e = f32_to_bf16_rne(y[d]);
    const size_t at = which == 1 ? (bh * bt + off) * Dh + d : (bh * Dh + d) * bt + off;
    dst[at] = a.pool.format == kF16 ? f32_to_f16_bits(bf16_lo(e)) : e;
  }
}

// head_dim 128 or 256, rows of 16-byte pieces: a row is 16 (32) lanes of 8 elements.  The groups
// of lanes of a token share its heads out, so that a lane turns the same elements of every head and
// computes its sines and cosines once.  Behind the workgroups of the queries' and keys' rows come
// those that put the values into the pool (values_to_pool), in the same launch.
//
// PAIRS: which element turns with which.  kAdjacent: 2i and 2i + 1, in one lane; kHalves: i and
// i + R / 2, a lane R / 16 further (R a multiple of 16), by a shuffle; kFull: the same at R = D, by DPP
// (or a permlane swap at 256).
enum { kAdjacent, kHalves, kFull };

__device__ __forceinline__ void unpack8(const u32x4_t &w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = bf16_lo(w[i]);
    x[2 * i + 1] = bf16_hi(w[i]);
  }
}
__device__ __forceinline__ u32x4_t load8(const uint16_t *p) { return *reinterpret_cast<const u32x4_t *>(p); }
// Outputs and values may lie anywhere (ALIGNED: at 16 bytes): what a row's numbers are does not
// depend on it.
template <bool ALIGNED>
__device__ __forceinline__ u32x4_t load8_any(const uint16_t *p) {
  if constexpr (ALIGNED) return load8(p);
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
  return w;
}
template <bool ALIGNED>
__device__ __forceinline__ void store8_any(uint16_t *p, const u32x4_t &w) {
  if constexpr (ALIGNED) {
    *reinterpret_cast<u32x4_t *>(p) = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    p[2 * i] = (uint16_t)w[i];
    p[2 * i + 1] = (uint16_t)(w[i] >> 16);
  }
}
__device__ __forceinline__ u32x4_t to_f16(const u32x4_t &w) {
  u32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; i++) r[i] = pack_f16(bf16_lo(w[i]), bf16_hi(w[i]));
  return r;
}

// Puts the values of one kv head of 16 tokens into a bf16 or fp16 pool.  V lies dim-major, 16 tokens
// of a dim side by side, so tokens that fill a whole block are turned in LDS and written 16 bytes a
// lane; rows of the call that fill a block need not start at a multiple of 16 of them, so a workgroup
// takes the runs that start in its 16 rows (a run: neighbouring rows in neighbouring slots of one
// block), wherever they end.  Runs that do not fill a block are written element by element, a
// row per wavefront.  The 16 rows are loaded beside their slots, which only say where they go.
template <int D, bool ALIGNED>
__device__ __forceinline__ void values_to_pool(const QkRopeArgs &a, int tile, int h) {
  constexpr int BT = kFastBlockTokens;
  constexpr int LT = D / 8, ROUND = 256 / LT;  // lanes a row, rows a round
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i0 = tile * BT;
  const bool f16 = a.pool.format == kF16;
  uint16_t *const v_dst = static_cast<uint16_t *>(a.v_dst);
  const uint16_t *const src = a.v + (size_t)h * D;
  __shared__ uint16_t lv[BT][D + 8];
  // 16 rows from row i on (the call's last again past it) into registers, and from there to LDS as stored
  u32x4_t w[BT / ROUND];
  auto load_rows = [&](int i) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < BT / ROUND; r++)
      w[r] = load8_any<ALIGNED>(src + min(i + r * ROUND + tid / LT, a.n - 1) * a.v_stride + 8 * (tid % LT));
  };
  auto rows_to_lds = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < BT / ROUND; r++)
      *reinterpret_cast<u32x4_t *>(&lv[r * ROUND + tid / LT][8 * (tid % LT)]) = f16 ? to_f16(w[r]) : w[r];
    __syncthreads();
  };
  load_rows(i0);
  // lane l: the slot of row i0 - 1 + l
  const int i = i0 - 1 + lane;
  const int64_t slot = lane <= 32 && i >= 0 && i < a.n ? a.slots[i] : -1;
  const bool valid = slot >= 0 && slot / BT < a.pool.n_blocks;
  const int64_t prev = __shfl_up(slot, 1);
  const bool prev_valid = __shfl_up((int)valid, 1) != 0;
  const bool start = !(lane > 0 && prev_valid && slot == prev + 1) || slot % BT == 0;
  if (tid >= 1 && tid <= BT && i < a.n && !valid && h == 0) atomicOr(a.err, kErrBadBlock);
  const uint64_t starts = __ballot(valid && start && lane >= 1 && lane <= BT);
  const uint64_t conts = __ballot(valid && !start);
  auto slot_of = [&](int l) __attribute__((always_inline)) {
    return ((int64_t)__builtin_amdgcn_readlane((int)(slot >> 32), l) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)slot, l);
  };
  rows_to_lds();

  // runs that do not fill a block: this workgroup's own rows from LDS, further ones from memory
  uint64_t whole = 0, loose = 0;
  for (uint64_t m = starts; m; m &= m - 1) {
    const int l0 = __builtin_ctzll(m);
    const int len = 1 + __builtin_ctzll(~(conts >> (l0 + 1)));  // a run ends with its block: within the 33 slots
    if (len == BT) whole |= 1ull << l0;
    else loose |= ((1ull << len) - 1) << l0;
  }
  for (int k = 0; k < wave; k++) loose &= loose - 1;
  while (loose) {  // a row a wavefront
    const int l = __builtin_ctzll(loose);
    const int64_t at = slot_of(l);
    uint16_t *out = v_dst + ((size_t)(at / BT) * a.kv_heads + h) * (D * BT) + at % BT;
#pragma unroll
    for (int d = lane; d < D; d += 64) {
      uint16_t x;
      if (l <= BT) {
        x = lv[l - 1][d];
      } else {
        x = src[(i0 - 1 + l) * a.v_stride + d];
        if (f16) x = f32_to_f16_bits(bf16_lo(x));
      }
      out[d * BT] = x;
    }
    for (int j = 0; j < 4; j++) loose &= loose - 1;
  }
  for (; whole; whole &= whole - 1) {
    const int l0 = __builtin_ctzll(whole);
    if (l0 != 1) {
      load_rows(i0 - 1 + l0);
      __syncthreads();  // the rows before these have been read
      rows_to_lds();
    }
    uint16_t *out = v_dst + ((size_t)(slot_of(l0) / BT) * a.kv_heads + h) * (D * BT);
#pragma unroll
    for (int r = 0; r < D * 2 / 256; r++) {
      const int d = (r * 256 + tid) >> 1, half = tid & 1;
      u32x4_t o;
#pragma unroll
      for (int x = 0; x < 4; x++)
        o[x] = (uint32_t)lv[8 * half + 2 * x][d] | ((uint32_t)lv[8 * half + 2 * x + 1][d] << 16);
      *reinterpret_cast<u32x4_t *>(out + d * BT + 8 * half) = o;
    }
  }
}

// GP: groups of lanes that share a token's rows out.  row_wgs: workgroups of rows.
template <int D, int PAIRS, int GP, bool ALIGNED>
__global__ __launch_bounds__(256) void qk_rope_kernel(const QkRopeArgs a, int row_wgs) {
  constexpr int BT = kFastBlockTokens;
  constexpr int LT = D / 8;
  constexpr int TOKENS = 256 / LT / GP;  // of a workgroup
  constexpr int FLIGHT = 3;              // rows of a group in flight
  if ((int)blockIdx.x >= row_wgs) {
    const int x = blockIdx.x - row_wgs;
    values_to_pool<D, ALIGNED>(a, x / a.kv_heads, x % a.kv_heads);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int c = tid % LT, group = tid / LT;
  const int i = blockIdx.x * TOKENS + group / GP;
  const bool live = i < a.n;
  const int token = min(i, a.n - 1);
  const int R = a.rotary_dim;
  const bool turned = 8 * c < R;
  const int heads = a.q_heads + a.kv_heads + (a.v_out ? a.kv_heads : 0);
  u32x4_t raw[FLIGHT];
  auto load_rows = [&](int h0) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < FLIGHT; k++) {
      const int h = min(h0 + k * GP, heads - 1);
      const uint16_t *src = h < a.q_heads ? a.q + token * a.q_stride + (size_t)h * D
                            : h < a.q_heads + a.kv_heads
                                ? a.k + token * a.k_stride + (size_t)(h - a.q_heads) * D
                                : a.v + token * a.v_stride + (size_t)(h - a.q_heads - a.kv_heads) * D;
      raw[k] = load8_any<ALIGNED>(src + 8 * c);
    }
  };
  load_rows(group % GP);  // in flight behind the angles
  float cs[8], sn[8];
  if (R > 0) {
    const int pos = a.positions[token];
    const int f0 = PAIRS == kAdjacent ? 4 * c : 8 * c < R / 2 ? 8 * c : 8 * c - R / 2;  // (R / 2: a multiple of 8)
    float freq[8];
#pragma unroll
    for (int e = 0; e < (PAIRS == kAdjacent ? 4 : 8); e++) freq[e] = turned ? a.inv_freq[f0 + e] : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (PAIRS == kAdjacent && (e & 1)) continue;
      turn(pos, freq[PAIRS == kAdjacent ? e / 2 : e], cs[e], sn[e]);
      if (PAIRS == kAdjacent) {
        cs[e + 1] = cs[e];
        sn[e + 1] = sn[e];
        sn[e] = -sn[e];
      } else if (8 * c < R / 2) {
        sn[e] = -sn[e];
      }
    }
  }
  const int partner = 8 * c < R / 2 ? lane + R / 16 : turned ? lane - R / 16 : lane;
  float wq[8] = {}, wk[8] = {};
  if (a.q_weight) unpack8(load8(a.q_weight + 8 * c), wq);
  if (a.k_weight) unpack8(load8(a.k_weight + 8 * c), wk);
#pragma unroll
  for (int e = 0; e < 8; e++) {
    wq[e] += a.offset;
    wk[e] += a.offset;
  }
  // the key's row of kv head 0 in the pool
  uint16_t *k_row = nullptr;
  if (a.slots) {
    const int64_t slot = a.slots[token];
    if (slot >= 0 && slot / BT < a.pool.n_blocks)
      k_row = static_cast<uint16_t *>(a.k_dst) + ((size_t)(slot / BT) * a.kv_heads * BT + slot % BT) * D;
    else if (live && group % GP == 0 && c == 0)
      atomicOr(a.err, kErrBadBlock);
  }
  for (int h0 = group % GP; h0 < heads; h0 += GP * FLIGHT) {
    if (h0 >= GP) load_rows(h0);
#pragma unroll
    for (int k = 0; k < FLIGHT; k++) {
      const int h = h0 + k * GP;
      const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
      float y[8];
      unpack8(raw[k], y);
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e++) sum += y[e] * y[e];
      sum = row_sum16(sum);
      if constexpr (LT == 32) sum += xor16_other(sum, lane);
      if (!is_v && (is_q ? a.q_weight : a.k_weight)) {
        const float inv = 1.0f / sqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = y[e] * inv * (is_q ? wq[e] : wk[e]);
      }
      if (R > 0) {
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
          z[e] = PAIRS == kAdjacent ? y[e ^ 1]
                 : PAIRS == kHalves ? __shfl(y[e], partner)
                 : LT == 32         ? xor16_other(y[e], lane)
                                    : dpp<0x128>(y[e]);  // row_ror 8
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = turned && !is_v ? y[e] * cs[e] + z[e] * sn[e] : y[e];
      }
      if (!live || h >= heads) continue;
      u32x4_t w;
#pragma unroll
      for (int e = 0; e < 4; e++) w[e] = pack_bf16(y[2 * e], y[2 * e + 1]);
      if (is_q) {
        store8_any<ALIGNED>(a.q_out + ((size_t)i * a.q_heads + h) * D + 8 * c, w);
      } else if (is_v) {
        store8_any<ALIGNED>(a.v_out + ((size_t)i * a.kv_heads + (h - a.q_heads - a.kv_heads)) * D + 8 * c, raw[k]);
      } else if (a.k_out) {
        store8_any<ALIGNED>(a.k_out + ((size_t)i * a.kv_heads + (h - a.q_heads)) * D + 8 * c, w);
      } else if (k_row) {
        store8_any<true>(k_row + (h - a.q_heads) * (BT * D) + 8 * c, a.pool.format == kF16 ? to_f16(w) : w);
      }
    }
  }
}

template <int D, int PAIRS, int GP, bool ALIGNED>
void launch_rope_t(const QkRopeArgs &a, hipStream_t s) {
  constexpr int TOKENS = 256 / (D / 8) / GP;
  const int row_wgs = (a.n + TOKENS - 1) / TOKENS;
  const int value_wgs = a.k_out ? 0 : (a.n + kFastBlockTokens - 1) / kFastBlockTokens * a.kv_heads;
  hipLaunchKernelGGL((qk_rope_kernel<D, PAIRS, GP, ALIGNED>), dim3(row_wgs + value_wgs), dim3(256), 0, s, a, row_wgs);
}

// Few tokens: one a workgroup, its rows side by side; many: four groups of lanes a token, whose sines and
// cosines then serve more heads.  Measured on MI355X, one a workgroup / four groups (us), with append:
// Hq32 / Hkv4, head_dim 128: 256 tokens 4.6 / 7.1, 512 5.6 / 7.5, 1024 8.5 / 8.1, 4096 24.1 / 18.3; Hq16 / Hkv8
// 4.4 / 5.7, 5.5 / 6.1, 8.1 / 7.0, 22.9 / 15.5; Hq16 / Hkv2, head_dim 256: 5.1 / 6.3, 6.8 / 6.8, 10.5 / 9.2, 30.4 / 25.0.
template <int D, int PAIRS>
void launch_rope_p(const QkRopeArgs &a, bool aligned, hipStream_t s) {
  constexpr int ALL = 256 / (D / 8);
  if (!aligned) launch_rope_t<D, PAIRS, ALL, false>(a, s);
  else if (a.n >= 1024) launch_rope_t<D, PAIRS, 4, true>(a, s);
  else launch_rope_t<D, PAIRS, ALL, true>(a, s);
}

template <int D>
void launch_rope_d(const QkRopeArgs &a, bool aligned, hipStream_t s) {
  if (a.adjacent) launch_rope_p<D, kAdjacent>(a, aligned, s);
  else if (a.rotary_dim == D) launch_rope_p<D, kFull>(a, aligned, s);
  else launch_rope_p<D, kHalves>(a, aligned, s);
}

bool at16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

bool qk_rope_pieces(const QkRopeArgs &a) {
  return (a.head_dim == 128 || a.head_dim == 256) && a.rotary_dim % 16 == 0 && at16(a.q) && at16(a.k) &&
         a.q_stride % 8 == 0 && a.k_stride % 8 == 0 && at16(a.q_weight) && at16(a.k_weight);
}

hipError_t launch_qk_rope(const QkRopeArgs &a, hipStream_t s) {
  if (a.n <= 0) return hipSuccess;
  if (qk_rope_pieces(a)) {
    const bool aligned = at16(a.q_out) && at16(a.k_out) && at16(a.v_out) && at16(a.v) && a.v_stride % 8 == 0;
    if (!a.k_out && a.pool.block_tokens != kFastBlockTokens) return hipErrorInvalidValue;
    if (a.head_dim == 128) launch_rope_d<128>(a, aligned, s);
    else launch_rope_d<256>(a, aligned, s);
    return hipGetLastError();
  }
  const bool values = a.v_out || !a.k_out;
  hipLaunchKernelGGL(qk_rope_generic_kernel, dim3(a.n, a.q_heads + a.kv_heads * (values ? 2 : 1)), dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace llh
