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
// nearest whole turn then goes to v_sin_f32 / v_cos_f32, which take turns, as f32.
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

}  // namespace

hipError_t launch_qk_rope(const QkRopeArgs &a, hipStream_t s) {
  if (a.n <= 0) return hipSuccess;
  const bool values = a.v_out || !a.k_out;
  hipLaunchKernelGGL(qk_rope_generic_kernel, dim3(a.n, a.q_heads + a.kv_heads * (values ? 2 : 1)), dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace llh
