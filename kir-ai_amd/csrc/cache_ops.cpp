// Host side of the operators around an evicting cache: norms and rotation on the way in
// (qkrope.hip), selection and compaction (evict.hip).
#include <cmath>

#include "host_state.h"

using namespace llh;

namespace {

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_rope(llh_ctx *ctx, const llh_qk_rope_desc *d, const void *d_q_out) {
  if (d->num_tokens < 0) return ctx->fail(LLH_ERR_INVALID_SHAPE, "negative token count");
  if (d->num_q_heads <= 0 || d->num_kv_heads <= 0 || d->head_dim <= 0)
    return ctx->fail(LLH_ERR_INVALID_SHAPE, "head counts and head_dim must be positive");
  if (d->rotary_dim < 0 || d->rotary_dim > d->head_dim || d->rotary_dim % 2)
    return ctx->fail(LLH_ERR_INVALID_SHAPE, "rotary_dim must be even and at most head_dim");
  if (d->pairs != LLH_ROPE_HALVES && d->pairs != LLH_ROPE_ADJACENT)
    return ctx->fail(LLH_ERR_INVALID_SHAPE, "unknown rotation pairs");
  if (d->head_dim > kRopeMaxDim) {
    ctx->not_handled++;
    return ctx->fail(LLH_ERR_UNSUPPORTED, "norm and rotation take head_dim <= " + std::to_string(kRopeMaxDim));
  }
  if (d->q_stride < (int64_t)d->num_q_heads * d->head_dim || d->k_stride < (int64_t)d->num_kv_heads * d->head_dim)
    return ctx->fail(LLH_ERR_INVALID_SHAPE, "a token's stride must hold its heads");
  if (!std::isfinite(d->eps) || d->eps < 0.0f || !std::isfinite(d->weight_offset))
    return ctx->fail(LLH_ERR_NON_FINITE, "eps must be finite and >= 0, the weight offset finite");
  if ((int64_t)d->num_q_heads + 2 * (int64_t)d->num_kv_heads > 65535)
    return ctx->fail(LLH_ERR_INVALID_SHAPE, "too many heads");
  if (d->num_tokens == 0) return LLH_OK;
  if (!d->d_q || !d->d_k || !d_q_out || (d->rotary_dim > 0 && (!d->d_inv_freq || !d->d_positions)))
    return ctx->fail(LLH_ERR_NULL, "null device pointer in norm and rotation call");
  if (!aligned(d->d_q, 2) || !aligned(d->d_k, 2) || !aligned(d_q_out, 2) || !aligned(d->d_q_weight, 2) ||
      !aligned(d->d_k_weight, 2) || !aligned(d->d_inv_freq, 4) || !aligned(d->d_positions, 4))
    return ctx->fail(LLH_ERR_INVALID_SHAPE, "a pointer is not aligned to its elements");
  return LLH_OK;
}

QkRopeArgs rope_args(const llh_qk_rope_desc *d, void *d_q_out) {
  QkRopeArgs a{};
  a.q = static_cast<const uint16_t *>(d->d_q);
  a.k = static_cast<const uint16_t *>(d->d_k);
  a.v = static_cast<const uint16_t *>(d->d_v);
  a.q_stride = d->q_stride;
  a.k_stride = d->k_stride;
  a.v_stride = d->v_stride;
  a.q_weight = static_cast<const uint16_t *>(d->d_q_weight);
  a.k_weight = static_cast<const uint16_t *>(d->d_k_weight);
  a.inv_freq = d->d_inv_freq;
  a.positions = d->d_positions;
  a.q_out = static_cast<uint16_t *>(d_q_out);
  a.n = d->num_tokens;
  a.q_heads = d->num_q_heads;
  a.kv_heads = d->num_kv_heads;
  a.head_dim = d->head_dim;
  a.rotary_dim = d->rotary_dim;
  a.adjacent = d->pairs == LLH_ROPE_ADJACENT;
  a.eps = d->eps;
  a.offset = d->weight_offset;
  return a;
}

}  // namespace

extern "C" {

size_t llh_qk_rope_workspace_bytes(int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim) {
  if (num_tokens <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
  return 2 * align_up((size_t)num_tokens * num_kv_heads * head_dim * sizeof(uint16_t));
}

size_t llh_kv_select_workspace_bytes(int32_t num_seqs, int32_t kv_heads, int32_t max_seq_len) {
  if (num_seqs <= 0 || kv_heads <= 0 || max_seq_len <= 0 || max_seq_len > kSelectMaxLen) return 0;
  return select_scratch_bytes(num_seqs, kv_heads, max_seq_len);
}

int llh_qk_norm_rope(llh_ctx *ctx, const llh_qk_rope_desc *desc, void *d_q_out, void *d_k_out, void *stream) {
  if (!ctx || !desc) return LLH_ERR_NULL;
  return guarded(ctx, [&]() -> int {
    const int st = check_rope(ctx, desc, d_q_out);
    if (st != LLH_OK || desc->num_tokens == 0) return st;
    if (!d_k_out) return ctx->fail(LLH_ERR_NULL, "null device pointer in norm and rotation call");
    if (!aligned(d_k_out, 2)) return ctx->fail(LLH_ERR_INVALID_SHAPE, "a pointer is not aligned to its elements");
    const DeviceGuard on(ctx);
    if (on.status != hipSuccess) return ctx->hip_fail(on.status, "hipSetDevice");
    QkRopeArgs a = rope_args(desc, d_q_out);
    a.k_out = static_cast<uint16_t *>(d_k_out);
    a.v = nullptr;
    a.v_stride = 0;
    const hipError_t e = launch_qk_rope(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return ctx->hip_fail(e, "norm and rotation launch");
    return LLH_OK;
  });
}

int llh_qk_norm_rope_append(llh_ctx *ctx, llh_kv_pool *pool, const llh_qk_rope_desc *desc, const int64_t *d_slots,
                            void *d_q_out, void *stream) {
  if (!ctx || !pool || !desc) return LLH_ERR_NULL;
  return guarded(ctx, [&]() -> int {
    int st = check_rope(ctx, desc, d_q_out);
    if (st != LLH_OK) return st;
    if (desc->num_kv_heads != pool->view.kv_heads || desc->head_dim != pool->view.head_dim)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "kv heads and head_dim must be the pool's");
    if (desc->v_stride < (int64_t)desc->num_kv_heads * desc->head_dim)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "a token's stride must hold its heads");
    if (desc->num_tokens == 0) return LLH_OK;
    if (!desc->d_v || !d_slots) return ctx->fail(LLH_ERR_NULL, "null device pointer in norm and rotation call");
    if (!aligned(desc->d_v, 2) || !aligned(d_slots, 8))
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "a pointer is not aligned to its elements");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const DeviceGuard on(ctx);
    if (on.status != hipSuccess) return ctx->hip_fail(on.status, "hipSetDevice");
    QkRopeArgs a = rope_args(desc, d_q_out);
    if (is16(pool->view.format) && (pool->view.block_tokens == kFastBlockTokens || !qk_rope_pieces(a))) {
      a.slots = d_slots;
      a.pool = pool->view;
      a.k_dst = pool->k;
      a.v_dst = pool->v;
      a.err = ctx->err_word(s);
      ctx->append_calls++;
      const hipError_t e = launch_qk_rope(a, s);
      if (e != hipSuccess) return ctx->hip_fail(e, "norm, rotation and append launch");
      return LLH_OK;
    }
    // other pools: the bf16 rows in the stream's scratch, then the append kernel
    const size_t bytes = llh_qk_rope_workspace_bytes(desc->num_tokens, desc->num_kv_heads, desc->head_dim) / 2;
    WsLease lease;
    char *ws = nullptr;
    st = lease.acquire_ops(ctx, s, 2 * bytes, &ws);
    if (st != LLH_OK) return st;
    a.k_out = reinterpret_cast<uint16_t *>(ws);
    a.v_out = reinterpret_cast<uint16_t *>(ws + bytes);
    const hipError_t e = launch_qk_rope(a, s);
    if (e != hipSuccess) return ctx->hip_fail(e, "norm and rotation launch");
    return llh_kv_append(ctx, pool, d_slots, a.k_out, a.v_out, desc->num_tokens, stream);
  });
}

int llh_kv_select(llh_ctx *ctx, const llh_kv_select_desc *desc, const float *d_weights, int32_t *d_keep,
                  int32_t *d_kept_lens, void *stream) {
  if (!ctx || !desc) return LLH_ERR_NULL;
  return guarded(ctx, [&]() -> int {
    if (desc->num_seqs < 0 || desc->num_seqs > 65535)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "num_seqs must be 0 .. 65535");
    if (desc->kv_heads <= 0 || desc->kv_heads > 65535)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "kv_heads must be 1 .. 65535");
    if (desc->budget <= 0 || desc->sinks < 0 || desc->recent < 0 ||
        (int64_t)desc->sinks + desc->recent > desc->budget)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "budget must be positive and hold the sinks and the recent tokens");
    if (desc->max_seq_len < 0 || desc->max_seq_len > kSelectMaxLen || desc->weights_stride < desc->max_seq_len)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "max_seq_len must be 0 .. 2^30 and at most weights_stride");
    if (desc->keep_stride < std::min(desc->budget, desc->max_seq_len))
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "keep_stride must hold the kept positions");
    if (desc->num_seqs == 0) return LLH_OK;
    if (!d_weights || !d_keep || !d_kept_lens || !desc->d_seq_lens)
      return ctx->fail(LLH_ERR_NULL, "null device pointer in selection call");
    if (!aligned(d_weights, 4) || !aligned(d_keep, 4) || !aligned(d_kept_lens, 4) || !aligned(desc->d_seq_lens, 4))
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "a pointer is not aligned to its elements");
    if (d_kept_lens == desc->d_seq_lens)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "the kept lengths must not replace the lengths they come from");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const DeviceGuard on(ctx);
    if (on.status != hipSuccess) return ctx->hip_fail(on.status, "hipSetDevice");
    SelectArgs a{};
    a.weights = d_weights;
    a.seq_lens = desc->d_seq_lens;
    a.keep = d_keep;
    a.kept_lens = d_kept_lens;
    a.weights_stride = desc->weights_stride;
    a.keep_stride = desc->keep_stride;
    a.err = ctx->err_word(s);
    a.num_seqs = desc->num_seqs;
    a.kv_heads = desc->kv_heads;
    a.max_seq_len = desc->max_seq_len;
    a.budget = desc->budget;
    a.sinks = desc->sinks;
    a.recent = desc->recent;
    WsLease lease;
    const size_t bytes = select_scratch_bytes(a.num_seqs, a.kv_heads, a.max_seq_len);
    if (bytes) {
      char *ws = nullptr;
      const int st = lease.acquire_ops(ctx, s, bytes, &ws);
      if (st != LLH_OK) return st;
      a.scratch = ws;
    }
    const hipError_t e = launch_kv_select(a, s);
    if (e != hipSuccess) return ctx->hip_fail(e, "selection launch");
    return LLH_OK;
  });
}

int llh_kv_compact(llh_ctx *ctx, llh_kv_pool *pool, const llh_kv_compact_desc *desc, void *stream) {
  if (!ctx || !pool || !desc) return LLH_ERR_NULL;
  return guarded(ctx, [&]() -> int {
    const PoolView &pv = pool->view;
    if (desc->num_seqs < 0 || desc->num_seqs > 65535)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "num_seqs must be 0 .. 65535");
    if (pv.kv_heads > 65535) return ctx->fail(LLH_ERR_INVALID_SHAPE, "too many heads");
    if (desc->src_max_blocks <= 0 || desc->dst_max_blocks <= 0)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "block-table rows must not be empty");
    if (desc->max_kept < 0 || desc->max_kept > desc->keep_stride ||
        desc->max_kept > (int64_t)desc->dst_max_blocks * pv.block_tokens)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "max_kept must fit keep_stride and the destination rows");
    // (a launch dimension's threads, 512 a block, and the kernels' 32-bit offsets inside a block)
    if (((int64_t)desc->max_kept + pv.block_tokens - 1) / pv.block_tokens > kCompactMaxBlocks ||
        desc->max_kept > kSelectMaxLen || (int64_t)pv.block_tokens * pv.head_dim > (1 << 30))
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "max_kept must be at most 2^30 tokens in 2^22 blocks");
    if ((desc->d_weights_in == nullptr) != (desc->d_weights_out == nullptr))
      return ctx->fail(LLH_ERR_NULL, "weights are moved from an input to an output: both or neither");
    if (desc->d_weights_in && (desc->weights_in_stride < 0 || desc->weights_out_stride < desc->max_kept))
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "weights_out_stride must hold the kept tokens");
    if (pv.format == LLH_KV_INT8_ROW) {
      ctx->not_handled++;
      return ctx->fail(LLH_ERR_UNSUPPORTED, "a token's scale spans all heads, which keep different tokens");
    }
    if (desc->num_seqs == 0 || desc->max_kept == 0) return LLH_OK;
    if (!desc->d_seq_lens || !desc->d_kept_lens || !desc->d_keep || !desc->d_src_tables || !desc->d_dst_tables)
      return ctx->fail(LLH_ERR_NULL, "null device pointer in compaction call");
    if (!aligned(desc->d_seq_lens, 4) || !aligned(desc->d_kept_lens, 4) || !aligned(desc->d_keep, 4) ||
        !aligned(desc->d_src_tables, 4) || !aligned(desc->d_dst_tables, 4) || !aligned(desc->d_weights_in, 4) ||
        !aligned(desc->d_weights_out, 4))
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "a pointer is not aligned to its elements");
    if (desc->d_weights_in && desc->d_weights_in == desc->d_weights_out)
      return ctx->fail(LLH_ERR_INVALID_SHAPE, "the weights' output must not be their input");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const DeviceGuard on(ctx);
    if (on.status != hipSuccess) return ctx->hip_fail(on.status, "hipSetDevice");
    CompactArgs a{};
    a.pool = pv;
    a.k_dst = pool->k;
    a.v_dst = pool->v;
    a.ks_dst = pool->ks;
    a.vs_dst = pool->vs;
    a.seq_lens = desc->d_seq_lens;
    a.kept_lens = desc->d_kept_lens;
    a.keep = desc->d_keep;
    a.src_tables = desc->d_src_tables;
    a.dst_tables = desc->d_dst_tables;
    a.w_in = desc->d_weights_in;
    a.w_out = desc->d_weights_out;
    a.keep_stride = desc->keep_stride;
    a.w_in_stride = desc->weights_in_stride;
    a.w_out_stride = desc->weights_out_stride;
    a.err = ctx->err_word(s);
    a.num_seqs = desc->num_seqs;
    a.max_kept = desc->max_kept;
    a.src_max_blocks = desc->src_max_blocks;
    a.dst_max_blocks = desc->dst_max_blocks;
    const hipError_t e = launch_kv_compact(a, s);
    if (e != hipSuccess) return ctx->hip_fail(e, "compaction launch");
    return LLH_OK;
  });
}

}  // extern "C"
