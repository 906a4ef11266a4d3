// Every call below is refused before anything is launched: the context and the pool are host
// objects, and no GPU is needed.  Prints one line per wrong status.
#include <cmath>
#include <cstdio>
#include <initializer_list>

#include "host_state.h"

static int failures = 0;

static void expect(const char *what, int got, int want) {
  if (got != want) {
    std::printf("%s: status %d, expected %d\n", what, got, want);
    failures++;
  }
}

// A device pointer that nothing may read: aligned, and not mapped.
template <typename T>
static T *dev(uintptr_t off = 0) { return reinterpret_cast<T *>(uintptr_t{0x10000} + off); }

static llh_ctx ctx;

static llh_kv_pool pool_of(int32_t format, int32_t bt, int32_t heads, int32_t dim) {
  llh_kv_pool p;
  p.ctx = &ctx;
  p.k = p.v = p.ks = p.vs = dev<void>();
  p.view = llh::PoolView{format, bt, heads, dim, 8, p.k, p.v, p.ks, p.vs};
  return p;
}

static llh_qk_rope_desc rope() {
  llh_qk_rope_desc d{};
  d.num_tokens = 3;
  d.num_q_heads = 4;
  d.num_kv_heads = 2;
  d.head_dim = 64;
  d.rotary_dim = 64;
  d.pairs = LLH_ROPE_HALVES;
  d.eps = 1e-6f;
  d.q_stride = 4 * 64;
  d.k_stride = d.v_stride = 2 * 64;
  d.d_q = d.d_k = d.d_v = d.d_q_weight = d.d_k_weight = dev<void>();
  d.d_inv_freq = dev<float>();
  d.d_positions = dev<int32_t>();
  return d;
}

template <typename F>
static void rope_case(const char *what, int want, F change) {
  llh_kv_pool pool = pool_of(LLH_KV_BF16, 16, 2, 64);
  llh_qk_rope_desc d = rope();
  change(d);
  expect(what, llh_qk_norm_rope(&ctx, &d, dev<void>(), dev<void>(), nullptr), want);
  expect(what, llh_qk_norm_rope_append(&ctx, &pool, &d, dev<int64_t>(), dev<void>(), nullptr), want);
}

static void rope_cases() {
  using D = llh_qk_rope_desc;
  rope_case("no tokens", LLH_OK, [](D &d) { d.num_tokens = 0; });
  rope_case("negative tokens", LLH_ERR_INVALID_SHAPE, [](D &d) { d.num_tokens = -1; });
  rope_case("no query heads", LLH_ERR_INVALID_SHAPE, [](D &d) { d.num_q_heads = 0; });
  rope_case("no kv heads", LLH_ERR_INVALID_SHAPE, [](D &d) { d.num_kv_heads = 0; });
  rope_case("no dims", LLH_ERR_INVALID_SHAPE, [](D &d) { d.head_dim = 0; });
  rope_case("odd rotation", LLH_ERR_INVALID_SHAPE, [](D &d) { d.rotary_dim = 31; });
  rope_case("negative rotation", LLH_ERR_INVALID_SHAPE, [](D &d) { d.rotary_dim = -2; });
  rope_case("rotation past the head", LLH_ERR_INVALID_SHAPE, [](D &d) { d.rotary_dim = 66; });
  rope_case("unknown pairs", LLH_ERR_INVALID_SHAPE, [](D &d) { d.pairs = 2; });
  rope_case("query stride", LLH_ERR_INVALID_SHAPE, [](D &d) { d.q_stride = 4 * 64 - 1; });
  rope_case("key stride", LLH_ERR_INVALID_SHAPE, [](D &d) { d.k_stride = 0; });
  rope_case("eps", LLH_ERR_NON_FINITE, [](D &d) { d.eps = NAN; });
  rope_case("negative eps", LLH_ERR_NON_FINITE, [](D &d) { d.eps = -1e-6f; });
  rope_case("offset", LLH_ERR_NON_FINITE, [](D &d) { d.weight_offset = INFINITY; });
  rope_case("null queries", LLH_ERR_NULL, [](D &d) { d.d_q = nullptr; });
  rope_case("null keys", LLH_ERR_NULL, [](D &d) { d.d_k = nullptr; });
  rope_case("null frequencies", LLH_ERR_NULL, [](D &d) { d.d_inv_freq = nullptr; });
  rope_case("null positions", LLH_ERR_NULL, [](D &d) { d.d_positions = nullptr; });
  rope_case("odd address", LLH_ERR_INVALID_SHAPE, [](D &d) { d.d_k = dev<void>(1); });
  rope_case("unaligned positions", LLH_ERR_INVALID_SHAPE, [](D &d) { d.d_positions = dev<int32_t>(2); });
  rope_case("too many heads", LLH_ERR_INVALID_SHAPE, [](D &d) {
    d.num_q_heads = 65536;
    d.q_stride = int64_t{65536} * 64;
  });
  llh_qk_rope_desc d = rope();
  llh_kv_pool pool = pool_of(LLH_KV_BF16, 16, 2, 64);
  expect("null query output", llh_qk_norm_rope(&ctx, &d, nullptr, dev<void>(), nullptr), LLH_ERR_NULL);
  expect("null key output", llh_qk_norm_rope(&ctx, &d, dev<void>(), nullptr, nullptr), LLH_ERR_NULL);
  expect("null slots", llh_qk_norm_rope_append(&ctx, &pool, &d, nullptr, dev<void>(), nullptr), LLH_ERR_NULL);
  expect("unaligned slots", llh_qk_norm_rope_append(&ctx, &pool, &d, dev<int64_t>(4), dev<void>(), nullptr),
         LLH_ERR_INVALID_SHAPE);
  expect("null desc", llh_qk_norm_rope(&ctx, nullptr, dev<void>(), dev<void>(), nullptr), LLH_ERR_NULL);
  expect("null pool", llh_qk_norm_rope_append(&ctx, nullptr, &d, dev<int64_t>(), dev<void>(), nullptr), LLH_ERR_NULL);
  d.d_v = nullptr;
  expect("null values", llh_qk_norm_rope_append(&ctx, &pool, &d, dev<int64_t>(), dev<void>(), nullptr), LLH_ERR_NULL);
  d = rope();
  d.v_stride = 127;
  expect("value stride", llh_qk_norm_rope_append(&ctx, &pool, &d, dev<int64_t>(), dev<void>(), nullptr),
         LLH_ERR_INVALID_SHAPE);
  d = rope();
  llh_kv_pool other = pool_of(LLH_KV_BF16, 16, 4, 64);
  expect("another pool's heads", llh_qk_norm_rope_append(&ctx, &other, &d, dev<int64_t>(), dev<void>(), nullptr),
         LLH_ERR_INVALID_SHAPE);
  d.head_dim = 514;
  d.q_stride = d.k_stride = d.v_stride = 4096;
  expect("head_dim", llh_qk_norm_rope(&ctx, &d, dev<void>(), dev<void>(), nullptr), LLH_ERR_UNSUPPORTED);
}

struct Weights {
  llh_kv_pool pool = pool_of(LLH_KV_BF16, 16, 2, 64);
  int32_t seqs = 2, heads = 4, blocks = 8, max_len = 100, window = 0, chunk = 4;
  const int32_t *lens = dev<int32_t>(), *tables = dev<int32_t>(), *starts = dev<int32_t>();
  const void *q = dev<void>();
  void *out = dev<void>();
  float scale = 0.125f, decay = 1.0f;
  const float *in = nullptr;
  float *w = dev<float>();
  int64_t stride = 128;
};

template <typename F>
static void weights_case(const char *what, int want, F change) {
  Weights c;
  change(c);
  llh_decode_desc d{c.seqs, c.heads, c.blocks, c.max_len, c.window, 0, c.lens, c.tables, nullptr};
  expect(what, llh_paged_decode_weights(&ctx, &c.pool, &d, c.q, c.out, c.scale, c.in, c.w, c.stride, c.decay, nullptr),
         want);
  llh_prefill_desc p{c.seqs, c.heads, c.blocks, c.window, 8, c.chunk, c.starts, c.lens, c.tables, nullptr};
  expect(what, llh_paged_prefill_weights(&ctx, &c.pool, &p, c.max_len, c.q, c.out, c.scale, c.in, c.w, c.stride, c.decay,
                                         nullptr), want);
}

static void weights_cases() {
  weights_case("no sequences", LLH_OK, [](Weights &c) { c.seqs = 0; });
  weights_case("negative sequences", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.seqs = -1; });
  weights_case("too many sequences", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.seqs = 65536; });
  weights_case("heads", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.heads = 5; });
  weights_case("blocks", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.blocks = 0; });
  weights_case("window", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.window = -1; });
  weights_case("negative length", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.max_len = -1; });
  weights_case("length past the bound", LLH_ERR_INVALID_SHAPE, [](Weights &c) {
    c.max_len = (1 << 30) + 1;
    c.stride = int64_t{1} << 31;
    c.blocks = 1 << 27;
  });
  // (tiles of 128 positions by 1024 threads: a launch dimension holds 2^32 threads)
  weights_case("length past a launch", LLH_ERR_INVALID_SHAPE, [](Weights &c) {
    c.max_len = (1 << 28) + 1;
    c.stride = int64_t{1} << 31;
    c.blocks = 1 << 27;
  });
  weights_case("weights stride", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.stride = 99; });
  weights_case("empty weights", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.stride = c.max_len = 0; });
  weights_case("null queries", LLH_ERR_NULL, [](Weights &c) { c.q = nullptr; });
  weights_case("null output", LLH_ERR_NULL, [](Weights &c) { c.out = nullptr; });
  weights_case("null weights", LLH_ERR_NULL, [](Weights &c) { c.w = nullptr; });
  weights_case("null lengths", LLH_ERR_NULL, [](Weights &c) { c.lens = nullptr; });
  weights_case("null tables", LLH_ERR_NULL, [](Weights &c) { c.tables = nullptr; });
  weights_case("odd query address", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.q = dev<void>(1); });
  weights_case("unaligned weights", LLH_ERR_INVALID_SHAPE, [](Weights &c) { c.w = dev<float>(2); });
  weights_case("scale", LLH_ERR_NON_FINITE, [](Weights &c) { c.scale = NAN; });
  weights_case("decay", LLH_ERR_NON_FINITE, [](Weights &c) { c.decay = INFINITY; });
  weights_case("head_dim", LLH_ERR_UNSUPPORTED, [](Weights &c) { c.pool = pool_of(LLH_KV_BF16, 16, 2, 516); });
  Weights c;
  llh_decode_desc d{2, 4, 8, 129, 0, 0, c.lens, c.tables, nullptr};
  expect("span past the table row",
         llh_paged_decode_weights(&ctx, &c.pool, &d, c.q, c.out, 1.0f, nullptr, c.w, 256, 1.0f, nullptr),
         LLH_ERR_INVALID_SHAPE);
  for (int chunk : {0, -1, LLH_WEIGHTS_MAX_CHUNK + 1}) {
    llh_prefill_desc p{2, 4, 8, 0, 8, chunk, c.starts, c.lens, c.tables, nullptr};
    expect("chunk length",
           llh_paged_prefill_weights(&ctx, &c.pool, &p, 100, c.q, c.out, 1.0f, nullptr, c.w, 128, 1.0f, nullptr),
           chunk > 0 ? LLH_ERR_UNSUPPORTED : LLH_ERR_INVALID_SHAPE);
  }
  llh_prefill_desc p{2, 4, 8, 0, 8, 4, nullptr, c.lens, c.tables, nullptr};
  expect("null starts",
         llh_paged_prefill_weights(&ctx, &c.pool, &p, 100, c.q, c.out, 1.0f, nullptr, c.w, 128, 1.0f, nullptr),
         LLH_ERR_NULL);
  expect("null desc",
         llh_paged_decode_weights(&ctx, &c.pool, nullptr, c.q, c.out, 1.0f, nullptr, c.w, 128, 1.0f, nullptr),
         LLH_ERR_NULL);
  expect("workspace of nothing", (int)llh_weights_workspace_bytes(0, 1, 16, 128, 100), 0);
}

template <typename F>
static void select_case(const char *what, int want, F change) {
  llh_kv_select_desc d{2, 2, 100, 32, 4, 8, 128, 32, dev<int32_t>()};
  const float *w = dev<float>();
  int32_t *keep = dev<int32_t>(), *kept = dev<int32_t>(64);
  change(d, w, keep, kept);
  expect(what, llh_kv_select(&ctx, &d, w, keep, kept, nullptr), want);
}

static void select_cases() {
  using D = llh_kv_select_desc;
  using W = const float *;
  using K = int32_t *;
  select_case("no sequences", LLH_OK, [](D &d, W &, K &, K &) { d.num_seqs = 0; });
  select_case("negative sequences", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.num_seqs = -1; });
  select_case("too many sequences", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.num_seqs = 65536; });
  select_case("no heads", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.kv_heads = 0; });
  select_case("too many heads", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.kv_heads = 65536; });
  select_case("length past the bound", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) {
    d.max_seq_len = (1 << 30) + 1;
    d.weights_stride = d.max_seq_len;
  });
  select_case("no budget", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.budget = d.sinks = d.recent = 0; });
  select_case("negative sinks", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.sinks = -1; });
  select_case("negative recent", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.recent = -1; });
  select_case("over the budget", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.recent = 29; });
  select_case("sum past 32 bits", LLH_ERR_INVALID_SHAPE,
              [](D &d, W &, K &, K &) { d.sinks = d.recent = INT32_MAX; });
  select_case("weights stride", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.weights_stride = 99; });
  select_case("negative length", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.max_seq_len = -1; });
  select_case("keep stride", LLH_ERR_INVALID_SHAPE, [](D &d, W &, K &, K &) { d.keep_stride = 31; });
  select_case("null weights", LLH_ERR_NULL, [](D &, W &w, K &, K &) { w = nullptr; });
  select_case("null positions", LLH_ERR_NULL, [](D &, W &, K &k, K &) { k = nullptr; });
  select_case("null kept lengths", LLH_ERR_NULL, [](D &, W &, K &, K &n) { n = nullptr; });
  select_case("null lengths", LLH_ERR_NULL, [](D &d, W &, K &, K &) { d.d_seq_lens = nullptr; });
  select_case("unaligned weights", LLH_ERR_INVALID_SHAPE, [](D &, W &w, K &, K &) { w = dev<float>(2); });
  select_case("lengths in place", LLH_ERR_INVALID_SHAPE, [](D &, W &, K &, K &n) { n = dev<int32_t>(); });
}

template <typename F>
static void compact_case(const char *what, int want, F change, int32_t format = LLH_KV_BF16) {
  llh_kv_pool pool = pool_of(format, 16, 2, 64);
  llh_kv_compact_desc d{2,
                        32,
                        8,
                        2,
                        32,
                        128,
                        32,
                        dev<int32_t>(),
                        dev<int32_t>(),
                        dev<int32_t>(),
                        dev<int32_t>(),
                        dev<int32_t>(),
                        dev<float>(),
                        dev<float>(4096)};
  change(d);
  expect(what, llh_kv_compact(&ctx, &pool, &d, nullptr), want);
}

static void compact_cases() {
  using D = llh_kv_compact_desc;
  compact_case("no sequences", LLH_OK, [](D &d) { d.num_seqs = 0; });
  compact_case("nothing kept", LLH_OK, [](D &d) { d.max_kept = 0; });
  compact_case("negative sequences", LLH_ERR_INVALID_SHAPE, [](D &d) { d.num_seqs = -1; });
  compact_case("too many sequences", LLH_ERR_INVALID_SHAPE, [](D &d) { d.num_seqs = 65536; });
  compact_case("no source row", LLH_ERR_INVALID_SHAPE, [](D &d) { d.src_max_blocks = 0; });
  compact_case("no destination row", LLH_ERR_INVALID_SHAPE, [](D &d) { d.dst_max_blocks = 0; });
  compact_case("negative kept", LLH_ERR_INVALID_SHAPE, [](D &d) { d.max_kept = -1; });
  compact_case("keep stride", LLH_ERR_INVALID_SHAPE, [](D &d) { d.keep_stride = 31; });
  compact_case("destination row", LLH_ERR_INVALID_SHAPE, [](D &d) { d.max_kept = d.keep_stride = 33; });
  // (the blocks of the largest int, rounded up, pass it; 2^22 blocks of 512 threads are a launch's most)
  compact_case("kept tokens past an int's blocks", LLH_ERR_INVALID_SHAPE, [](D &d) {
    d.max_kept = INT32_MAX;
    d.keep_stride = d.weights_out_stride = int64_t{1} << 31;
    d.dst_max_blocks = INT32_MAX;
  });
  compact_case("kept tokens past a launch", LLH_ERR_INVALID_SHAPE, [](D &d) {
    d.max_kept = (1 << 26) + 1;
    d.keep_stride = d.weights_out_stride = int64_t{1} << 31;
    d.dst_max_blocks = INT32_MAX;
  });
  compact_case("weights in alone", LLH_ERR_NULL, [](D &d) { d.d_weights_out = nullptr; });
  compact_case("weights out alone", LLH_ERR_NULL, [](D &d) { d.d_weights_in = nullptr; });
  compact_case("weights out stride", LLH_ERR_INVALID_SHAPE, [](D &d) { d.weights_out_stride = 31; });
  compact_case("weights in place", LLH_ERR_INVALID_SHAPE, [](D &d) { d.d_weights_out = dev<float>(); });
  compact_case("unaligned table", LLH_ERR_INVALID_SHAPE, [](D &d) { d.d_dst_tables = dev<int32_t>(2); });
  compact_case("null lengths", LLH_ERR_NULL, [](D &d) { d.d_seq_lens = nullptr; });
  compact_case("null kept lengths", LLH_ERR_NULL, [](D &d) { d.d_kept_lens = nullptr; });
  compact_case("null positions", LLH_ERR_NULL, [](D &d) { d.d_keep = nullptr; });
  compact_case("null source", LLH_ERR_NULL, [](D &d) { d.d_src_tables = nullptr; });
  compact_case("null destination", LLH_ERR_NULL, [](D &d) { d.d_dst_tables = nullptr; });
  compact_case("int8 rows", LLH_ERR_UNSUPPORTED, [](D &) {}, LLH_KV_INT8_ROW);
}

int main() {
  rope_cases();
  weights_cases();
  select_cases();
  compact_cases();
  std::printf("%d wrong\n", failures);
  return failures != 0;
}
