// C entries of the operators for batches of sequences: checks of arguments, then the launches.
#include <exception>
#include <string>

#include "batch.h"
#include "internal.h"

using namespace spx;

namespace {

// The context's device for the length of a call, the caller's afterwards.
struct OnDevice {
  int was = -1;
  hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&was);
    if (err == hipSuccess && was != device) err = hipSetDevice(device);
    else was = -1;
  }
  ~OnDevice() { if (was >= 0) (void)hipSetDevice(was); }
};

// No exception leaves a C entry (error texts allocate).
template <class F>
int entry(F f) {
  try {
    return f();
  } catch (const std::exception &) {
    return -1;
  }
}

bool pow2(int v) { return v > 0 && (v & (v - 1)) == 0; }
bool page_ok(int p) { return pow2(p) && p >= 16 && p <= 256; }
int log2_of(int v) { return 31 - __builtin_clz((unsigned)v); }
bool row_type(int t) { return t == SPX_F32 || t == SPX_F16 || t == SPX_BF16; }
int64_t size_of(int t) { return t == SPX_F32 ? 4 : 2; }
bool aligned(const void *p, int64_t a) { return (uintptr_t)p % (uintptr_t)a == 0; }
// Arrays of 32-bit numbers. (Kernels read some of them by scalar loads, which drop an address's last two bits.)
template <class... T>
bool words(T... p) { return (aligned(p, 4) && ...); }

// nullptr, or what is wrong with the shape.
const char *shape_error(const spx_kv4_shape *s) {
  if (!s) return "null shape";
  if (s->head_dim != 64 && s->head_dim != 128) return "head_dim must be 64 or 128";
  if (s->n_kv < 1 || s->n_kv > 1024) return "n_kv must be in 1..1024";
  if (!page_ok(s->page_tokens)) return "page_tokens must be a power of two in 16..256";
  if (s->n_pages < 1 || (int64_t)s->n_pages * s->page_tokens > INT32_MAX) return "n_pages must be positive, n_pages * page_tokens below 2^31";
  return nullptr;
}

int rows_call(const char *who, spx_ctx *ctx, const spx_kv4_shape *shape, const void *pool, int type, const void *k, int64_t ld_k,
              const void *v, int64_t ld_v, int rows, const int32_t *slots, bool write) {
  const std::string name(who);
  if (const char *e = shape_error(shape)) return fail(name + ": " + e);
  if (rows < 0 || rows > 1 << 24) return fail(name + ": rows must be in 0..2^24");
  if (!row_type(type)) return fail(name + ": type must be SPX_F32, SPX_F16 or SPX_BF16");
  if (rows > 0 && (!pool || !k || !v || !slots)) return fail(name + ": null argument");
  const int64_t width = (int64_t)shape->n_kv * shape->head_dim;
  if (rows > 1 && (ld_k < width || ld_v < width)) return fail(name + ": leading dimension too small");
  if (!aligned(pool, 16) || !aligned(k, size_of(type)) || !aligned(v, size_of(type)) || !aligned(slots, 4))
    return fail(name + ": the pool's address must be a multiple of 16, the others of their elements' size");
  if (!ctx) return fail(name + ": null context");
  if (rows == 0) return 0;
  OnDevice dev(ctx->device);
  if (dev.err != hipSuccess) return hip_fail(dev.err, who);
  Kv4Rows a{};
  a.pool = (uint8_t *)const_cast<void *>(pool);
  a.n_kv = shape->n_kv;
  a.page = log2_of(shape->page_tokens);
  a.n_pages = shape->n_pages;
  a.rows = rows;
  a.k = const_cast<void *>(k);
  a.v = const_cast<void *>(v);
  a.ld_k = ld_k;
  a.ld_v = ld_v;
  a.slots = slots;
  if (write) SPX_HIP(launch_kv4_append(a, shape->head_dim, type, ctx->stream));
  else SPX_HIP(launch_kv4_read(a, shape->head_dim, type, ctx->stream));
  return 0;
}

}  // namespace

extern "C" {

int spx_pages_plan(spx_ctx *ctx, int n_seq, int page_tokens, int table_cols, int n_pages, int rows, const int32_t *lens,
                   const int32_t *add, const int32_t *n_free, int32_t *tables, int32_t *free_list, int32_t *lens_out,
                   int32_t *n_free_out, int32_t *q_start, int32_t *slots, int32_t *positions, int32_t *status) {
  return entry([&] {
    if (!lens || !add || !n_free || !tables || !free_list || !lens_out || !n_free_out || !q_start || !status)
      return fail("spx_pages_plan: null argument");
    if (n_seq < 1 || n_seq > PLAN_MAX_SEQ) return fail("spx_pages_plan: n_seq must be in 1..4096");
    if (!page_ok(page_tokens)) return fail("spx_pages_plan: page_tokens must be a power of two in 16..256");
    if (table_cols < 1 || (int64_t)n_seq * table_cols > INT32_MAX) return fail("spx_pages_plan: table_cols must be positive, n_seq * table_cols below 2^31");
    if (n_pages < 1 || (int64_t)n_pages * page_tokens > INT32_MAX) return fail("spx_pages_plan: n_pages must be positive, n_pages * page_tokens below 2^31");
    if (rows < 0 || rows > 1 << 18) return fail("spx_pages_plan: rows must be in 0..262144");
    if (rows > 0 && (!slots || !positions)) return fail("spx_pages_plan: null argument");
    if (!words(lens, add, n_free, tables, free_list, lens_out, n_free_out, q_start, slots, positions, status))
      return fail("spx_pages_plan: addresses must be multiples of 4");
    if (!ctx) return fail("spx_pages_plan: null context");
    OnDevice dev(ctx->device);
    if (dev.err != hipSuccess) return hip_fail(dev.err, "spx_pages_plan");
    PlanArgs a{n_seq, log2_of(page_tokens), table_cols, n_pages, rows, lens, add, n_free, tables, free_list, lens_out, n_free_out, q_start, slots, positions, status};
    SPX_HIP(launch_pages_plan(a, ctx->stream));
    return 0;
  });
}

int64_t spx_kv4_bytes(const spx_kv4_shape *shape) {
  if (shape_error(shape)) return 0;
  return (int64_t)shape->n_pages * shape->n_kv * (shape->page_tokens / 16) * (18 * shape->head_dim);
}

int spx_kv4_append(spx_ctx *ctx, const spx_kv4_shape *shape, void *pool, int type, const void *k, int64_t ld_k, const void *v,
                   int64_t ld_v, int rows, const int32_t *slots) {
  return entry([&] { return rows_call("spx_kv4_append", ctx, shape, pool, type, k, ld_k, v, ld_v, rows, slots, true); });
}

int spx_kv4_read(spx_ctx *ctx, const spx_kv4_shape *shape, const void *pool, int type, int rows, const int32_t *slots, void *k,
                 int64_t ld_k, void *v, int64_t ld_v) {
  return entry([&] { return rows_call("spx_kv4_read", ctx, shape, pool, type, k, ld_k, v, ld_v, rows, slots, false); });
}

int64_t spx_kv4_attention_ws(const spx_kv4_shape *shape, int n_heads, int rows, int n_seq, int max_kv) {
  if (shape_error(shape) || n_heads < 1 || n_heads > 1024 || n_heads % shape->n_kv || rows < 1 || rows > 1 << 18 || n_seq < 1 ||
      n_seq > PLAN_MAX_SEQ || max_kv < 0)
    return 0;
  return kv4_attention_ws(shape->head_dim, n_heads / shape->n_kv, shape->n_kv, rows, n_seq, max_kv);
}

int spx_kv4_attention(spx_ctx *ctx, const spx_kv4_shape *shape, const void *pool, int type, const void *q, int64_t ld_q,
                      int n_heads, int rows, int n_seq, const int32_t *q_start, const int32_t *kv_lens, const int32_t *tables,
                      int table_cols, float scale, int window, int max_kv, void *out, int64_t ld_out, void *ws,
                      int64_t ws_bytes) {
  return entry([&] {
    if (const char *e = shape_error(shape)) return fail(std::string("spx_kv4_attention: ") + e);
    if (!row_type(type)) return fail("spx_kv4_attention: type must be SPX_F32, SPX_F16 or SPX_BF16");
    if (n_heads < 1 || n_heads > 1024 || n_heads % shape->n_kv) return fail("spx_kv4_attention: n_heads must be a multiple of n_kv, at most 1024");
    if (rows < 0 || rows > 1 << 18) return fail("spx_kv4_attention: rows must be in 0..262144");
    if (n_seq < 0 || n_seq > PLAN_MAX_SEQ) return fail("spx_kv4_attention: n_seq must be in 0..4096");
    if (window < 0) return fail("spx_kv4_attention: window must not be negative");
    if (max_kv < 0) return fail("spx_kv4_attention: max_kv must not be negative");
    const bool work = rows > 0 && n_seq > 0;
    if (work && (!pool || !q || !out || !q_start || !kv_lens || !tables)) return fail("spx_kv4_attention: null argument");
    if ((work && table_cols < 1) || table_cols < 0 || (int64_t)table_cols * shape->page_tokens > 1 << 30)
      return fail("spx_kv4_attention: table_cols must be positive, table_cols * page_tokens at most 2^30");
    const int64_t width = (int64_t)n_heads * shape->head_dim;
    if (rows > 1 && (ld_q < width || ld_out < width)) return fail("spx_kv4_attention: leading dimension too small");
    if (!aligned(pool, 16) || !aligned(q, size_of(type)) || !aligned(out, size_of(type)) || !words(q_start, kv_lens, tables))
      return fail("spx_kv4_attention: the pool's address must be a multiple of 16, the others of their elements' size");
    if (!(scale < __builtin_inff())) return fail("spx_kv4_attention: scale must be finite");
    const int64_t want = spx_kv4_attention_ws(shape, n_heads, rows, n_seq, max_kv);
    if (work && want > 0 && (!ws || ws_bytes < want || !aligned(ws, 16)))
      return fail("spx_kv4_attention: ws must hold " + std::to_string(want) + " bytes at an address that is a multiple of 16");
    if (!ctx) return fail("spx_kv4_attention: null context");
    if (!work) return 0;
    OnDevice dev(ctx->device);
    if (dev.err != hipSuccess) return hip_fail(dev.err, "spx_kv4_attention");
    Kv4Attn a{};
    a.pool = (const uint8_t *)pool;
    a.n_kv = shape->n_kv;
    a.page = log2_of(shape->page_tokens);
    a.n_pages = shape->n_pages;
    a.q = q;
    a.out = out;
    a.ld_q = ld_q;
    a.ld_out = ld_out;
    a.group = n_heads / shape->n_kv;
    a.rows = rows;
    a.n_seq = n_seq;
    a.cols = table_cols;
    a.window = window > 1 << 30 ? 0 : window;  // (no sequence is longer)
    a.q_start = q_start;
    a.kv_lens = kv_lens;
    a.tables = tables;
    a.part = (float *)ws;
    a.scale = (float)((scale > 0.0f ? (double)scale : 1.0 / __builtin_sqrt((double)shape->head_dim)) * 1.4426950408889634);
    SPX_HIP(launch_kv4_attention(a, shape->head_dim, type, max_kv, ctx->stream));
    return 0;
  });
}

int64_t spx_logprobs_ws(int rows, int vocab, int top_n) {
  if (rows < 1 || rows > 1 << 18 || vocab < 1 || vocab > 1 << 24 || top_n < 0 || top_n > 32) return 0;
  const int64_t parts = logprobs_parts(rows, vocab);
  return parts > 1 ? rows * parts * (16 + 8 * (int64_t)top_n) : 0;
}

int spx_logprobs(spx_ctx *ctx, int type, const void *logits, int64_t ld, int rows, int vocab, float logit_scale,
                 const int32_t *targets, int top_n, float *logp, float *entropy, int32_t *top_ids, float *top_logp, void *ws,
                 int64_t ws_bytes) {
  return entry([&] {
    if (!row_type(type)) return fail("spx_logprobs: type must be SPX_F32, SPX_F16 or SPX_BF16");
    if (rows < 0 || rows > 1 << 18) return fail("spx_logprobs: rows must be in 0..262144");
    if (vocab < 1 || vocab > 1 << 24) return fail("spx_logprobs: vocab must be in 1..2^24");
    if (top_n < 0 || top_n > 32) return fail("spx_logprobs: top_n must be in 0..32");
    if (!(logit_scale > 0.0f) || !(logit_scale < __builtin_inff())) return fail("spx_logprobs: logit_scale must be positive and finite");
    if (rows > 0 && (!logits || (top_n > 0 && (!top_ids || !top_logp)))) return fail("spx_logprobs: null argument");
    if ((targets != nullptr) != (logp != nullptr)) return fail("spx_logprobs: targets and logp go together");
    if (rows > 1 && ld < vocab) return fail("spx_logprobs: leading dimension too small");
    if (!aligned(logits, size_of(type)) || !words(targets, logp, entropy, top_ids, top_logp))
      return fail("spx_logprobs: addresses must be multiples of the elements' size");
    const int64_t want = spx_logprobs_ws(rows, vocab, top_n);
    if (rows > 0 && want > 0 && (!ws || ws_bytes < want || !aligned(ws, 16)))
      return fail("spx_logprobs: ws must hold " + std::to_string(want) + " bytes at an address that is a multiple of 16");
    if (!ctx) return fail("spx_logprobs: null context");
    if (rows == 0) return 0;
    OnDevice dev(ctx->device);
    if (dev.err != hipSuccess) return hip_fail(dev.err, "spx_logprobs");
    LogprobArgs a{logits, ld, rows, vocab, top_n, logit_scale, targets, logp, entropy, top_logp, top_ids, ws};
    SPX_HIP(launch_logprobs(a, type, ctx->stream));
    return 0;
  });
}

}  // extern "C"
