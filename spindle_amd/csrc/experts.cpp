// C entries of the operators of a mixture of experts over a batch: checks of arguments, then the launches.
#include <string>

#include "entry.h"
#include "experts.h"

using namespace spx;

namespace {

// nullptr, or what is wrong with the sizes of a routing.
const char *moe_error(int rows, int k, int n_expert) {
  if (rows < 0 || rows > MOE_MAX_ROWS) return "rows must be in 0..262144";
  if (n_expert < 1 || n_expert > MOE_MAX_E) return "n_expert must be in 1..1024";
  if (k < 1 || k > MOE_MAX_K) return "k must be in 1..32";
  return nullptr;
}

const char *mx4_error(const spx_mx4 *m) {
  if (!m) return "null matrix";
  if (spx_mx4_bytes(m->rows, m->cols) <= 0) return "a matrix has 1 or more rows, and columns in 1..2^20";
  if (!m->data) return "null data";
  if (!aligned(m->data, 16)) return "a matrix's address must be a multiple of 16";
  return nullptr;
}

// Rows in sorted order and back: the checks that the three calls share.
const char *join_error(int type, int rows, int k, int width) {
  if (!row_type(type)) return "type must be SPX_F32, SPX_F16 or SPX_BF16";
  if (const char *e = moe_error(rows, k, 1)) return e;
  if (width < 1 || width > 1 << 20) return "width must be in 1..2^20";
  return nullptr;
}

int run_on(spx_ctx *ctx, const char *who, bool work, hipError_t (*f)(const void *, int, hipStream_t), const void *a, int type) {
  if (!ctx) return fail(std::string(who) + ": null context");
  if (!work) return 0;
  OnDevice dev(ctx->device);
  if (dev.err != hipSuccess) return hip_fail(dev.err, who);
  const hipError_t e = f(a, type, ctx->stream);
  return e == hipSuccess ? 0 : hip_fail(e, who);
}
// launch(args, type, stream) as run_on takes it.
template <class A, hipError_t (*L)(const A &, int, hipStream_t)>
hipError_t launched(const void *a, int type, hipStream_t s) { return L(*(const A *)a, type, s); }

}  // namespace

extern "C" {

int spx_moe_route(spx_ctx *ctx, int type, const void *logits, int64_t ld, int rows, int n_expert, int k, int norm, int32_t *chosen,
                  float *weights) {
  return entry([&] {
    const char *who = "spx_moe_route";
    const std::string name = std::string(who) + ": ";
    if (!row_type(type)) return fail(name + "type must be SPX_F32, SPX_F16 or SPX_BF16");
    if (const char *e = moe_error(rows, k, n_expert)) return fail(name + e);
    if (k > n_expert) return fail(name + "k must be at most n_expert");
    if (norm != 0 && norm != 1) return fail(name + "norm must be 0 or 1");
    if (rows > 0 && (!logits || !chosen || !weights)) return fail(name + "null argument");
    if (rows > 1 && ld < n_expert) return fail(name + "leading dimension too small");
    if (!aligned(logits, size_of(type)) || !words(chosen, weights)) return fail(name + "addresses must be multiples of the elements' size");
    RouteArgs a{};
    a.logits = logits;
    a.ld = ld;
    a.rows = rows;
    a.n_expert = n_expert;
    a.k = k;
    a.norm = norm;
    a.chosen = chosen;
    a.weights = weights;
    return run_on(ctx, who, rows > 0, launched<RouteArgs, launch_moe_route>, &a, type);
  });
}

int spx_moe_route_grad(spx_ctx *ctx, int type, const void *logits, int64_t ld, int rows, int n_expert, int k, int norm,
                       const int32_t *chosen, const float *d_weights, void *d_logits, int64_t ld_d) {
  return entry([&] {
    const char *who = "spx_moe_route_grad";
    const std::string name = std::string(who) + ": ";
    if (!row_type(type)) return fail(name + "type must be SPX_F32, SPX_F16 or SPX_BF16");
    if (const char *e = moe_error(rows, k, n_expert)) return fail(name + e);
    if (k > n_expert) return fail(name + "k must be at most n_expert");
    if (norm != 0 && norm != 1) return fail(name + "norm must be 0 or 1");
    if (rows > 0 && (!logits || !chosen || !d_weights || !d_logits)) return fail(name + "null argument");
    if (rows > 1 && (ld < n_expert || ld_d < n_expert)) return fail(name + "leading dimension too small");
    if (!aligned(logits, size_of(type)) || !aligned(d_logits, size_of(type)) || !words(chosen, d_weights))
      return fail(name + "addresses must be multiples of the elements' size");
    RouteArgs a{};
    a.logits = logits;
    a.ld = ld;
    a.rows = rows;
    a.n_expert = n_expert;
    a.k = k;
    a.norm = norm;
    a.chosen = const_cast<int32_t *>(chosen);
    a.d_weights = d_weights;
    a.d_logits = d_logits;
    a.ld_d = ld_d;
    return run_on(ctx, who, rows > 0, launched<RouteArgs, launch_moe_route_grad>, &a, type);
  });
}

int64_t spx_moe_sort_ws(int rows, int k, int n_expert) {
  if (moe_error(rows, k, n_expert) || rows == 0) return 0;
  const int blocks = moe_sort_blocks((int64_t)rows * k);
  return blocks > 1 ? (int64_t)blocks * (n_expert + 1) * 4 : 0;
}

int spx_moe_sort(spx_ctx *ctx, int rows, int k, int n_expert, const int32_t *chosen, int32_t *starts, int32_t *order, int32_t *place,
                 void *ws, int64_t ws_bytes) {
  return entry([&] {
    const char *who = "spx_moe_sort";
    const std::string name = std::string(who) + ": ";
    if (const char *e = moe_error(rows, k, n_expert)) return fail(name + e);
    if (!starts || (rows > 0 && (!chosen || !order || !place))) return fail(name + "null argument");
    if (!words(chosen, starts, order, place)) return fail(name + "addresses must be multiples of 4");
    const int64_t want = spx_moe_sort_ws(rows, k, n_expert);
    if (want > 0 && (!ws || ws_bytes < want || !aligned(ws, 16)))
      return fail(name + "ws must hold " + std::to_string(want) + " bytes at an address that is a multiple of 16");
    SortArgs a{rows * k, n_expert, chosen, starts, order, place, (int32_t *)ws};
    const auto go = [](const void *p, int, hipStream_t s) { return launch_moe_sort(*(const SortArgs *)p, s); };
    return run_on(ctx, who, true, go, &a, 0);
  });
}

int spx_moe_gather(spx_ctx *ctx, int type, const void *x, int64_t ld_x, int rows, int k, int width, const int32_t *order,
                   const float *weights, void *out, int64_t ld_out) {
  return entry([&] {
    const char *who = "spx_moe_gather";
    const std::string name = std::string(who) + ": ";
    if (const char *e = join_error(type, rows, k, width)) return fail(name + e);
    if (rows > 0 && (!x || !order || !out)) return fail(name + "null argument");
    if ((rows > 1 && ld_x < width) || ((int64_t)rows * k > 1 && ld_out < width)) return fail(name + "leading dimension too small");
    if (!aligned(x, size_of(type)) || !aligned(out, size_of(type)) || !words(order, weights))
      return fail(name + "addresses must be multiples of the elements' size");
    JoinArgs a{};
    a.x = x;
    a.out = out;
    a.ld_x = ld_x;
    a.ld_out = ld_out;
    a.rows = rows;
    a.k = k;
    a.width = width;
    a.order = order;
    a.weights = weights;
    return run_on(ctx, who, rows > 0, launched<JoinArgs, launch_moe_gather>, &a, type);
  });
}

int spx_moe_combine(spx_ctx *ctx, int type, const void *y, int64_t ld_y, int rows, int k, int width, const int32_t *place,
                    const float *weights, void *out, int64_t ld_out) {
  return entry([&] {
    const char *who = "spx_moe_combine";
    const std::string name = std::string(who) + ": ";
    if (const char *e = join_error(type, rows, k, width)) return fail(name + e);
    if (rows > 0 && (!y || !place || !out)) return fail(name + "null argument");
    if (((int64_t)rows * k > 1 && ld_y < width) || (rows > 1 && ld_out < width)) return fail(name + "leading dimension too small");
    if (!aligned(y, size_of(type)) || !aligned(out, size_of(type)) || !words(place, weights))
      return fail(name + "addresses must be multiples of the elements' size");
    JoinArgs a{};
    a.x = y;
    a.out = out;
    a.ld_x = ld_y;
    a.ld_out = ld_out;
    a.rows = rows;
    a.k = k;
    a.width = width;
    a.place = place;
    a.weights = weights;
    return run_on(ctx, who, rows > 0, launched<JoinArgs, launch_moe_combine>, &a, type);
  });
}

int spx_moe_combine_grad(spx_ctx *ctx, int type, const void *d_out, int64_t ld_d, const void *y, int64_t ld_y, int rows, int k, int width,
                         const int32_t *order, const int32_t *place, const float *weights, void *d_y, int64_t ld_dy, float *d_weights) {
  return entry([&] {
    const char *who = "spx_moe_combine_grad";
    const std::string name = std::string(who) + ": ";
    if (const char *e = join_error(type, rows, k, width)) return fail(name + e);
    if (rows > 0 && (!d_out || !y || !order || !place || !weights || !d_y || !d_weights)) return fail(name + "null argument");
    if ((rows > 1 && ld_d < width) || ((int64_t)rows * k > 1 && (ld_y < width || ld_dy < width))) return fail(name + "leading dimension too small");
    if (!aligned(d_out, size_of(type)) || !aligned(y, size_of(type)) || !aligned(d_y, size_of(type)) || !words(order, place, weights, d_weights))
      return fail(name + "addresses must be multiples of the elements' size");
    JoinArgs a{};
    a.x = y;
    a.d = d_out;
    a.out = d_y;
    a.ld_x = ld_y;
    a.ld_d = ld_d;
    a.ld_out = ld_dy;
    a.rows = rows;
    a.k = k;
    a.width = width;
    a.order = order;
    a.place = place;
    a.weights = weights;
    a.d_weights = d_weights;
    return run_on(ctx, who, rows > 0, launched<JoinArgs, launch_moe_combine_grad>, &a, type);
  });
}

int64_t spx_mx4_bytes(int rows, int cols) {
  if (rows < 1 || cols < 1 || cols > 1 << 20) return 0;
  return (int64_t)rows * (mx4_padded(cols) / 32 * 17);
}

int spx_mx4_quantize(spx_ctx *ctx, int type, const void *x, int64_t ld_x, const spx_mx4 *m) {
  return entry([&] {
    const char *who = "spx_mx4_quantize";
    const std::string name = std::string(who) + ": ";
    if (const char *e = mx4_error(m)) return fail(name + e);
    if (!row_type(type)) return fail(name + "type must be SPX_F32, SPX_F16 or SPX_BF16");
    if (!x) return fail(name + "null argument");
    if (m->rows > 1 && ld_x < m->cols) return fail(name + "leading dimension too small");
    if (!aligned(x, size_of(type))) return fail(name + "addresses must be multiples of the elements' size");
    Mx4Rows a{mx4_parts(m->data, m->rows, m->cols), const_cast<void *>(x), ld_x, m->rows, m->cols, mx4_padded(m->cols) / MX4_STEP};
    return run_on(ctx, who, true, launched<Mx4Rows, launch_mx4_quantize>, &a, type);
  });
}

int spx_mx4_read(spx_ctx *ctx, const spx_mx4 *m, int type, void *out, int64_t ld_out) {
  return entry([&] {
    const char *who = "spx_mx4_read";
    const std::string name = std::string(who) + ": ";
    if (const char *e = mx4_error(m)) return fail(name + e);
    if (!row_type(type)) return fail(name + "type must be SPX_F32, SPX_F16 or SPX_BF16");
    if (!out) return fail(name + "null argument");
    if (m->rows > 1 && ld_out < m->cols) return fail(name + "leading dimension too small");
    if (!aligned(out, size_of(type))) return fail(name + "addresses must be multiples of the elements' size");
    Mx4Rows a{mx4_parts(m->data, m->rows, m->cols), out, ld_out, m->rows, m->cols, mx4_padded(m->cols) / MX4_STEP};
    return run_on(ctx, who, true, launched<Mx4Rows, launch_mx4_read>, &a, type);
  });
}

int spx_mx4_matmul(spx_ctx *ctx, int type, const void *x, int64_t ld_x, int x_rows, const spx_mx4 *w, const spx_mx4 *up, int n_expert,
                   const int32_t *starts, const int32_t *order, int k, int rows, int out_type, void *out, int64_t ld_out) {
  return entry([&] {
    const char *who = "spx_mx4_matmul";
    const std::string name = std::string(who) + ": ";
    if (const char *e = mx4_error(w)) return fail(name + e);
    if (up) {
      if (const char *e = mx4_error(up)) return fail(name + e);
      if (up->rows != w->rows || up->cols != w->cols) return fail(name + "w and up must have one shape");
    }
    if (!row_type(type) && type != SPX_MX4) return fail(name + "type must be SPX_F32, SPX_F16, SPX_BF16 or SPX_MX4");
    if (!row_type(out_type)) return fail(name + "out_type must be SPX_F32, SPX_F16 or SPX_BF16");
    if (n_expert < 1 || n_expert > MOE_MAX_E || w->rows % n_expert) return fail(name + "n_expert must be in 1..1024 and divide w's rows");
    if (!starts && (n_expert != 1 || order)) return fail(name + "n_expert above 1 and order need starts");
    if (w->rows / n_expert > 1 << 20) return fail(name + "a matrix of an expert has at most 2^20 rows");
    if (k < 1 || k > MOE_MAX_K) return fail(name + "k must be in 1..32");
    if (rows < 0 || rows > 1 << 23 || x_rows < 0 || x_rows > 1 << 23) return fail(name + "rows and x_rows must be in 0..2^23");
    if (!order && x_rows < rows) return fail(name + "x_rows must be at least rows where there is no order");
    const int n = w->rows / n_expert;
    if (rows > 0 && (!out || (x_rows > 0 && !x))) return fail(name + "null argument");
    if ((type != SPX_MX4 && x_rows > 1 && ld_x < w->cols) || (rows > 1 && ld_out < n)) return fail(name + "leading dimension too small");
    if (!aligned(x, type == SPX_MX4 ? 16 : size_of(type)) || !aligned(out, size_of(out_type)) || !words(starts, order))
      return fail(name + "a matrix's address must be a multiple of 16, the others of their elements' size");
    Mx4Product a{};
    a.x = x;
    if (type == SPX_MX4) a.x_scales = mx4_parts(const_cast<void *>(x), x_rows, w->cols).scales;
    a.ld_x = ld_x;
    a.ld_out = ld_out;
    a.x_rows = x_rows;
    a.cols = w->cols;
    a.steps = mx4_padded(w->cols) / MX4_STEP;
    a.n = n;
    a.n_expert = n_expert;
    a.k = k;
    a.rows = rows;
    a.w = mx4_parts(w->data, w->rows, w->cols);
    if (up) a.up = mx4_parts(up->data, up->rows, up->cols);
    a.starts = starts;
    a.order = order;
    a.out = out;
    struct Typed { const Mx4Product &a; int out_type; } t{a, out_type};
    const auto go = [](const void *p, int ty, hipStream_t s) { return launch_mx4_matmul(((const Typed *)p)->a, ty, ((const Typed *)p)->out_type, s); };
    return run_on(ctx, who, rows > 0 && x_rows > 0, go, &t, type);
  });
}

}  // extern "C"
