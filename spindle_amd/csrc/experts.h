// Operators of a mixture of experts over a batch: the router, sorting by expert, gathering and joining rows
// with their gradients (moe.hip), and matrices in microscaled 4-bit floats with their products (mx4.hip).
// Their C entries, with the checks of arguments, are in experts.cpp.
#pragma once
#include "../../include/spx.h"
#include "common.h"

namespace spx {

constexpr int MOE_MAX_E = 1024, MOE_MAX_K = 32, MOE_MAX_ROWS = 1 << 18;

struct RouteArgs {
  const void *logits;
  int64_t ld;
  int rows, n_expert, k, norm;
  int32_t *chosen;          // the gradient reads them
  float *weights;
  const float *d_weights;   // the gradient's
  void *d_logits;
  int64_t ld_d;
};
hipError_t launch_moe_route(const RouteArgs &a, int type, hipStream_t s);
hipError_t launch_moe_route_grad(const RouteArgs &a, int type, hipStream_t s);

struct SortArgs {
  int n, n_expert;  // entries
  const int32_t *chosen;
  int32_t *starts, *order, *place, *counts;  // counts: scratch [blocks][n_expert + 1]
};
int moe_sort_blocks(int64_t n);
hipError_t launch_moe_sort(const SortArgs &a, hipStream_t s);

struct JoinArgs {
  const void *x;    // gather: rows; combine: sorted rows
  const void *d;    // combine's gradient: d_out
  void *out;
  int64_t ld_x, ld_d, ld_out;
  int rows, k, width;
  const int32_t *order, *place;
  const float *weights;
  float *d_weights;
};
hipError_t launch_moe_gather(const JoinArgs &a, int type, hipStream_t s);
hipError_t launch_moe_combine(const JoinArgs &a, int type, hipStream_t s);
hipError_t launch_moe_combine_grad(const JoinArgs &a, int type, hipStream_t s);

// A matrix's parts: codes [rows][padded / 2], scale bytes [rows][padded / 32].
constexpr int MX4_STEP = 128;  // columns that rows are padded to
struct Mx4 {
  uint8_t *codes, *scales;
};
inline int mx4_padded(int cols) { return (cols + MX4_STEP - 1) / MX4_STEP * MX4_STEP; }
inline Mx4 mx4_parts(void *data, int64_t rows, int cols) { return {(uint8_t *)data, (uint8_t *)data + rows * (mx4_padded(cols) / 2)}; }

struct Mx4Rows {  // quantize: x is read; read: written
  Mx4 m;
  void *x;
  int64_t ld_x;
  int rows, cols, steps;  // steps: padded columns / 128
};
hipError_t launch_mx4_quantize(const Mx4Rows &a, int type, hipStream_t s);
hipError_t launch_mx4_read(const Mx4Rows &a, int type, hipStream_t s);

struct Mx4Product {
  const void *x;  // rows, or an SPX_MX4's codes
  const uint8_t *x_scales;
  int64_t ld_x, ld_out;
  int x_rows, cols, steps, n, n_expert, k, rows;
  Mx4 w, up;  // up.codes null: W x alone
  const int32_t *starts, *order;
  void *out;
};
hipError_t launch_mx4_matmul(const Mx4Product &a, int type, int out_type, hipStream_t s);

}  // namespace spx
