// Matrices in microscaled 4-bit floats: rows in (spx_mx4_quantize), values out (spx_mx4_read) and products
// (spx_mx4_matmul). include/spx.h states the format and its layout.
//
// The layout is the matrix cores': an instruction's 128 columns of a row are 64 bytes of codes and four scale
// bytes, of which lane group g of a wave takes the g-th 16 bytes and the g-th scale, one block of 32.
#include <atomic>
#include <type_traits>

#include "dev.h"
#include "experts.h"
#include "rows.h"

namespace spx {

typedef int i8v __attribute__((ext_vector_type(8)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------ rows in and out
// A thread has eight columns, the four threads of a quad a block, sixteen threads a step of 128 columns. Bound by their bytes: 8191
// rows of 2048 in bf16 9.1 us in and 9.6 us out (42 MB each), 16384 of 1024 in fp32 13 and 14.8 us (76 MB, from and to the
// last cache).
struct Eight {
  int row, c8;  // columns 8 c8 ..
};
__device__ __forceinline__ Eight eight_of(const Mx4Rows &a, int log_t, int &step) {
  step = 1 << log_t;
  return {(int)((blockIdx.x + blockIdx.y * gridDim.x) * (256 >> log_t) + (threadIdx.x >> log_t)), (int)(threadIdx.x & ((1 << log_t) - 1))};
}

// Magnitudes order as integers, NaN above all. With u the largest one's bits, floor(log2) - 2 + 127 is u >> 23 less
// 2, at least 0 (what is below the normal numbers included).
template <class R, bool VEC>
__global__ __launch_bounds__(256) void k_mx4_quantize(const Mx4Rows a, int log_t) {
  typedef typename R::E E;
  int step;
  const Eight p = eight_of(a, log_t, step);
  if ((uint32_t)p.row >= (uint32_t)a.rows) return;
  const E *src = (const E *)a.x + (int64_t)p.row * a.ld_x;
  for (int c = p.c8; c < a.steps * 16; c += step) {  // (threads of a step of columns stay together)
    float x[8];
    if (c * 8 + 8 <= a.cols) get8<R, VEC>(src + c * 8, x);
    else
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = c * 8 + j < a.cols ? row_get(R{}, src[c * 8 + j]) : 0.0f;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));
    const bool bad = m >= 0x7f800000u;
    const uint32_t e = m >> 23, byte = bad ? 255u : e > 2u ? e - 2u : 0u;
    uint32_t w = 0;
    if (!bad) {
      // the conversion rounds value / scale to nearest, ties to the even code, and takes the scale's exponent alone
      const float scale = __uint_as_float(byte << 23);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
    }
    *(uint32_t *)(a.m.codes + (int64_t)p.row * (a.steps * 64) + c * 4) = w;
    // a step's four scales as one word: each quad's byte at its place, joined across the sixteen lanes
    uint32_t s = byte << (8 * (c >> 2 & 3));
    s |= (uint32_t)__builtin_amdgcn_mov_dpp((int)s, 0x124, 0xF, 0xF, true);
    s |= (uint32_t)__builtin_amdgcn_mov_dpp((int)s, 0x128, 0xF, 0xF, true);
    if ((c & 15) == 0) *(uint32_t *)(a.m.scales + (int64_t)p.row * (a.steps * 4) + (c >> 2)) = s;
  }
}

template <class R, bool VEC>
__global__ __launch_bounds__(256) void k_mx4_read(const Mx4Rows a, int log_t) {
  typedef typename R::E E;
  int step;
  const Eight p = eight_of(a, log_t, step);
  if ((uint32_t)p.row >= (uint32_t)a.rows) return;
  E *dst = (E *)a.x + (int64_t)p.row * a.ld_x;
  for (int c = p.c8; c * 8 < a.cols; c += step) {
    const uint32_t w = *(const uint32_t *)(a.m.codes + (int64_t)p.row * (a.steps * 64) + c * 4);
    const float scale = __uint_as_float((uint32_t)a.m.scales[(int64_t)p.row * (a.steps * 4) + (c >> 2)] << 23);
    f2v v[4];
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    const float x[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
    if (c * 8 + 8 <= a.cols) put8<R, VEC>(dst + c * 8, x);
    else
      for (int j = 0; c * 8 + j < a.cols; j++) dst[c * 8 + j] = row_put(R{}, x[j]);
  }
}

// Whether rows at p, ld apart, lie at multiples of 16 bytes.
static bool on16(const void *p, int64_t ld, int64_t size) { return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0; }

template <class R>
static void rows_in_out(const Mx4Rows &a, bool in, hipStream_t s) {
  const bool vec = on16(a.x, a.ld_x, sizeof(typename R::E));
  int log_t = 4;
  while (log_t < 8 && (1 << log_t) < a.steps * 16) log_t++;
  const int each = 256 >> log_t;
  const int64_t blocks = ((int64_t)a.rows + each - 1) / each, wide = blocks < 1 << 20 ? blocks : 1 << 20;
  const dim3 grid((unsigned)wide, (unsigned)((blocks + wide - 1) / wide)), block(256);
  if (in) {
    if (vec) hipLaunchKernelGGL((k_mx4_quantize<R, true>), grid, block, 0, s, a, log_t);
    else hipLaunchKernelGGL((k_mx4_quantize<R, false>), grid, block, 0, s, a, log_t);
  } else {
    if (vec) hipLaunchKernelGGL((k_mx4_read<R, true>), grid, block, 0, s, a, log_t);
    else hipLaunchKernelGGL((k_mx4_read<R, false>), grid, block, 0, s, a, log_t);
  }
}
#define MX4_BY_TYPE(type, CALL)               \
  switch (type) {                             \
  case T_F32: { CALL(RowF32); break; }        \
  case T_F16: { CALL(RowF16); break; }        \
  case T_BF16: { CALL(RowBF16); break; }      \
  default: return hipErrorInvalidValue;       \
  }
hipError_t launch_mx4_quantize(const Mx4Rows &a, int type, hipStream_t s) {
#define CALL(R) rows_in_out<R>(a, true, s)
  MX4_BY_TYPE(type, CALL)
#undef CALL
  return hipGetLastError();
}
hipError_t launch_mx4_read(const Mx4Rows &a, int type, hipStream_t s) {
#define CALL(R) rows_in_out<R>(a, false, s)
  MX4_BY_TYPE(type, CALL)
#undef CALL
  return hipGetLastError();
}

// ------------------------------------------------------------------ products
// Kinds of x: 4-bit, or 16- and 32-bit rows as bf16 parts whose sum is the value (bf16 one, f16 two, fp32 three).
struct XMx4 { typedef RowF32 R; static constexpr int PARTS = 0; };
struct XBF16 { typedef RowBF16 R; static constexpr int PARTS = 1; };
struct XF16 { typedef RowF16 R; static constexpr int PARTS = 2; };
struct XF32 { typedef RowF32 R; static constexpr int PARTS = 3; };

// The rows of a tile: which expert's, where they start, how many (0: there is no such tile).
struct Tile { int expert, row, count; };
// The t-th tile of `most` rows: without starts of all rows, with them expert by expert (each one's last may be part
// filled). Every lane of a wave gets it.
__device__ __forceinline__ Tile tile_of(const Mx4Product &a, int t, int most) {
  if (!a.starts) {
    const int r = t * most;
    return {0, r, r < a.rows ? min(most, a.rows - r) : 0};
  }
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b = 0; b < a.n_expert; b += 64) {
    const int e = b + lane;
    int lo = 0, hi = 0;
    if (e < a.n_expert) {
      lo = min(max(a.starts[e], 0), a.rows);
      hi = min(max(a.starts[e + 1], lo), a.rows);
    }
    const int tiles = (hi - lo + most - 1) / most, upto = before + wave_scan(tiles);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(upto > t);
    if (past) {
      const int l = (int)__builtin_ctzll(past), r = lane_i(lo, l) + (t - (lane_i(upto, l) - lane_i(tiles, l))) * most;
      return {b + l, r, min(most, lane_i(hi, l) - r)};
    }
    before = lane_i(upto, 63);
  }
  return {0, 0, 0};
}
// Tiles of `most` rows that there may be.
static int64_t tiles_most(const Mx4Product &a, int most) {
  if (!a.starts) return ((int64_t)a.rows + most - 1) / most;
  const int64_t t = (int64_t)a.rows / most + a.n_expert;
  return t < a.rows ? t : a.rows;
}

// Row i's row of x, -1: none.
__device__ __forceinline__ int source_of(const Mx4Product &a, int i) {
  int r = i;
  if (a.order) {
    const int entry = a.order[i];
    r = entry >= 0 ? entry / a.k : -1;
  }
  return r < a.x_rows ? r : -1;
}

// A value as bf16 parts, each the upper half of what is left: 8 bits a part, and what is taken off is exact. An infinity
// or a NaN is its first part (rare: a way of its own, six instructions a value less).
template <int P>
__device__ __forceinline__ void parts_of(const float *x, b8v (&part)[P]) {
  uint32_t u[P][8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    float r = x[j];
#pragma unroll
    for (int p = 0; p < P; p++) {
      u[p][j] = __float_as_uint(r);
      r -= __uint_as_float(u[p][j] & 0xffff0000u);
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) most = max(most, u[0][j] & 0x7fffffffu);
  if (__builtin_expect(most >= 0x7f800000u, 0)) {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if ((u[0][j] & 0x7f800000u) == 0x7f800000u) {
        if (u[0][j] & 0x7fffffu) u[0][j] = 0x7fc00000u;  // (a NaN's upper half might be infinity's)
#pragma unroll
        for (int p = 1; p < P; p++) u[p][j] = 0;
      }
  }
#pragma unroll
  for (int p = 0; p < P; p++) {
    i4v w;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = (int)__builtin_amdgcn_perm(u[p][2 * j + 1], u[p][2 * j], 0x07060302u);
    part[p] = __builtin_bit_cast(b8v, w);
  }
}
// One of the parts: off1, off2 are the masks of what the first and the second leave to it (zero where it is no later one).
template <int P>
__device__ __forceinline__ b8v part_at(const float *x, uint32_t off1, uint32_t off2) {
  uint32_t u[8], most = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    float r = x[j] - __uint_as_float(__float_as_uint(x[j]) & off1);
    if (P > 2) r -= __uint_as_float(__float_as_uint(r) & off2);
    u[j] = __float_as_uint(r);
    most = max(most, __float_as_uint(x[j]) & 0x7fffffffu);
  }
  if (__builtin_expect(most >= 0x7f800000u, 0)) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t v = __float_as_uint(x[j]);
      if ((v & 0x7f800000u) == 0x7f800000u) u[j] = off1 ? 0u : v & 0x7fffffu ? 0x7fc00000u : v;
    }
  }
  i4v w;
#pragma unroll
  for (int j = 0; j < 4; j++) w[j] = (int)__builtin_amdgcn_perm(u[2 * j + 1], u[2 * j], 0x07060302u);
  return __builtin_bit_cast(b8v, w);
}
// Eight codes as values in bf16, which holds them exactly.
__device__ __forceinline__ b8v values_of(uint32_t w, float scale) {
  b2v v[4];
  v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
  v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
  v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  b8v r;
#pragma unroll
  for (int j = 0; j < 4; j++) { r[2 * j] = v[j][0]; r[2 * j + 1] = v[j][1]; }
  return r;
}
// BYTE: which byte of ws and xs is the scale.
template <int BYTE>
__device__ __forceinline__ f4v mfma_mx4(i4v w, int ws, i4v x, int xs, f4v acc) {
  const i8v A = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, B = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc, 4, 4, BYTE, ws, BYTE, xs);
}

typedef float f16v __attribute__((ext_vector_type(16)));
// 32 rows of the matrix against 32 of x, 64 columns: lane l has row l % 32 of either, block l / 32, and of the products
// those of row l % 32 of x with rows 8 (i / 4) + 4 (l / 32) + i % 4 of the matrix. (These run at 7.3 PFLOP/s here, those of
// 16 rows and 128 columns at 4.7 to 5.9; of the bf16 ones 32 x 32 x 16 at 2.1, 16 x 16 x 32 at 1.3 to 2.0.)
__device__ __forceinline__ f16v mfma_mx4_32(i4v w, int ws, i4v x, int xs, f16v acc) {
  const i8v A = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, B = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, acc, 4, 4, 0, ws, 0, xs);
}

// v over 1 + exp(-v), with the hardware's exponential and reciprocal, each good to a unit in the last place (a division and
// an exponential rounded correctly are forty instructions: a third of a gated tile's time). The exponential's argument h = -v log2(e) is
// rounded, which moves the exponential by up to |v| 2^-24. FINE: l is what that rounding took off, and the constant's own,
// and e (1 + l ln 2) has it back. Evaluated over -86..88 with both instructions exact, the result is then off by 4 * 2^-24 of itself at
// most; without, by 17 * 2^-24 at -20 and 65 * 2^-24 at -80. That is a hundredth of what rounding to f16 moves it and less of bf16's, so
// only fp32 outputs take the six instructions more (1% of an fp32 product by expert, 3 - 5% of a 16-bit one). Below -87, where the reciprocal leaves the
// normal numbers, a zero is as good: it is off by 87 * 2^-126 at most. (There e, and of infinities l, may be no number: e stays as it is.)
template <bool FINE>
__device__ __forceinline__ float silu(float v) {
  constexpr float L = 1.4426950408889634f, L2 = (float)(1.4426950408889634 - (double)L), LN2 = 0.6931471805599453f;
  const float h = v * -L;
  float e = __builtin_amdgcn_exp2f(h);
  if (FINE) {
    const float l = fmaf(v, -L2, fmaf(v, -L, -h));
    e = fabsf(v) < 88.0f ? fmaf(e, l * LN2, e) : e;
  }
  return v * __builtin_amdgcn_rcpf(1.0f + e);
}

struct Vecs { int x, out; };  // rows of x lie at multiples of 16 bytes, of out at multiples of four elements

// Four neighbours of a row of out. (The casts round to nearest even.)
template <class E>
__device__ __forceinline__ void put4(const Mx4Product &a, int i, int c, f4v v, bool vec) {
  E *dst = (E *)a.out + (int64_t)i * a.ld_out + c;
  alignas(16) const E e[4] = {(E)v[0], (E)v[1], (E)v[2], (E)v[3]};
  if (vec && c + 4 <= a.n) {
    if constexpr (sizeof(e) == 8) *(uint2 *)dst = *(const uint2 *)e;
    else *(uint4 *)dst = *(const uint4 *)e;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (c + j < a.n) dst[j] = e[j];
  }
}
__device__ __forceinline__ void put4_by(const Mx4Product &a, int out_type, int i, int c, f4v v, bool vec) {
  if (out_type == T_F32) put4<float>(a, i, c, v, vec);
  else if (out_type == T_F16) put4<_Float16>(a, i, c, v, vec);
  else put4<__bf16>(a, i, c, v, vec);
}

// Where a workgroup works. Tiles of one expert and row tile lie beside each other on one XCD (workgroups go to the eight in
// turn), so that its L2 gives the rows of x and the matrices again. False: there is no such tile.
__device__ __forceinline__ bool tile_place(const Mx4Product &a, int most, int columns, Tile &tile, int &column) {
  const int lane = threadIdx.x & 63;
  const uint64_t id = blockIdx.x + (uint64_t)blockIdx.y * gridDim.x;
  const auto at_of = [&](int tiles, int &t) {  // which of `tiles` tiles of rows is the workgroup's, and which column
    const uint64_t all = (uint64_t)tiles * columns, each = (all + 7) / 8, at = (id & 7) * each + (id >> 3);
    if ((id >> 3) >= each || at >= all) return false;
    t = (int)(all >> 32 ? at / columns : (uint32_t)at / (uint32_t)columns);  // (the wide division is slow)
    column = (int)(at - (uint64_t)t * columns);
    return true;
  };
  int t;
  if (!a.starts) {
    if (!at_of((a.rows + most - 1) / most, t)) return false;
    tile = tile_of(a, t, most);
    return true;
  }
  const auto experts = [&](int b, int &lo, int &tiles) {  // a lane's expert b + lane: its first row, its tiles
    const int e = b + lane;
    lo = 0;
    int hi = 0;
    if (e < a.n_expert) {
      lo = min(max(a.starts[e], 0), a.rows);
      hi = min(max(a.starts[e + 1], lo), a.rows);
    }
    tiles = (hi - lo + most - 1) / most;
    return hi;
  };
  if (a.n_expert > 256) {
    int all = 0;
    for (int b = 0; b < a.n_expert; b += 64) {
      int lo, tiles;
      experts(b, lo, tiles);
      all += lane_i(wave_scan(tiles), 63);
    }
    if (!at_of(all, t)) return false;
    tile = tile_of(a, t, most);
    return tile.count > 0;
  }
  int lo[4], hi[4], tiles[4], upto[4], all = 0;  // (all loads under way at once, each made once)
#pragma unroll
  for (int c = 0; c < 4; c++) hi[c] = experts(64 * c, lo[c], tiles[c]);
#pragma unroll
  for (int c = 0; c < 4; c++) {
    upto[c] = all + wave_scan(tiles[c]);
    all = lane_i(upto[c], 63);
  }
  if (!at_of(all, t)) return false;
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const unsigned long long past = __builtin_amdgcn_ballot_w64(upto[c] > t);
    if (past) {
      const int l = (int)__builtin_ctzll(past), r = lane_i(lo[c], l) + (t - (lane_i(upto[c], l) - lane_i(tiles[c], l))) * most;
      tile = {64 * c + l, r, min(most, lane_i(hi[c], l) - r)};
      return true;
    }
  }
  return false;
}

// ------------------------------------------------------------------ rows of x
// Eight columns of a row as they lie in memory, zeros behind the last and where there is no row.
template <class E>
struct Raw8 { uint4 v[sizeof(E) / 2]; };
template <class E>
__device__ __forceinline__ Raw8<E> raw8(const Mx4Product &a, const E *row, int c, bool vec) {
  Raw8<E> r;
  if (row && vec && c + 8 <= a.cols) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; i++) r.v[i] = ((const uint4 *)(row + c))[i];
  } else {
    alignas(16) E e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = row && c + j < a.cols ? row[c + j] : (E)0;
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; i++) r.v[i] = ((const uint4 *)e)[i];
  }
  return r;
}

// The same where rows lie at multiples of 16 bytes and cols is a multiple of 8: no branch, so that a thread's loads go out
// together (`row` is some row of x where there is none: its products are not stored).
template <class E>
__device__ __forceinline__ Raw8<E> raw8_whole(const Mx4Product &a, const E *row, int c) {
  Raw8<E> r;
  const uint4 *const from = (const uint4 *)(row + min(c, a.cols - 8));
#pragma unroll
  for (int i = 0; i < (int)sizeof(E) / 2; i++) r.v[i] = from[i];
  if (c >= a.cols)
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; i++) r.v[i] = make_uint4(0, 0, 0, 0);
  return r;
}

// How rows of x come: copied to LDS as they lie (bf16, whole turns), loaded in whole pieces, or by elements where need be.
enum { X_COPIED, X_WHOLE, X_ANY };

// ------------------------------------------------------------------ products of many 4-bit rows
// MT rows of x against 64 WN rows of the matrix (gated: half of them up's), 256 columns a turn, four waves of MF * 32 rows of x
// and 64 of the matrix each. Codes and scales are copied to LDS without a register, the codes a turn ahead, the
// scales two turns at a time: 128 bytes of a row, a whole cache line, as neighbouring lanes' addresses. Measured on 24 KB a
// turn from the L2, in bytes a clock and CU: 57 so, 25 by half lines (the other half is fetched again the next time), 16
// where neighbouring lanes are in different rows, as they are when a wave loads its own rows into registers.
// In LDS a row's eight pieces of 16 bytes stand at piece ^ (row / 2 & 7), so that what sixteen lanes read at a time (0-3, 12-15
// and 20-27 of each half) lies in other banks.
// 4095 rows of 2048 columns to eight of 128 experts each, gated, 768 columns out: 108-116 us, 1.8 PFLOP/s; 4096 x 4096 to 4096 55 us,
// 2.5. Of a turn's 1900 clocks 1000 are the matrix instructions of the CU's two workgroups; the copies' way into LDS takes as
// long, and the clock falls to 1.5 - 1.6 GHz under the load. A workgroup's search and first copies (6000 clocks) and its way out
// (4000) are hidden by the other's turns in part.
template <int MT>
struct Four {
  static constexpr int WM = MT == 32 ? 1 : 2, WN = 4 / WM, MF = MT / 32 / WM, ROWS = WN * 64;
  struct Lds {
    uint8_t x[2][MT * 128], w[2][ROWS * 128];
    uint32_t scales[MT + ROWS][4];  // of x's rows, then the matrix's
  };
};
typedef __attribute__((address_space(3))) void *lds_ptr;
// A wave's copies from memory to LDS: 16 or 4 bytes a lane, one lane's behind the other's. The address is the same for all
// lanes but for `lane`, 32 bits.
__device__ __forceinline__ rsrc_t from_here(const void *base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)0xffffffffu, 0x00020000);
}
__device__ __forceinline__ void copy16_lds(rsrc_t base, uint32_t lane, int all, void *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_ptr)to, 16, (int)lane, all, 0, 0);
}
__device__ __forceinline__ void copy16_lds(const void *from, void *to) { __builtin_amdgcn_global_load_lds(from, (lds_ptr)to, 16, 0, 0); }
__device__ __forceinline__ void copy4_lds(rsrc_t base, uint32_t lane, int all, void *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_ptr)to, 4, (int)lane, all, 0, 0);
}
// Waits until the wave's copies, loads and LDS accesses are done, then for the workgroup's other waves. No access to
// memory moves across.
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);  // (vmcnt and lgkmcnt 0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 32 rows of COLS neighbouring columns of out from a wave's products (or the gated ones'), through LDS of its own: a lane has
// four neighbours of a row, 8 or 16 bytes, and stored so each store would touch 32 rows. row(r): row r's number, -1: it is not stored.
template <int COLS, bool FP32, class F, class G>
__device__ __forceinline__ void put_rows(const Mx4Product &a, int out_type, bool vec, uint8_t *lds, int c0, F row, G value) {
  const int lane = threadIdx.x & 63, m = lane & 31, g = lane >> 5;
  constexpr int size = FP32 ? 4 : 2, pitch = COLS * size + 16;
#pragma unroll
  for (int t = 0; t < COLS / 32; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f4v v = value(t, i);
      uint8_t *const to = lds + m * pitch + (32 * t + 8 * i + 4 * g) * size;
      if constexpr (FP32) *(f4v *)to = v;
      else if (out_type == T_F16) {
        alignas(8) const _Float16 e[4] = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        *(uint2 *)to = *(const uint2 *)e;
      } else {
        alignas(8) const __bf16 e[4] = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        *(uint2 *)to = *(const uint2 *)e;
      }
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  constexpr int pieces = COLS * size / 16, each = 16 / size;
  for (int p = lane; p < 32 * pieces; p += 64) {
    const int r = p / pieces, q = p & (pieces - 1), i = row(r), c = c0 + q * each;
    if (i < 0 || c >= a.n) continue;
    const uint4 v = *(const uint4 *)(lds + r * pitch + q * 16);
    uint8_t *const to = (uint8_t *)a.out + ((int64_t)i * a.ld_out + c) * size;
    if (vec && c + each <= a.n) *(uint4 *)to = v;
    else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (size == 4) {
          if (c + j < a.n) ((uint32_t *)to)[j] = w[j];
        } else {
          if (c + 2 * j < a.n) ((uint16_t *)to)[2 * j] = (uint16_t)w[j];
          if (c + 2 * j + 1 < a.n) ((uint16_t *)to)[2 * j + 1] = (uint16_t)(w[j] >> 16);
        }
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int MT, bool GATED>
__global__ __launch_bounds__(256, MT == 64 ? 3 : 2) void k_mx4_four(const Mx4Product a, const Vecs vec, int out_type, int columns) {
  typedef Four<MT> T;
  constexpr int MF = T::MF, WN = T::WN, COLS = GATED ? 32 : 64, WC = 2 * WN, XC = MT / 32;  // WC, XC: a wave's copies a turn
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int s_src[MT];
  typename T::Lds &b = *(typename T::Lds *)lds;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, m = lane & 31, g = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  Tile tile;
  int column;
  if (!tile_place(a, MT, columns, tile, column)) return;
  int src = -1;
  if (tid < MT && tid < tile.count) src = source_of(a, tile.row + tid);
  const int col0 = column * WN * COLS;
  // the matrix from the workgroup's first row on
  const int64_t row0 = (int64_t)tile.expert * a.n + col0;
  const rsrc_t wcodes = from_here(a.w.codes + row0 * (a.steps * 64)), wscales = from_here(a.w.scales + row0 * (a.steps * 4));
  const rsrc_t ucodes = GATED ? from_here(a.up.codes + row0 * (a.steps * 64)) : wcodes, uscales = GATED ? from_here(a.up.scales + row0 * (a.steps * 4)) : wscales;
  const rsrc_t xcodes = from_here(a.x), xscales = from_here(a.x_scales);
  // A wave copies 8 WC rows of the matrix from row `from` on, eight at a time; row r stands for wave column r / 64, its
  // (r % 64)-th, gated: of w the first half of these, of up the second.
  const int from = wave * (8 * WC), r8 = lane >> 3;
  uint32_t wrow[WC];  // rows times steps
#pragma unroll
  for (int j = 0; j < WC; j++) {
    const int r = from + 8 * j + r8;
    wrow[j] = (uint32_t)min((r >> 6) * COLS + (r & (COLS - 1)), a.n - 1 - col0) * (uint32_t)a.steps;
  }
  const auto is_up = [&](int j) { return GATED && (WC == 8 ? j >= 4 : (wave & 1) != 0); };
  // the piece of a row that a lane copies (the last turn may have half of a row: that twice, the second one unused)
  const auto piece = [&](int j, int s) {
    const int p = (lane & 7) ^ (((j & 1) << 2) | (lane >> 4));
    return (uint32_t)(s + 1 < a.steps ? p : p & 3) * 16u;
  };
  const auto bring_w = [&](int s, int at) {
#pragma unroll
    for (int j = 0; j < WC; j++) copy16_lds(is_up(j) ? ucodes : wcodes, wrow[j] * 64u + piece(j, s), s * 64, b.w[at] + (from + 8 * j) * 128);
  };
  bring_w(0, 0);
  if (tid < MT) s_src[tid] = src;
  __syncthreads();
  // ... and XC times eight rows of x (one that there is none for: some row, which is not stored)
  uint32_t xrow[XC];
#pragma unroll
  for (int j = 0; j < XC; j++) xrow[j] = (uint32_t)max(s_src[(wave * XC + j) * 8 + r8], 0) * (uint32_t)a.steps;
  const auto bring_x = [&](int s, int at) {
#pragma unroll
    for (int j = 0; j < XC; j++)
      if ((wave * XC + j) * 8 < tile.count) copy16_lds(xcodes, xrow[j] * 64u + piece(wave * XC + j, s), s * 64, b.x[at] + (wave * XC + j) * 1024);
  };
  // scales of steps s0 .. s0 + 3 (behind the last: the last again, which nothing uses), sixteen rows a copy
  const auto bring_scales = [&](int s0) {
    const int s = min(s0 + (lane & 3), a.steps - 1) * 4, r16 = lane >> 2;
#pragma unroll
    for (int j = 0; j < WC / 2; j++) {
      const int r = from + 16 * j + r16;
      const uint32_t row = (uint32_t)min((r >> 6) * COLS + (r & (COLS - 1)), a.n - 1 - col0) * (uint32_t)a.steps;
      copy4_lds(is_up(2 * j) ? uscales : wscales, row * 4u + s, 0, b.scales[MT + from + 16 * j]);
    }
    for (int j = wave; j < MT / 16; j += 4) copy4_lds(xscales, (uint32_t)max(s_src[j * 16 + r16], 0) * (uint32_t)a.steps * 4u + s, 0, b.scales[j * 16]);
  };
  bring_scales(0);
  bring_x(0, 0);
  f16v acc[MF][2] = {};
  i4v xsc[MF], wsc[2];  // a row's scales of four steps
  // LIVE: the wave's fragments of x that have rows (what the others hold is never stored)
  const auto turns = [&](auto live) {
    constexpr int LIVE = decltype(live)::value;
    for (int s4 = 0; s4 < a.steps; s4 += 4) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int s = s4 + 2 * i;
        if (s >= a.steps) break;
        // what this turn reads has been brought, by every wave, and the reads of the last one's buffers are done
        wait_and_meet();
        if (i == 0) {
#pragma unroll
          for (int f = 0; f < LIVE; f++) xsc[f] = *(const i4v *)b.scales[(wm * MF + f) * 32 + m];
#pragma unroll
          for (int t = 0; t < 2; t++) wsc[t] = *(const i4v *)b.scales[MT + wn * 64 + t * 32 + m];
        }
        if (i == 1 && s4 + 4 < a.steps) bring_scales(s4 + 4);
        if (s + 2 < a.steps) {
          bring_w(s + 2, i ^ 1);
          bring_x(s + 2, i ^ 1);
        }
        if (LIVE == 0) continue;
        const uint8_t *const x = b.x[i] + wm * MF * 4096 + m * 128, *const w = b.w[i] + wn * 8192 + m * 128;
#pragma unroll
        for (int h = 0; h < 4; h++) {  // blocks 2h and 2h + 1
          if (h == 2 && s + 1 >= a.steps) break;
          const int u = ((2 * h + g) ^ (m >> 1 & 7)) * 16, j = 2 * i + (h >> 1), shift = 16 * (h & 1) + 8 * g;
          i4v wv[2];
#pragma unroll
          for (int t = 0; t < 2; t++) wv[t] = *(const i4v *)(w + t * 4096 + u);
#pragma unroll
          for (int f = 0; f < LIVE; f++) {
            const i4v xv = *(const i4v *)(x + f * 4096 + u);
#pragma unroll
            for (int t = 0; t < 2; t++) acc[f][t] = mfma_mx4_32(wv[t], wsc[t][j] >> shift, xv, xsc[f][j] >> shift, acc[f][t]);
          }
        }
      }
    }
  };
  const int rows = tile.count - wm * MF * 32;
  if (MF == 2 && rows > 32) turns(std::integral_constant<int, MF>{});
  else if (rows > 0) turns(std::integral_constant<int, 1>{});
  else turns(std::integral_constant<int, 0>{});
  wait_and_meet();  // (all waves' reads of LDS are done)
  const auto out = [&](auto fp32) {
    constexpr bool FP32 = decltype(fp32)::value;
#pragma unroll
    for (int f = 0; f < MF; f++) {
      const int r0 = (wm * MF + f) * 32;
      if (r0 >= tile.count) break;
      put_rows<COLS, FP32>(a, out_type, vec.out, lds + wave * 9216, col0 + wn * COLS, [&](int r) { return s_src[r0 + r] < 0 ? -1 : tile.row + r0 + r; },
                           [&](int t, int i) {
                             f4v v;
#pragma unroll
                             for (int j = 0; j < 4; j++) v[j] = GATED ? silu<FP32>(acc[f][0][4 * i + j]) * acc[f][1][4 * i + j] : acc[f][t][4 * i + j];
                             return v;
                           });
    }
  };
  if (out_type == T_F32) out(std::true_type{});
  else out(std::false_type{});
}

// ------------------------------------------------------------------ products of many 16- and 32-bit rows
// The same with x as bf16 parts and the matrix's codes made values in registers, 64 columns a turn: lane half g has block g of
// either operand, eight columns an instruction. The codes come 256 columns at a time (whole cache lines), four turns;
// bf16 rows are copied to LDS as they lie where they can be, others go through registers, a turn ahead. 4095 rows of 4096 columns
// to 2048: bf16 63-68 us (1.0 PFLOP/s, a library product of bf16 matrices of 8192 reaches 1.2), fp16 153, fp32 224 (each product
// two and three times); 216 rows of 2048 columns to eight of 128 experts, gated: 60-61 us, 3.6 TB/s, fp16 93, fp32 110.
template <class X, int MT>
struct Wide {
  static constexpr int P = X::PARTS, WM = MT == 32 ? 1 : 2, WN = 4 / WM, MF = MT / 32 / WM, ROWS = WN * 64;
  static constexpr int BUFS = P == 1 || (P == 2 && MT == 64) ? 2 : 1;  // (two workgroups a CU)
  struct Lds {
    uint8_t x[BUFS][P][MT * 128], w[2][ROWS * 128];
    uint32_t scales[ROWS][4];
  };
};

template <class X, int MT, bool GATED, int WAY>
__global__ __launch_bounds__(256, 2) void k_mx4_wide(const Mx4Product a, const Vecs vec, int out_type, int columns) {
  typedef Wide<X, MT> T;
  typedef typename X::R::E E;
  constexpr int P = T::P, MF = T::MF, WN = T::WN, BUFS = T::BUFS, COLS = GATED ? 32 : 64, WC = 2 * WN, XC = MT / 32;  // WC, XC: a wave's copies
  constexpr bool COPY = WAY == X_COPIED;
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int s_src[MT];
  // 32 rows of fp32 leave no room for it: there lane m of each wave has row m's (20 rows of 2048 columns to 151936 87 us, with one
  // workgroup a CU 110; 216 rows to eight of 128 experts, gated, 111 and 148).
  constexpr bool IN_LANES = 2 * (sizeof(typename T::Lds) + sizeof(s_src)) > 163840;
  static_assert(2 * sizeof(typename T::Lds) <= 163840 && (!IN_LANES || MT == 32), "two workgroups a CU");
  typename T::Lds &b = *(typename T::Lds *)lds;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, m = lane & 31, g = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  Tile tile;
  int column;
  if (!tile_place(a, MT, columns, tile, column)) return;
  int my_src = -1;
  if (IN_LANES) my_src = m < tile.count ? source_of(a, tile.row + m) : -1;
  else if (tid < MT) s_src[tid] = tid < tile.count ? source_of(a, tile.row + tid) : -1;
  const auto src_of = [&](int r) {  // (every lane of the wave calls it)
    if constexpr (IN_LANES) return __shfl(my_src, r);
    else return s_src[r];
  };
  const int col0 = column * WN * COLS;
  const int64_t row0 = (int64_t)tile.expert * a.n + col0;
  const rsrc_t wcodes = from_here(a.w.codes + row0 * (a.steps * 64)), wscales = from_here(a.w.scales + row0 * (a.steps * 4));
  const rsrc_t ucodes = GATED ? from_here(a.up.codes + row0 * (a.steps * 64)) : wcodes, uscales = GATED ? from_here(a.up.scales + row0 * (a.steps * 4)) : wscales;
  const int from = wave * (8 * WC), r8 = lane >> 3;
  uint32_t wrow[WC];
#pragma unroll
  for (int j = 0; j < WC; j++) {
    const int r = from + 8 * j + r8;
    wrow[j] = (uint32_t)min((r >> 6) * COLS + (r & (COLS - 1)), a.n - 1 - col0) * (uint32_t)a.steps;
  }
  const auto is_up = [&](int j) { return GATED && (WC == 8 ? j >= 4 : (wave & 1) != 0); };
  const auto slot = [&](int j) { return (lane & 7) ^ (((j & 1) << 2) | (lane >> 4)); };  // the piece of a row that a lane copies
  const auto bring_w = [&](int s, int at) {
#pragma unroll
    for (int j = 0; j < WC; j++) {
      const int p = slot(j);
      copy16_lds(is_up(j) ? ucodes : wcodes, wrow[j] * 64u + (uint32_t)(s + 1 < a.steps ? p : p & 3) * 16u, s * 64, b.w[at] + (from + 8 * j) * 128);
    }
  };
  const auto bring_scales = [&](int s0) {
    const int s = min(s0 + (lane & 3), a.steps - 1) * 4, r16 = lane >> 2;
#pragma unroll
    for (int j = 0; j < WC / 2; j++) {
      const int r = from + 16 * j + r16;
      const uint32_t row = (uint32_t)min((r >> 6) * COLS + (r & (COLS - 1)), a.n - 1 - col0) * (uint32_t)a.steps;
      copy4_lds(is_up(2 * j) ? uscales : wscales, row * 4u + s, 0, b.scales[from + 16 * j]);
    }
  };
  bring_w(0, 0);
  bring_scales(0);
  __syncthreads();
  // rows of x: XC times eight of them a wave, a lane eight columns; there is none: some row, which is not stored, or zeros
  const E *xr[XC];
#pragma unroll
  for (int j = 0; j < XC; j++) {
    const int src = src_of((wave * XC + j) * 8 + r8);
    xr[j] = WAY != X_ANY || src >= 0 ? (const E *)a.x + (int64_t)max(src, 0) * a.ld_x : nullptr;
  }
  const auto copy_x = [&](int turn, int at) {
#pragma unroll
    for (int j = 0; j < XC; j++)
      if ((wave * XC + j) * 8 < tile.count)
        copy16_lds(xr[j] + turn * 64 + slot(wave * XC + j) * 8, b.x[at][0] + (wave * XC + j) * 1024);
  };
  Raw8<E> xw[COPY ? 1 : XC];
  const auto load_x = [&](int turn) {
#pragma unroll
    for (int j = 0; j < XC; j++) {
      if constexpr (WAY == X_ANY) xw[j] = raw8<E>(a, xr[j], turn * 64 + (lane & 7) * 8, vec.x);
      else xw[j] = raw8_whole<E>(a, xr[j], turn * 64 + (lane & 7) * 8);
    }
  };
  const auto put_x = [&](int at) {
#pragma unroll
    for (int j = 0; j < XC; j++) {
      uint8_t *const to = b.x[at][0] + (wave * XC + j) * 1024 + r8 * 128 + slot(wave * XC + j) * 16;
      if constexpr (P == 1) *(uint4 *)to = xw[j].v[0];
      else {
        alignas(16) E e[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; i++) ((uint4 *)e)[i] = xw[j].v[i];
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = row_get(typename X::R{}, e[i]);
        b8v part[P];
        parts_of(x, part);
#pragma unroll
        for (int p = 0; p < P; p++) *(b8v *)(to + p * MT * 128) = part[p];
      }
    }
  };
  const int turns = (a.cols + 63) / 64;
  if (COPY) copy_x(0, 0);
  else {
    load_x(0);
    if (BUFS == 2) {
      put_x(0);
      load_x(1);
    }
  }
  f16v acc[MF][2] = {};
  i4v wsc[2];  // a row's scales of four steps
  const auto all_turns = [&](auto live) {
    constexpr int LIVE = decltype(live)::value;
    for (int t4 = 0; t4 < turns; t4 += 4) {  // 256 columns of codes
      const int at = t4 >> 2 & 1;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int turn = t4 + i;
        if (turn >= turns) break;
        // what this turn reads has been brought, by every wave, and the reads of the last one's buffers are done
        wait_and_meet();
        if (i == 0 && at == 0) {
#pragma unroll
          for (int t = 0; t < 2; t++) wsc[t] = *(const i4v *)b.scales[wn * 64 + t * 32 + m];
        }
        if (i == 0 && t4 + 4 < turns) bring_w((t4 >> 1) + 2, at ^ 1);
        if (i == 1 && at == 0 && t4 + 8 < turns) bring_scales((t4 >> 1) + 4);
        const int xb = BUFS == 2 ? i & 1 : 0;
        if (COPY) {
          if (turn + 1 < turns) copy_x(turn + 1, xb ^ 1);
        } else if (BUFS == 2) {
          if (turn + 1 < turns) put_x(xb ^ 1);
          if (turn + 2 < turns) load_x(turn + 2);
        } else {
          put_x(0);
          __syncthreads();
          if (turn + 1 < turns) load_x(turn + 1);
        }
        if (LIVE == 0) continue;
        const uint8_t *const x = b.x[xb][0] + wm * MF * 4096 + m * 128, *const w = b.w[at] + wn * 8192 + m * 128 + ((2 * i + g) ^ (m >> 1 & 7)) * 16;
        const int shift = 16 * (i & 1) + 8 * g;
        i4v codes[2];
        float scale[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
          codes[t] = *(const i4v *)(w + t * 4096);
          const int two = at ? (i < 2 ? wsc[t][2] : wsc[t][3]) : (i < 2 ? wsc[t][0] : wsc[t][1]);
          scale[t] = __uint_as_float(((uint32_t)two >> shift & 255u) << 23);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          b8v v[2];
#pragma unroll
          for (int t = 0; t < 2; t++) v[t] = values_of((uint32_t)codes[t][j], scale[t]);
          const int u = ((4 * g + j) ^ (m >> 1 & 7)) * 16;
#pragma unroll
          for (int f = 0; f < LIVE; f++)
#pragma unroll
            for (int p = P - 1; p >= 0; p--) {
              const b8v xv = *(const b8v *)(x + p * MT * 128 + f * 4096 + u);
#pragma unroll
              for (int t = 0; t < 2; t++) acc[f][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[t], xv, acc[f][t], 0, 0, 0);
            }
        }
      }
    }
  };
  const int rows = tile.count - wm * MF * 32;
  if (MF == 2 && rows > 32) all_turns(std::integral_constant<int, MF>{});
  else if (rows > 0) all_turns(std::integral_constant<int, 1>{});
  else all_turns(std::integral_constant<int, 0>{});
  wait_and_meet();  // (all waves' reads of LDS are done)
  const auto out = [&](auto fp32) {
    constexpr bool FP32 = decltype(fp32)::value;
#pragma unroll
    for (int f = 0; f < MF; f++) {
      const int r0 = (wm * MF + f) * 32;
      if (r0 >= tile.count) break;
      put_rows<COLS, FP32>(a, out_type, vec.out, lds + wave * 9216, col0 + wn * COLS, [&](int r) { return src_of(r0 + r) < 0 ? -1 : tile.row + r0 + r; },
                           [&](int t, int i) {
                             f4v v;
#pragma unroll
                             for (int j = 0; j < 4; j++) v[j] = GATED ? silu<FP32>(acc[f][0][4 * i + j]) * acc[f][1][4 * i + j] : acc[f][t][4 * i + j];
                             return v;
                           });
    }
  };
  if (out_type == T_F32) out(std::true_type{});
  else out(std::false_type{});
}

// ------------------------------------------------------------------ products of few rows
// Sixteen rows of x against 16 RT rows of the matrix (gated: half of them up's): W X^T, a lane's four sums being four
// neighbours of one row of out. Bound by the matrix's bytes. The workgroup's eight waves take the steps of 256 columns in turn, each
// by itself: codes and scales are copied to LDS of the wave's own as whole cache lines (straight into registers neighbouring
// lanes would be in different rows, at a quarter of the rate), x goes into registers; while a wave waits, the sixteen of a CU
// have others at work. The sums meet at the end. 2048 columns to 151936: one row of fp32 43-45 us (165 MB, 3.8 TB/s), nine of bf16
// 40 us; without the conversions and products one row would take 37 us, without x and scales either 32.
constexpr int FEW_W = 8;
template <int RT>
struct FewLds {
  uint8_t codes[RT][16 * 128];
  uint32_t scales[RT][2][16];
};

template <class X, int RT, bool GATED, int WAY>
__global__ __launch_bounds__(FEW_W * 64, 4) void k_mx4_few(const Mx4Product a, const Vecs vec, int out_type) {
  constexpr int P = X::PARTS, COLS = GATED ? RT * 8 : RT * 16;  // COLS: out's columns
  typedef typename X::R R;
  typedef typename R::E E;
  __shared__ __align__(16) FewLds<RT> ring[FEW_W];
  static_assert(sizeof(ring) >= FEW_W * RT * 64 * sizeof(f4v), "the sums fit in its place");
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, m = lane & 15, g = lane >> 4;
  const Tile tile = tile_of(a, blockIdx.y + blockIdx.z * gridDim.y, 16);
  if (tile.count <= 0) return;
  // Few rows of several parts: the parts are columns of their own, one instruction for all; lane m has part m / rows of row m % rows.
  const bool apart = P > 1 && tile.count * P <= 16;
  const int part_of = apart ? m / tile.count : 0, r = apart ? m - part_of * tile.count : m;
  const int i = tile.row + r, src = r < tile.count && part_of < (P > 1 ? P : 1) ? source_of(a, i) : -1, n0 = blockIdx.x * COLS;
  FewLds<RT> &b = ring[wave];
  const int64_t row0 = (int64_t)tile.expert * a.n + n0;
  const rsrc_t wcodes = from_here(a.w.codes + row0 * (a.steps * 64)), wscales = from_here(a.w.scales + row0 * (a.steps * 4));
  const rsrc_t ucodes = GATED ? from_here(a.up.codes + row0 * (a.steps * 64)) : wcodes, uscales = GATED ? from_here(a.up.scales + row0 * (a.steps * 4)) : wscales;
  const auto row_of = [&](int t, int r) { return (uint32_t)min((GATED ? t % (RT / 2 < 1 ? 1 : RT / 2) : t) * 16 + r, a.n - 1 - n0) * (uint32_t)a.steps; };
  const auto is_up = [&](int t) { return GATED && t >= RT / 2; };
  const auto bring = [&](int s) {  // (the last step may have half of a row: that twice, the second one unused)
    const bool both = s + 1 < a.steps;
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int p = (lane & 7) ^ (((j & 1) << 2) | (lane >> 4));
        copy16_lds(is_up(t) ? ucodes : wcodes, row_of(t, j * 8 + (lane >> 3)) * 64u + (uint32_t)(both ? p : p & 3) * 16u, s * 64, b.codes[t] + j * 1024);
      }
      // (two steps' scales of sixteen rows: half of the lanes)
      if (lane < 32) copy4_lds(is_up(t) ? uscales : wscales, row_of(t, m) * 4u + (uint32_t)(min(s + (lane >> 4), a.steps - 1) * 4), 0, b.scales[t][0]);
    }
  };
  // x's eight columns of group g of each instruction: of 16-bit rows for the whole step, of 32-bit ones for half of it (registers
  // for sixteen waves a CU)
  constexpr int XN = P == 3 ? 4 : 8;
  Raw8<E> x[P == 0 ? 1 : XN];
  i4v xc[2];
  int xs[2];
  const E *const xrow = P > 0 && (src >= 0 || WAY == X_WHOLE) ? (const E *)a.x + (int64_t)max(src, 0) * a.ld_x : nullptr;
  const auto load_x = [&](int s, int h0) {
    if constexpr (P == 0) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int at = min(s + h, a.steps - 1);  // (behind the last: that again, unused)
        xc[h] = *(const i4v *)((const uint8_t *)a.x + (int64_t)max(src, 0) * (a.steps * 64) + at * 64 + g * 16);
        xs[h] = a.x_scales[(int64_t)max(src, 0) * (a.steps * 4) + at * 4 + g];
      }
    } else {
#pragma unroll
      for (int j = 0; j < XN; j++) {
        const int c = (s + h0 + (j >> 2)) * 128 + g * 32 + (j & 3) * 8;
        if constexpr (WAY == X_ANY) x[j] = raw8<E>(a, xrow, c, vec.x);
        else x[j] = raw8_whole<E>(a, xrow, c);
      }
    }
  };
  f4v acc[RT] = {};
  const uint32_t off1 = part_of >= 1 ? 0xffff0000u : 0u, off2 = part_of >= 2 ? 0xffff0000u : 0u;  // what a lane's part leaves out
  const auto steps = [&](auto how) {
    constexpr bool APART = decltype(how)::value;
    for (int s = wave * 2; s < a.steps; s += 2 * FEW_W) {
      bring(s);
      load_x(s, 0);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0f70);  // (vmcnt 0)
      asm volatile("" ::: "memory");
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (h && s + 1 >= a.steps) break;
        if (XN == 4 && h) load_x(s, 1);
        i4v w[RT];
        int ws[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) {
          w[t] = *(const i4v *)(b.codes[t] + m * 128 + ((4 * h + g) ^ (m >> 1 & 7)) * 16);
          ws[t] = ((const uint8_t *)&b.scales[t][h][m])[g];
        }
        if constexpr (P == 0) {
#pragma unroll
          for (int t = 0; t < RT; t++) acc[t] = mfma_mx4<0>(w[t], ws[t], xc[h], xs[h], acc[t]);
        } else {
#pragma unroll
          for (int c = 0; c < 4; c++) {
            constexpr int PP = APART ? 1 : P;
            b8v part[PP];
            if constexpr (P == 1) part[0] = __builtin_bit_cast(b8v, x[(XN == 4 ? 0 : h * 4) + c].v[0]);
            else {
              alignas(16) E e[8];
#pragma unroll
              for (int k = 0; k < (int)sizeof(E) / 2; k++) ((uint4 *)e)[k] = x[(XN == 4 ? 0 : h * 4) + c].v[k];
              float v[8];
#pragma unroll
              for (int k = 0; k < 8; k++) v[k] = row_get(R{}, e[k]);
              if constexpr (APART) part[0] = part_at<P>(v, off1, off2);
              else parts_of(v, part);
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
              const b8v v = values_of((uint32_t)w[t][c], __uint_as_float((uint32_t)ws[t] << 23));
#pragma unroll
              for (int p = PP - 1; p >= 0; p--) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, part[p], acc[t], 0, 0, 0);
            }
          }
        }
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xc07f);  // (lgkmcnt 0: the reads of what the next step is brought over)
    }
  };
  if constexpr (P > 1) {
    if (apart) steps(std::true_type{});
    else steps(std::false_type{});
  } else steps(std::false_type{});
  __syncthreads();
  f4v(*const sums)[RT][64] = (f4v(*)[RT][64])ring;
#pragma unroll
  for (int t = 0; t < RT; t++) sums[wave][t][lane] = acc[t];
  __syncthreads();
  if (src < 0 || part_of > 0) return;
  constexpr int OUT = GATED ? RT / 2 : RT;
  for (int t = wave; t < OUT; t += FEW_W) {
    const auto total = [&](int u) {
      f4v v = {};
      for (int p = apart ? P - 1 : 0; p >= 0; p--) {  // (the smallest parts first)
        const int l = lane + p * tile.count;
#pragma unroll
        for (int w = 0; w < FEW_W; w += 4) v += (sums[w][u][l] + sums[w + 1][u][l]) + (sums[w + 2][u][l] + sums[w + 3][u][l]);
      }
      return v;
    };
    f4v v = total(t);
    if (GATED) {
      const f4v u = total(t + OUT);
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = (out_type == T_F32 ? silu<true>(v[j]) : silu<false>(v[j])) * u[j];
    }
    if (n0 + 16 * t + 4 * g < a.n) put4_by(a, out_type, i, n0 + 16 * t + 4 * g, v, vec.out);
  }
}

// Tiles over the launch's second and third dimension.
static dim3 tile_grid(int64_t columns, int64_t tiles) {
  const int64_t y = tiles < 32768 ? tiles : 32768;
  return dim3((unsigned)columns, (unsigned)y, (unsigned)((tiles + y - 1) / y));
}

// The devices on which a kernel has been allowed more than 64 KB of LDS.
struct Allowed {
  std::atomic<uint64_t> set{0};
  hipError_t lds(const void *kernel, unsigned bytes) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess || bytes <= 65536 || (dev < 64 && (set.load() >> dev & 1))) return e;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess && dev < 64) set |= 1ull << dev;
    return e;
  }
};

template <class X, int MT>
static hipError_t tiled(const Mx4Product &a, const Vecs &x_vec, int out_type, hipStream_t s) {
  constexpr int ROWS = Four<MT>::ROWS;
  const int wide = a.up.codes ? ROWS / 2 : ROWS, columns = (a.n + wide - 1) / wide;
  const int64_t blocks = (tiles_most(a, MT) * columns + 7) / 8 * 8, x = blocks < 1 << 20 ? blocks : 1 << 20;
  const dim3 grid((unsigned)x, (unsigned)((blocks + x - 1) / x));
  const Vecs vec = {x_vec.x, on16(a.out, a.ld_out, out_type == T_F32 ? 4 : 2)};
  static Allowed allowed[4];
  const auto launch = [&](void (*k)(Mx4Product, Vecs, int, int), int which, unsigned bytes) {
    if (const hipError_t e = allowed[which].lds((const void *)k, bytes); e != hipSuccess) return e;
    hipLaunchKernelGGL(k, grid, dim3(256), bytes, s, a, vec, out_type, columns);
    return hipGetLastError();
  };
  if constexpr (X::PARTS == 0) {
    constexpr unsigned bytes = sizeof(typename Four<MT>::Lds);
    return a.up.codes ? launch(k_mx4_four<MT, true>, 0, bytes) : launch(k_mx4_four<MT, false>, 1, bytes);
  } else {
    constexpr unsigned bytes = sizeof(typename Wide<X, MT>::Lds);
    if constexpr (X::PARTS == 1)
      if (vec.x && a.cols % 64 == 0) return a.up.codes ? launch(k_mx4_wide<X, MT, true, X_COPIED>, 0, bytes) : launch(k_mx4_wide<X, MT, false, X_COPIED>, 1, bytes);
    if constexpr (X::PARTS > 1)
      if (vec.x && a.cols % 8 == 0) return a.up.codes ? launch(k_mx4_wide<X, MT, true, X_WHOLE>, 0, bytes) : launch(k_mx4_wide<X, MT, false, X_WHOLE>, 1, bytes);
    return a.up.codes ? launch(k_mx4_wide<X, MT, true, X_ANY>, 2, bytes) : launch(k_mx4_wide<X, MT, false, X_ANY>, 3, bytes);
  }
}

template <class X, int RT, bool GATED>
static hipError_t few(const Mx4Product &a, const Vecs &vec, int out_type, hipStream_t s) {
  constexpr int COLS = GATED ? RT * 8 : RT * 16;
  const dim3 grid = tile_grid((a.n + COLS - 1) / COLS, tiles_most(a, 16)), block(FEW_W * 64);
  if (X::PARTS == 0 || (vec.x && a.cols % 8 == 0)) hipLaunchKernelGGL((k_mx4_few<X, RT, GATED, X_WHOLE>), grid, block, 0, s, a, vec, out_type);
  else if constexpr (X::PARTS > 0) hipLaunchKernelGGL((k_mx4_few<X, RT, GATED, X_ANY>), grid, block, 0, s, a, vec, out_type);
  return hipGetLastError();
}

// Which kernel: by the rows that a matrix has on average and by the workgroups that there would be. Dense products in us, from
// a captured graph (rows of bf16, unless said otherwise; few / tiles of 64 rows):
//   2048 columns, 4096 rows of the matrix: 16 rows 4.6 / 13, 128 rows 9.4 / 15, 256 rows 15.8 / 17.7, 384 rows 22.5 / 19
//   4096 columns, 2048:                    64 rows 9.0 / 25, 256 rows 16 / 30, 384 rows 22.5 / 31
//   1024 columns, 1024:                    64 rows 3.7 / 8.9, 384 rows 6.4 / 9.1
//   2048 columns, 4096, fp32 rows:         128 rows 15 / 42, 384 rows 38 / 50
//   2048 columns, 4096, 4-bit rows:        64 rows 5.0 / 6.4, 128 rows 7.3 / 6.6, 256 rows 11.7 / 8.6
//   2048 columns, 151936, 9 rows:          40 / 49 (tiles of 32)
// so the few rows' kernel has up to 16 rows, and more where the tiles would leave CUs idle: up to 128 tiles, 192 of fp32 rows,
// 48 of 4-bit ones. By expert, 24 rows of 2048 to 8 of 128 experts take it 40 us (1.5 rows each), 216 rows 70 and in tiles of 32
// 61 (13.5 each). Tiles of 64 and 128 rows: 4095 rows of 4096 columns 81 and 70, 512 rows of 2048 columns 21 and 24, 250 rows
// each of 32 experts of 1024 columns 28 and 33; of 4-bit rows 4095 x 4096 35 and 28, 256 rows each of 128 experts 124 and 115.
template <class X>
static hipError_t product(const Mx4Product &a, int out_type, hipStream_t s) {
  constexpr int P = X::PARTS;
  const Vecs vec = {P == 0 || on16(a.x, a.ld_x, sizeof(typename X::R::E)), (uintptr_t)a.out % (out_type == T_F32 ? 16 : 8) == 0 && a.ld_out % 4 == 0};
  const bool gated = a.up.codes != nullptr;
  const int64_t each = a.starts ? a.rows / a.n_expert : a.rows;
  const int64_t tiles64 = tiles_most(a, 64) * ((a.n + (gated ? 63 : 127)) / (gated ? 64 : 128));
  const bool far = P == 0 && (int64_t)a.x_rows * a.steps * 64 > UINT32_MAX;  // (the tiles' addresses of 4-bit rows have 32 bits)
  if (far || each <= (a.starts ? 8 : 16) || tiles64 <= (P == 0 ? 48 : P == 3 ? 192 : 128)) {
    // rows of the matrix a workgroup: 64 where that makes half a workgroup a CU, else 16 (gated 32): 64 rows of 2048 columns to
    // 4096 6.3 and 10.8 us, 9 rows 5.6 and 4.1
    const bool many = tiles_most(a, 16) * ((a.n + 63) / 64) >= 128;
    if (gated) return many ? few<X, 4, true>(a, vec, out_type, s) : few<X, 2, true>(a, vec, out_type, s);
    return many ? few<X, 4, false>(a, vec, out_type, s) : few<X, 1, false>(a, vec, out_type, s);
  }
  if (each <= 24) return tiled<X, 32>(a, vec, out_type, s);
  if constexpr (P < 3)  // (fp32 parts of 128 rows leave LDS for one workgroup a CU: 4095 rows of 4096 columns 254 us instead of 218)
    if (each > (P == 0 ? 64 : 512)) return tiled<X, 128>(a, vec, out_type, s);
  return tiled<X, 64>(a, vec, out_type, s);
}
hipError_t launch_mx4_matmul(const Mx4Product &a, int type, int out_type, hipStream_t s) {
  switch (type) {
  case SPX_MX4: return product<XMx4>(a, out_type, s);
  case T_F32: return product<XF32>(a, out_type, s);
  case T_F16: return product<XF16>(a, out_type, s);
  case T_BF16: return product<XBF16>(a, out_type, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace spx
