// The paged 4-bit key / value cache: rows in (spx_kv4_append), values out (spx_kv4_read) and
// attention over it (spx_kv4_attention). include/spx.h states the format and the pool's layout.
//
// The layout is the matrix cores': a tile of 16 tokens of one head is one contiguous run of
// 18 * head_dim bytes, in which each lane of a wave finds the codes that it feeds to the matrix
// instructions in one load. Scales have 8 significant bits, so integer * scale (at most 3 + 8
// bits, or 8 times the scale) is exact in f16 and the matrix cores read the values themselves.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "batch.h"
#include "dev.h"
#include "kv4_order.h"

namespace spx {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));

constexpr float KV4_DMAX = 8160.0f;  // 8 * d stays finite in f16

// ------------------------------------------------------------------ 16-bit and 32-bit rows
struct RowF32 { typedef float E; };
struct RowF16 { typedef _Float16 E; };
struct RowBF16 { typedef uint16_t E; };

__device__ __forceinline__ float row_get(RowF32, float v) { return v; }
__device__ __forceinline__ float row_get(RowF16, _Float16 v) { return (float)v; }
__device__ __forceinline__ float row_get(RowBF16, uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float row_put(RowF32, float v) { return v; }
__device__ __forceinline__ _Float16 row_put(RowF16, float v) { return (_Float16)v; }
__device__ __forceinline__ uint16_t bf16_rne(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 64);  // NaN stays one
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
__device__ __forceinline__ uint16_t row_put(RowBF16, float v) { return bf16_rne(v); }

// ------------------------------------------------------------------ places in the pool
// Byte offset of the tile of token `t` of page `pg` (page: log2 of a page's tokens).
template <int HD>
__device__ __forceinline__ int64_t tile_at(int pg, int n_kv, int head, int page, int t) {
  return ((((int64_t)pg * n_kv + head) << (page - 4)) + (t >> 4)) * (18 * HD);
}
// Slot -> page and place in it; false for a slot outside the pool.
__device__ __forceinline__ bool slot_of(int slot, int page, int n_pages, int &pg, int &t) {
  pg = slot >> page;
  t = slot & ((1 << page) - 1);
  return slot >= 0 && pg < n_pages;
}

// A thread's piece of a row: eight channels of the key (kv = 0) or the value (1) of one head. Rows run
// fastest above the pieces of a row, so that a wave fills whole cache lines of a tile. (Four rows a
// thread, all loads under way at once, gain nothing: 8191 rows of 8 heads of 128 take 20 instead of 18
// us to write, 11.4 instead of 12.0 to read.)
template <int HD>
struct Piece {
  int row, head, kv, c8;  // c8: channels 8 c8 ..
};
template <int HD>
__device__ __forceinline__ Piece<HD> piece_of() {
  constexpr int PC = HD / 8;
  return {(int)(blockIdx.x * (256 / PC) + threadIdx.x / PC), (int)(blockIdx.y >> 1), (int)(blockIdx.y & 1), (int)(threadIdx.x % PC)};
}
// Eight values of a row. VEC: rows lie at multiples of 16 bytes.
template <class R, bool VEC>
__device__ __forceinline__ void get8(const typename R::E *src, float *x) {
  alignas(16) typename R::E e[8];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; i++) ((uint4 *)e)[i] = ((const uint4 *)src)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = src[j];
  }
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = row_get(R{}, e[j]);
}
template <class R, bool VEC>
__device__ __forceinline__ void put8(typename R::E *dst, const float *x) {
  alignas(16) typename R::E e[8];
#pragma unroll
  for (int j = 0; j < 8; j++) e[j] = row_put(R{}, x[j]);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; i++) ((uint4 *)dst)[i] = ((const uint4 *)e)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) dst[j] = e[j];
  }
}

// The same by a flag that is one for the launch; N values out.
template <class R>
__device__ __forceinline__ void get8_if(bool vec, const typename R::E *src, float *x) {
  if (vec) get8<R, true>(src, x);
  else get8<R, false>(src, x);
}
template <class R, int N>
__device__ __forceinline__ void put_if(bool vec, typename R::E *dst, const float *x) {
  typedef typename R::E E;
  alignas(16) E e[N];
#pragma unroll
  for (int i = 0; i < N; i++) e[i] = row_put(R{}, x[i]);
  if (vec) {
    if constexpr (sizeof(e) == 8) *(uint2 *)dst = *(const uint2 *)e;
    else
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; i++) ((uint4 *)dst)[i] = ((const uint4 *)e)[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) dst[i] = e[i];
  }
}

// ------------------------------------------------------------------ append
// The integer nearest to x / d, half to even, exactly: the quotient's estimate is off by at most
// one, and x - c d is exact (c d has at most 12 bits and is within a factor of two of x, or zero).
__device__ __forceinline__ float kv4_code_exact(float x, float d, float inv) {
  float c = rintf(x * inv);
  c = fminf(fmaxf(c, -9.0f), 9.0f);
  const float e = fmaf(-c, d, x) * (d < 0.0f ? -1.0f : 1.0f), h = 0.5f * fabsf(d);  // e: the rest, in d's direction
  const bool odd = ((int)c & 1) != 0;
  if (e > h || (e == h && odd)) c += 1.0f;
  else if (e < -h || (e == -h && odd)) c -= 1.0f;
  return c;
}
// Eight of them. x * inv is within 1.5e-6 of the quotient (at most 12, two roundings), so that only
// where one lies that near to a half is more than its rounding needed.
__device__ __forceinline__ void kv4_codes(const float *x, float d, float inv, uint32_t *c) {
  float f[8], off = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float y = x[j] * inv;
    f[j] = rintf(y);
    off = fmaxf(off, fabsf(y - f[j]));
  }
  if (off > 0.49999f)
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = kv4_code_exact(x[j], d, inv);
#pragma unroll
  for (int j = 0; j < 8; j++) c[j] = (uint32_t)(fminf(fmaxf(f[j], -8.0f), 7.0f) + 8.0f);
}

// A thread quantizes eight channels; the four threads of a quad share a group's scale. 8191 rows of 8
// heads of 128 (bf16, 43 MB in and out) take 18 us, where bytes alone would take 8: what bounds it are
// its narrow stores, a word of codes a thread and two bytes of scale a quad; 24 rows of four heads 3.5 us.
template <int HD>
__device__ __forceinline__ void append_piece(const Kv4Rows &a, float *x, int kv, int head, int c8, int slot) {
  int pg, t;
  const bool is = slot_of(slot, a.page, a.n_pages, pg, t);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);  // magnitudes order as integers, NaN above all
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));
  // the first value of that magnitude gives the sign: place << 1 | negative, the smallest of all
  uint32_t key = ~0u;
#pragma unroll
  for (int j = 7; j >= 0; j--)
    if ((__float_as_uint(x[j]) & 0x7fffffffu) == m) key = (uint32_t)(((c8 & 3) * 8 + j) << 1) | (__float_as_uint(x[j]) >> 31);
  key = min(key, (uint32_t)__builtin_amdgcn_mov_dpp((int)key, 0xB1, 0xF, 0xF, true));
  key = min(key, (uint32_t)__builtin_amdgcn_mov_dpp((int)key, 0x4E, 0xF, 0xF, true));
  if (!is) return;
  const bool bad = m >= 0x7f800000u;
  const float most = __uint_as_float(m | (key << 31));
  float d = row_get(RowBF16{}, bf16_rne(most * -0.125f));
  d = (float)(_Float16)fminf(fmaxf(d, -KV4_DMAX), KV4_DMAX) + 0.0f;  // (a scale of zero is +0)
  const float inv = d == 0.0f ? 0.0f : 1.0f / d;
  uint32_t c[8];
  if (bad) {  // (codes of a NaN group are 0)
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = 0.0f;
  }
  kv4_codes(x, d, inv, c);  // (a scale of zero has inv = 0: codes 0)
  const _Float16 dh = bad ? (_Float16)__builtin_nanf("") : (_Float16)d;
  constexpr int G = HD / 32;
  uint8_t *tile = a.pool + tile_at<HD>(pg, a.n_kv, head, a.page, t);
  const int ti = t & 15, g = c8 >> 2, h = c8 & 3;
  if (!kv) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) w |= c[j] << (4 * ((j >> 1) + 4 * (j & 1)));
    *(uint32_t *)(tile + ((h * 16 + ti) * G + g) * 4) = w;
    if (h == 0) *(_Float16 *)(tile + 16 * HD + (ti * G + g) * 2) = dh;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) w |= c[j] << (4 * j);
    uint8_t *vc = tile + 8 * HD + (ti >> 2) * 64 * G + (ti & 3) * G;
    if (HD == 128) {
      *(uint32_t *)(vc + c8 * 16) = w;
    } else {  // a lane of the attention kernels has four channels: two lanes' halves
      *(uint16_t *)(vc + (2 * c8) * 8) = (uint16_t)w;
      *(uint16_t *)(vc + (2 * c8 + 1) * 8) = (uint16_t)(w >> 16);
    }
    if (h == 0) *(_Float16 *)(tile + 17 * HD + (g * 16 + ti) * 2) = dh;
  }
}
template <int HD, class R, bool VEC>
__global__ __launch_bounds__(256) void k_kv4_append(const Kv4Rows a) {
  typedef typename R::E E;
  const Piece<HD> p = piece_of<HD>();
  if (p.row >= a.rows) return;  // (a quad has one row)
  const E *base = (p.kv ? (const E *)a.v : (const E *)a.k) + p.head * HD + p.c8 * 8;
  float x[8];
  get8<R, VEC>(base + p.row * (p.kv ? a.ld_v : a.ld_k), x);
  append_piece<HD>(a, x, p.kv, p.head, p.c8, a.slots[p.row]);
}

// ------------------------------------------------------------------ read
// The other way round: a word of codes and a scale in, 16 or 32 bytes out; 12 and 2.5 us for the same.
template <int HD, class R, bool VEC>
__global__ __launch_bounds__(256) void k_kv4_read(const Kv4Rows a) {
  typedef typename R::E E;
  constexpr int G = HD / 32;
  const Piece<HD> p = piece_of<HD>();
  if (p.row >= a.rows) return;
  E *base = (p.kv ? (E *)a.v : (E *)a.k) + p.head * HD + p.c8 * 8;
  float x[8] = {};
  int pg, t;
  if (slot_of(a.slots[p.row], a.page, a.n_pages, pg, t)) {
    const uint8_t *tile = a.pool + tile_at<HD>(pg, a.n_kv, p.head, a.page, t);
    const int ti = t & 15, g = p.c8 >> 2, h = p.c8 & 3;
    uint32_t w;
    float d;
    if (!p.kv) {
      w = *(const uint32_t *)(tile + ((h * 16 + ti) * G + g) * 4);
      d = (float)*(const _Float16 *)(tile + 16 * HD + (ti * G + g) * 2);
    } else {
      const uint8_t *vc = tile + 8 * HD + (ti >> 2) * 64 * G + (ti & 3) * G;
      if (HD == 128) w = *(const uint32_t *)(vc + p.c8 * 16);
      else w = *(const uint16_t *)(vc + (2 * p.c8) * 8) | (uint32_t) * (const uint16_t *)(vc + (2 * p.c8 + 1) * 8) << 16;
      d = (float)*(const _Float16 *)(tile + 17 * HD + (g * 16 + ti) * 2);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int nib = p.kv ? j : (j >> 1) + 4 * (j & 1);
      x[j] = (float)((int)((w >> (4 * nib)) & 15) - 8) * d;
    }
  }
  put8<R, VEC>(base + p.row * (p.kv ? a.ld_v : a.ld_k), x);
}

#define KV4_BY_TYPE(hd, type, CALL)                                                 \
  switch ((hd) * 64 + (type)) {                                                     \
  case 64 * 64 + T_F32: { CALL(64, RowF32); break; }                                \
  case 64 * 64 + T_F16: { CALL(64, RowF16); break; }                                \
  case 64 * 64 + T_BF16: { CALL(64, RowBF16); break; }                              \
  case 128 * 64 + T_F32: { CALL(128, RowF32); break; }                              \
  case 128 * 64 + T_F16: { CALL(128, RowF16); break; }                              \
  case 128 * 64 + T_BF16: { CALL(128, RowBF16); break; }                            \
  default: return hipErrorInvalidValue;                                             \
  }

static bool rows_aligned(const Kv4Rows &a, int size) {
  return (uintptr_t)a.k % 16 == 0 && (uintptr_t)a.v % 16 == 0 && a.ld_k * size % 16 == 0 && a.ld_v * size % 16 == 0;
}
static dim3 rows_grid(const Kv4Rows &a, int hd) { return dim3((unsigned)(((int64_t)a.rows * (hd / 8) + 255) / 256), 2u * a.n_kv); }

hipError_t launch_kv4_append(const Kv4Rows &a, int hd, int type, hipStream_t s) {
#define CALL(H, R)                                                  \
  if (rows_aligned(a, sizeof(R::E))) hipLaunchKernelGGL((k_kv4_append<H, R, true>), rows_grid(a, H), dim3(256), 0, s, a); \
  else hipLaunchKernelGGL((k_kv4_append<H, R, false>), rows_grid(a, H), dim3(256), 0, s, a)
  KV4_BY_TYPE(hd, type, CALL)
#undef CALL
  return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4Rows &a, int hd, int type, hipStream_t s) {
#define CALL(H, R)                                                \
  if (rows_aligned(a, sizeof(R::E))) hipLaunchKernelGGL((k_kv4_read<H, R, true>), rows_grid(a, H), dim3(256), 0, s, a); \
  else hipLaunchKernelGGL((k_kv4_read<H, R, false>), rows_grid(a, H), dim3(256), 0, s, a)
  KV4_BY_TYPE(hd, type, CALL)
#undef CALL
  return hipGetLastError();
}

// ------------------------------------------------------------------ attention
// The query heads of a key head and a sequence's new tokens together are rows that read the same
// keys and values: row r is token r / group, head r % group of the group. A workgroup takes 16 rows
// of one sequence and key head; its four waves take turns over the sequence's tokens, 32 at a time.
//
// S^T = K Q^T on v_mfma_f32_16x16x32_f16: a lane's column is its query row (lane % 16), its four
// rows are tokens, so a row's maximum and sum lie in four lanes and the probabilities are, as they
// come, the right operand of O^T = V^T P^T: lane l of 16 and quarter h holds tokens 4h .. 4h + 3 of
// each of the two tiles there.
//
// What bounds the kernel is the vector instructions that turn codes into operands. Key codes go in as
// they are: a nibble masked in place is a subnormal f16 (code * 2^-24, or 2^-20 from the high nibble
// of a byte, which the query makes up for), which the matrix cores multiply exactly, so a word of
// eight codes costs five instructions; a group's sum starts at -8 times the query's and is scaled
// afterwards, with one multiply-add a token, row and group. That start is several times what is left of
// the sum: harmless beside 16-bit rows, but SPX_F32 rows came out 6.5e-6 off instead of 3e-7, so theirs
// meet the integers -8 .. 7, at four more instructions a word. Values become integer * scale in f16
// (exact): their scale belongs to the token, which the sum runs over. 64 sequences of up to 16K tokens
// (32 heads over 4 of 128) read 382 MB in 93 us, 4.1 TB/s, where a copy reaches 5.1. By the counters the
// vector units are busy 71% of the time in which a CU has waves (2.6 a SIMD on average, which spend 43% of
// theirs at waits), and a CU has none for a quarter of the kernel's time. Loads of the next
// tiles issued before this one's work (209 registers, two waves a SIMD) gained nothing, nor did fewer
// registers with spills.
//
// A query row is scaled by a power of two to fill f16's range; in two parts (SPX_F32) it has 22 bits.
// Probabilities are held relative to a running maximum, times 2^10, so that small ones keep their
// bits in f16; a maximum that grows by less than 5 (a factor of 2^5) leaves the reference as it is.
// They are made in 32 bits and enter the second product in f16: in two parts (SPX_F32, SPX_F16), 22 bits,
// because one part's rounding (2^-11) would add to the output's own in SPX_F16; in one part, 11 bits, for
// SPX_BF16, where it is an eighth of the output's (2048 rows at 4096 tokens: 1.67e-3 off in norm with it,
// 1.66e-3 by the output's rounding alone). Their sum is of the unrounded ones here, of the rounded ones
// where k_kv4_rows has one part.
//
// The reference is kept in the units of the sums, unscaled: a probability's exponent is one multiply-add
// s * unlift + (10 - m * unlift), whose last term is rounded. Where that is past 2^12 (P_FAR) the sums have
// the reference taken off first: at 2^30 the rounding would be more than f16's whole range.
constexpr float P_LIFT = 10.0f, P_SLACK = 5.0f, P_FAR = 4096.0f;
// What the exponents add to s * unlift, for a reference of top = m * unlift (0 where no token has been seen).
__device__ __forceinline__ bool p_far(float top) { return fabsf(top) > P_FAR && top != -__builtin_inff(); }
__device__ __forceinline__ float p_ref(float top) { return top == -__builtin_inff() ? 0.0f : p_far(top) ? P_LIFT : P_LIFT - top; }

// The sequence and first row of job `job`: sequence s has jobs floor(start_s * group / BM) + s and
// on, enough for its rows whatever their number, and f ascends, so that one pass over q_start in
// parallel finds it. False when the job has no rows.
struct Job4 { int s, q0, nq, r0, n; };
template <int BM>
__device__ __forceinline__ bool job_of(const Kv4Attn &a, int job, Job4 &j) {
  const int lane = threadIdx.x & 63;
  int cnt = 0;
  for (int b = 0; b < a.n_seq; b += 64) {
    const int s = b + lane;
    const bool le = s < a.n_seq && (int)(((int64_t)min(max(a.q_start[s], 0), a.rows) * a.group) / BM) + s <= job;
    cnt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(le));
  }
  const int s = __builtin_amdgcn_readfirstlane(max(cnt - 1, 0));
  const int q0 = min(max(a.q_start[s], 0), a.rows), q1 = min(max(a.q_start[s + 1], 0), a.rows);
  j.s = s;
  j.q0 = q0;
  j.nq = q1 - q0;
  j.r0 = (job - ((int)((int64_t)q0 * a.group / BM) + s)) * BM;
  j.n = (int)min((int64_t)max(a.kv_lens[s], 0), (int64_t)a.cols << a.page);
  return j.nq > 0 && j.r0 >= 0 && j.r0 < j.nq * a.group;
}

// k_kv4_attn's jobs: where k_kv4_rows takes the sequences of more than KV4_FEW rows, each of the others
// has KV4_FEW / 16, whether it needs them or not. KV4_FEW by both kernels' times (k_kv4_attn / k_kv4_rows, us;
// 32 heads over 4 of 128, the same number of rows in every sequence):
//   rows              48         64         72         96         128
//   64 x 4096, bf16   99 / 121   122 / 122  148 / 128  174 / 150  224 / 113
//   64 x 4096, fp32   117 / 181  145 / 188  177 / 196  212 / 237  274 / 190
//   12 x 2048, bf16   26 / 32    30 / 34    34 / 35    39 / 37    46 / 37
//   1 x 4096, bf16    15 / 22    16 / 23    17 / 23    18 / 23    21 / 24
// 64 is where 16-bit batches change over; few or short sequences and fp32 would change over later, at about 96.
constexpr int KV4_FEW = 64;
__device__ __forceinline__ bool few_job(const Kv4Attn &a, int job, Job4 &j) {
  if (a.few == INT32_MAX) return job_of<16>(a, job, j);
  const int s = job / (KV4_FEW / 16);
  if (s >= a.n_seq) return false;
  j.s = s;
  j.q0 = min(max(a.q_start[s], 0), a.rows);
  j.nq = min(max(a.q_start[s + 1], 0), a.rows) - j.q0;
  j.r0 = job % (KV4_FEW / 16) * 16;
  j.n = (int)min((int64_t)max(a.kv_lens[s], 0), (int64_t)a.cols << a.page);
  const int rows = j.nq * a.group;
  return j.nq > 0 && rows <= a.few && j.r0 < rows;
}

__device__ __forceinline__ h2v bits_h2(uint32_t v) { return __builtin_bit_cast(h2v, v); }

// Constants held in registers: the instruction that masks and puts an exponent over the rest in one
// takes one constant from the scalar file and none from the instruction stream.
struct Const4 {
  uint32_t lo = 0x000f000fu, hi = 0x00f000f0u;  // scalar
  uint32_t e0 = 0x64006400u, e1 = 0x54005400u;  // vector: f16 1024 (ulp 1) and 64 (ulp 1/16)
};
__device__ __forceinline__ Const4 constants() {
  Const4 c;
  asm("" : "+s"(c.lo));
  asm("" : "+s"(c.hi));
  asm("" : "+v"(c.e0));
  asm("" : "+v"(c.e1));
  return c;
}
// Eight codes of a key word as eight f16 values, channels in order. EXACT: the integers code - 8.
// Otherwise the codes as subnormals, code * 2^-24 in elements 0, 1, 4, 5, code * 2^-20 in the others.
template <bool EXACT>
__device__ __forceinline__ h8v key_codes(uint32_t w, const Const4 &k) {
  const uint32_t w8 = w >> 8;
  if constexpr (EXACT) {
    const h2v o0 = {(_Float16)-1032.0f, (_Float16)-1032.0f}, o1 = {(_Float16)-72.0f, (_Float16)-72.0f};
    const h2v x[4] = {bits_h2((w & k.lo) | k.e0) + o0, bits_h2((w & k.hi) | k.e1) + o1, bits_h2((w8 & k.lo) | k.e0) + o0, bits_h2((w8 & k.hi) | k.e1) + o1};
    return __builtin_bit_cast(h8v, x);
  } else {
    const uint32_t x[4] = {w & k.lo, w & k.hi, w8 & k.lo, w8 & k.hi};
    return __builtin_bit_cast(h8v, x);
  }
}
// Byte b of the value words of two tokens as two channels' pairs of tokens: 1024 + code and 64 + code
// by an exponent put over the nibble, less what is too much, times the tokens' scales.
template <int HD>
__device__ __forceinline__ void value_pairs(uint32_t w0, uint32_t w1, int b, h2v d, const Const4 &k, h2v &even, h2v &odd) {
  const h2v o0 = {(_Float16)-1032.0f, (_Float16)-1032.0f}, o1 = {(_Float16)-72.0f, (_Float16)-72.0f};
  // HD 128: byte b of w0 and of w1; HD 64: both tokens' bytes lie in w0
  const uint32_t p = HD == 128 ? __builtin_amdgcn_perm(w1, w0, 0x0c040c00u + (uint32_t)b * 0x00010001u)
                               : __builtin_amdgcn_perm(w0, w0, 0x0c020c00u + (uint32_t)b * 0x00010001u);
  even = (bits_h2((p & k.lo) | k.e0) + o0) * d;
  odd = (bits_h2((p & k.hi) | k.e1) + o1) * d;
}
typedef float f2r __attribute__((ext_vector_type(2)));
// Two numbers as f16, and what that leaves of them.
__device__ __forceinline__ h2v half_pair(float a, float b) { return __builtin_convertvector((f2r{a, b}), h2v); }
__device__ __forceinline__ h2v half_rest(float a, float b, h2v top) { return half_pair(fmaf(-(float)top[0], 1.0f, a), fmaf(-(float)top[1], 1.0f, b)); }

// What a lane holds of a tile of 16 tokens: its token's key words, its four tokens' value words and
// scales.
template <int HD>
struct Tile4 {
  uint32_t k[HD / 32], v[HD / 32];
  h2v ks[4][HD / 64], vs[2];  // all groups' of a token; its channels' group's
};
template <int HD>
__device__ __forceinline__ void tile_load(Tile4<HD> &x, const uint8_t *tile, int lane) {
  constexpr int G = HD / 32;
  const int l = lane & 15, h = lane >> 4;
  const uint8_t *kc = tile + lane * 4 * G, *vc = kc + 8 * HD, *ks = tile + 16 * HD + h * 8 * G, *vs = tile + 17 * HD + ((l * G >> 4) * 16 + 4 * h) * 2;
  if constexpr (HD == 128) {
    const uint4 a = *(const uint4 *)kc, b = *(const uint4 *)vc, c = *(const uint4 *)ks, d = *(const uint4 *)(ks + 16);
    x.k[0] = a.x; x.k[1] = a.y; x.k[2] = a.z; x.k[3] = a.w;
    x.v[0] = b.x; x.v[1] = b.y; x.v[2] = b.z; x.v[3] = b.w;
    x.ks[0][0] = bits_h2(c.x); x.ks[0][1] = bits_h2(c.y); x.ks[1][0] = bits_h2(c.z); x.ks[1][1] = bits_h2(c.w);
    x.ks[2][0] = bits_h2(d.x); x.ks[2][1] = bits_h2(d.y); x.ks[3][0] = bits_h2(d.z); x.ks[3][1] = bits_h2(d.w);
  } else {
    const uint2 a = *(const uint2 *)kc, b = *(const uint2 *)vc;
    const uint4 c = *(const uint4 *)ks;
    x.k[0] = a.x; x.k[1] = a.y;
    x.v[0] = b.x; x.v[1] = b.y;
    x.ks[0][0] = bits_h2(c.x); x.ks[1][0] = bits_h2(c.y); x.ks[2][0] = bits_h2(c.z); x.ks[3][0] = bits_h2(c.w);
  }
  const uint2 c = *(const uint2 *)vs;
  x.vs[0] = bits_h2(c.x);
  x.vs[1] = bits_h2(c.y);
}

// The largest power of two that leaves |amax| at most 2^14 (1 for zero; at most 2^100). Zero for an
// infinity, which it makes a NaN: its scores would be infinities, of which a row that saw only -inf would
// look like one that sees nothing.
__device__ __forceinline__ float lift_of(float amax) {
  int e;
  (void)frexpf(amax, &e);
  const float lift = ldexpf(1.0f, min(max(14 - e, -126), 100));
  return amax == __builtin_inff() ? 0.0f : amax > 0.0f ? lift : 1.0f;
}

// What turns a sum of lifted queries and keys into an exponent, kept where it is a normal number and the
// sums (at most 2^14 * 2^16 * 128) times it stay finite. The limits change no result: sums are whole
// multiples of 2^-48, so that at 2^90 two that differ are further apart than any exponential's range, and
// at 2^-126 all are alike. (A lift of zero gives the upper limit: what is masked stays -inf.)
__device__ __forceinline__ float unlift_of(float scale, float lift) { return fminf(fmaxf(scale / lift, 0x1p-126f), 0x1p90f); }

// Long sequences are shared by workgroups: chunk blockIdx.z of `chunk` tokens (and every
// gridDim.z-th after it). A workgroup leaves its rows' (maximum, sum, output) for k_kv4_join where
// there is more than one chunk to them.
template <int HD, class R, int QP, int PP>
__global__ __launch_bounds__(256) void k_kv4_attn(const Kv4Attn a) {
  typedef typename R::E E;
  constexpr int G = HD / 32, NC = HD / 16, NW = 4;
  constexpr bool EXACT = QP == 2;
  __shared__ float so[NW][16][HD + 4], sm[NW][16], sl[NW][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, h = lane >> 4, head = blockIdx.y;
  Job4 j;
  if (!few_job(a, blockIdx.x, j)) return;
  const int rows = j.nq * a.group;
  const int r = j.r0 + l, tok = min(r, rows - 1) / a.group, g0 = min(r, rows - 1) % a.group;
  // the row's query, its scale and what it sees
  const E *qp = (const E *)a.q + (int64_t)(j.q0 + tok) * a.ld_q + (head * a.group + g0) * HD + 8 * h;
  float qv[G][8], amax = 0.0f;
#pragma unroll
  for (int g = 0; g < G; g++) {
    get8_if<R>(a.qvec, qp + 32 * g, qv[g]);
#pragma unroll
    for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(qv[g][i]));
  }
  amax = max32(max16(amax));
  const float lift = lift_of(amax), unlift = unlift_of(a.scale, lift) * (EXACT ? 1.0f : 16777216.0f);
  h8v qh[G], ql[G];
  f4v zero[G];  // where a group's sum starts
#pragma unroll
  for (int g = 0; g < G; g++) {
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float x = qv[g][i] * lift, down = !EXACT && i & 2 ? 0.0625f : 1.0f;
      const _Float16 top = (_Float16)x;
      const _Float16 low = (_Float16)(QP == 2 ? x - (float)top : 0.0f);
      all += (float)top + (float)low;
      qh[g][i] = (_Float16)((float)top * down);
      ql[g][i] = (_Float16)((float)low * down);
    }
    all = EXACT ? 0.0f : add32(add16(all)) * (-8.0f / 16777216.0f);
    zero[g] = f4v{all, all, all, all};
  }
  const int pos = j.n - j.nq + tok;
  const int hi = min(pos + 1, j.n), lo = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
  // all rows of the job together
  const int last = min(j.r0 + 15, rows - 1) / a.group, first = j.r0 / a.group;
  const int all_hi = min(j.n - j.nq + last + 1, j.n), all_lo = a.window > 0 ? max(j.n - j.nq + first + 1 - a.window, 0) : 0;
  const int from = all_lo & ~31, chunks = all_hi > from ? (all_hi - from + a.chunk - 1) / a.chunk : 1;
  if ((int)blockIdx.z >= chunks) return;

  f4v o[NC];
#pragma unroll
  for (int c = 0; c < NC; c++) o[c] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -__builtin_inff(), sum = 0.0f, ref = 0.0f;
  bool far = false;  // whether some lane's reference is past P_FAR
  const int *table = a.tables + (int64_t)j.s * a.cols;
  const int pm = (1 << a.page) - 1;

  // tokens that every row sees: tiles of them need no masks (a NaN there reaches every row)
  const int see_lo = a.window > 0 ? max(j.n - j.nq + last + 1 - a.window, 0) : 0, see_hi = min(j.n - j.nq + first + 1, j.n);

  const Const4 kc = constants();
  int base = 0, pages = -1;  // lane i holds the page id of entry base + i
  bool have = false;
  auto load = [&](Tile4<HD> *x, int t0) {  // which of the two tiles there are, as bits
    int in = 0;
    if (!have || ((t0 + 31) >> a.page) - base > 63) {
      have = true;
      base = t0 >> a.page;
      pages = table[min(base + lane, a.cols - 1)];
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int t = t0 + 16 * u;
      const int pg = t < all_hi ? lane_i(pages, (t >> a.page) - base) : -1;
      const bool ok = pg >= 0 && pg < a.n_pages;
      in |= (int)ok << u;
      tile_load<HD>(x[u], a.pool + tile_at<HD>(ok ? pg : 0, a.n_kv, head, a.page, ok ? t & pm : 0), lane);
    }
    return in;
  };
  auto step = [&](Tile4<HD> *x, int t0, int in, auto edge_) {
    constexpr bool edge = decltype(edge_)::value;
    float s[2][4], mt = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < 2; u++) {
      f4v acc[G];
#pragma unroll
      for (int g = 0; g < G; g++) {
        const h8v kf = key_codes<EXACT>(x[u].k[g], kc);
        acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[g], zero[g], 0, 0, 0);
        if (QP == 2) acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[g], acc[g], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float v = 0.0f;
#pragma unroll
        for (int g = 0; g < G; g++) v = fmaf((float)x[u].ks[i][g >> 1][g & 1], acc[g][i], v);
        const int t = t0 + 16 * u + 4 * h + i;
        s[u][i] = !edge || ((in >> u & 1) && t >= lo && t < hi) ? v : -__builtin_inff();
        mt = fmaxf(mt, s[u][i]);
      }
    }
    mt = max32(max16(mt));
    if (__builtin_amdgcn_ballot_w64((mt - m) * unlift > P_SLACK)) {  // (unlift is positive)
      const float mn = fmaxf(m, mt), f = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * unlift);
      m = mn;
      ref = p_ref(m * unlift);
      far = __builtin_amdgcn_ballot_w64(p_far(m * unlift)) != 0;
      sum *= f;
#pragma unroll
      for (int c = 0; c < NC; c++) o[c] *= f;
    }
    if (__builtin_expect(far, 0)) {
      const float off = p_far(m * unlift) ? m : 0.0f;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[u][i] -= off;
    }
    h2v p1[4], p2[4];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[u][i], unlift, ref)), y = __builtin_amdgcn_exp2f(fmaf(s[u][i + 1], unlift, ref));
        sum += x + y;
        p1[2 * u + i / 2] = half_pair(x, y);
        if (PP == 2) p2[2 * u + i / 2] = half_rest(x, y, p1[2 * u + i / 2]);
      }
    const h8v ph = __builtin_bit_cast(h8v, p1), pl = __builtin_bit_cast(h8v, p2);
    h2v vs[2][2] = {{x[0].vs[0], x[0].vs[1]}, {x[1].vs[0], x[1].vs[1]}};
    if (edge) {
      // values of tokens that no row may see count as zero (what lies there may be anything); a NaN
      // among the others reaches the rows that see its token and no others: which they are is a
      // product of 0s and 1s, and in the products below it counts as zero
      bool nan = false;
      h8v bad, sees;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int t = t0 + 16 * u + 4 * h + i;
          const _Float16 d = vs[u][i >> 1][i & 1];
          const bool is = (in >> u & 1) && t >= all_lo && t < all_hi, num = d == d;
          nan |= is && !num;
          bad[4 * u + i] = (_Float16)(is && !num ? 1.0f : 0.0f);
          sees[4 * u + i] = (_Float16)(s[u][i] == -__builtin_inff() ? 0.0f : 1.0f);
          vs[u][i >> 1][i & 1] = is && num ? d : (_Float16)0.0f;
        }
      if (__builtin_amdgcn_ballot_w64(nan)) {
        const f4v hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, sees, f4v{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[c][i] = hit[i] > 0.0f ? __builtin_nanf("") : o[c][i];
      }
    }
#pragma unroll
    for (int b = 0; b < NC / 2; b++) {
      h2v e[4], d[4];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          if constexpr (HD == 128) value_pairs<HD>(x[u].v[2 * i], x[u].v[2 * i + 1], b, vs[u][i], kc, e[2 * u + i], d[2 * u + i]);
          else value_pairs<HD>(x[u].v[i], 0u, b, vs[u][i], kc, e[2 * u + i], d[2 * u + i]);
        }
      const h8v ve = __builtin_bit_cast(h8v, e), vo = __builtin_bit_cast(h8v, d);
      o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ve, ph, o[2 * b], 0, 0, 0);
      o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vo, ph, o[2 * b + 1], 0, 0, 0);
      if (PP == 2) {
        o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ve, pl, o[2 * b], 0, 0, 0);
        o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vo, pl, o[2 * b + 1], 0, 0, 0);
      }
    }
  };
  for (int c = blockIdx.z; c < chunks; c += gridDim.z) {
    const int end = min(all_hi, from + (c + 1) * a.chunk);
    have = false;
    for (int t0 = from + c * a.chunk + 32 * wave; t0 < end; t0 += 32 * NW) {
      Tile4<HD> x[2];
      const int in = load(x, t0);
      if (in == 3 && t0 >= see_lo && t0 + 32 <= see_hi) step(x, t0, in, std::false_type{});
      else step(x, t0, in, std::true_type{});
    }
  }
  sum = add32(add16(sum));
  if (h == 0) { sm[wave][l] = m * unlift; sl[wave][l] = sum; }
  // row i of a lane's four is channels (4h + i) NC .. + NC - 1
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int c = 0; c < NC; c++) so[wave][l][(4 * h + i) * NC + c] = o[c][i];
  __syncthreads();
  // the waves' shares together: 16 threads a row
  const int row = threadIdx.x >> 4, part = threadIdx.x & 15;
  if (j.r0 + row >= rows) return;
  float mm = -__builtin_inff();
  for (int w = 0; w < NW; w++) mm = fmaxf(mm, sm[w][row]);
  float total = 0.0f, f[NW];
  for (int w = 0; w < NW; w++) {
    f[w] = sm[w][row] == mm ? 1.0f : __builtin_amdgcn_exp2f(sm[w][row] - mm);
    total += f[w] * sl[w][row];
  }
  const int rr = j.r0 + row;
  float v[NC];
#pragma unroll
  for (int c = 0; c < NC; c++) {
    v[c] = 0.0f;
    for (int w = 0; w < NW; w++) v[c] = fmaf(f[w], so[w][row][part * NC + c], v[c]);
  }
  if (min(chunks, (int)gridDim.z) == 1) {
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    E *dst = (E *)a.out + (int64_t)(j.q0 + rr / a.group) * a.ld_out + (head * a.group + rr % a.group) * HD + part * NC;
#pragma unroll
    for (int c = 0; c < NC; c++) v[c] *= inv;
    put_if<R, NC>(a.ovec, dst, v);
    return;
  }
  const int64_t at = (((int64_t)blockIdx.x * a.n_kv + head) * gridDim.z + blockIdx.z) * 16 + row;
  float *dst = a.part + at * HD + part * NC;
#pragma unroll
  for (int c = 0; c < NC; c += 4) *(float4 *)(dst + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
  if (part == 0) ((float2 *)(a.part + (int64_t)gridDim.x * a.n_kv * gridDim.z * 16 * HD))[at] = make_float2(mm, total);
}

// ------------------------------------------------------------------ attention of many rows
// Prompt chunks: a workgroup takes 128 rows of one sequence and key head, 32 a wave, and walks the
// tokens 64 at a time. Here the matrix cores have the work (4 * 128 operations a code and row), so
// codes become f16 values once for all four waves, in shared memory, while the 64 before them are
// worked on: wave w turns the w-th tile of 16 tokens. Products are v_mfma_f32_32x32x16_f16, whose
// left operand a wave reads once for 32 rows: S^T = K Q^T and O^T = V^T P^T as above, a lane's column
// being its row (lane % 32). Keys lie as [token][channel]; values as [channel][token] with bits 2 and 3
// of a token's number swapped, so that the eight tokens whose probabilities a lane has in a step lie
// together. 16-byte chunks of both are permuted by exclusive-or with row bits: a wave's reads and
// writes spread over all banks.
//
// Bound by the vector instructions beside the products: about 150 a block of 32 x 32 scores (a third
// of them conversions of codes, the rest maxima, exponentials and their rounding), where its products
// take 512 cycles. 2048 rows at 4096 tokens (32 heads over 4 of 128, bf16, 103 GFLOP) take 133 to
// 142 us by card, 725 to 775 TFLOP/s, where an 8192^3 product of the library reaches 1100. 32 rows a wave
// and two workgroups a CU, because 64 rows would leave one wave a SIMD, and 256 rows a workgroup no second
// one to even out what the rows of a prompt see.
//
// A group of 32 channels is one block of O^T, so a NaN group (written as zeros) can be given to the
// rows that see it afterwards: what was zeroed is kept as bits, 64 tokens a group.
typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int ROWS_BM = 128;

template <int HD>
struct alignas(256) Rows4 {  // a step's 64 tokens
  h8v k[64][HD / 8];  // [token][chunk ^ key_mix(token)]
  h8v v[HD][8];       // [channel][chunk ^ value_mix(channel)]
  uint32_t flag[4];   // of tile w: 1, a NaN group among its values; 2, it is not there
  unsigned long long nans[HD / 32];  // the tokens of NaN value groups
};

template <int HD>
__device__ __forceinline__ int key_mix(int t) { return HD == 128 ? t & 15 : t >> 1 & 7; }
__device__ __forceinline__ int value_mix(int ch) { return (ch >> 1 ^ ch >> 4) & 7; }

template <int HD, class R, int QP, int PP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void k_kv4_rows(const Kv4Attn a) {
  typedef typename R::E E;
  constexpr int G = HD / 32, KS = HD / 16, NC = HD / 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  Rows4<HD> *buf = (Rows4<HD> *)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  const RowsPlace place = rows_place(blockIdx.x, gridDim.x, a.n_kv);
  const int job = place.job, head = place.head;
  Job4 j;
  if (!job_of<ROWS_BM>(a, job, j)) return;
  const int rows = j.nq * a.group;
  if (rows <= a.few) return;  // k_kv4_attn's
  const int r = j.r0 + 32 * wave + col, rc = min(r, rows - 1), tok = rc / a.group;
  const E *qp = (const E *)a.q + (int64_t)(j.q0 + tok) * a.ld_q + (head * a.group + rc % a.group) * HD + 8 * h;
  float amax = 0.0f;
#pragma unroll
  for (int k = 0; k < KS; k++) {
    float x[8];
    get8_if<R>(a.qvec, qp + 16 * k, x);
#pragma unroll
    for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[i]));
  }
  amax = max32(amax);
  const float lift = lift_of(amax), unlift = unlift_of(a.scale, lift);
  h8v qh[KS], ql[KS];
#pragma unroll
  for (int k = 0; k < KS; k++) {
    float x[8];
    get8_if<R>(a.qvec, qp + 16 * k, x);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qh[k][i] = (_Float16)(x[i] * lift);
      if (QP == 2) ql[k][i] = (_Float16)(x[i] * lift - (float)qh[k][i]);
    }
  }
  const int pos = j.n - j.nq + tok, hi = min(pos + 1, j.n), lo = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
  const int last = min(j.r0 + ROWS_BM - 1, rows - 1) / a.group, first = j.r0 / a.group;
  const int all_hi = min(j.n - j.nq + last + 1, j.n), all_lo = a.window > 0 ? max(j.n - j.nq + first + 1 - a.window, 0) : 0;
  const int see_lo = a.window > 0 ? max(j.n - j.nq + last + 1 - a.window, 0) : 0, see_hi = min(j.n - j.nq + first + 1, j.n);
  const int from = all_lo & ~63, chunks = all_hi > from ? (all_hi - from + a.rchunk - 1) / a.rchunk : 1;
  if ((int)blockIdx.z >= chunks) return;
  const int *table = a.tables + (int64_t)j.s * a.cols;
  const int pm = (1 << a.page) - 1;

  f16v o[G];
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[g][i] = 0.0f;
  float m = -__builtin_inff(), sum = 0.0f;
  bool far = false;  // whether some lane's reference is past P_FAR

  // this wave's tile of the 64 tokens from t0
  const int l = lane & 15, hq = lane >> 4;
  uint32_t kw[G], vw[G];
  h2v ks[G / 2], vs[2];
  int in;                          // whether it is there
  int base = INT32_MIN, pages = -1;  // lane i holds the page id of entry base + i
  auto load = [&](int t0) {
    const int t = t0 + 16 * wave;
    int pg = -1;
    if (t < all_hi) {
      const int e = t >> a.page;
      if (base < 0 || e - base > 63) {
        base = e;
        pages = table[min(base + lane, a.cols - 1)];
      }
      pg = lane_i(pages, e - base);
    }
    in = pg >= 0 && pg < a.n_pages;
    const uint8_t *tile = a.pool + tile_at<HD>(in ? pg : 0, a.n_kv, head, a.page, in ? t & pm : 0);
    const uint8_t *kp = tile + lane * 4 * G, *vp = kp + 8 * HD;
    if constexpr (HD == 128) {
      const uint4 x = *(const uint4 *)kp, y = *(const uint4 *)vp;
      kw[0] = x.x; kw[1] = x.y; kw[2] = x.z; kw[3] = x.w;
      vw[0] = y.x; vw[1] = y.y; vw[2] = y.z; vw[3] = y.w;
      const uint2 z = *(const uint2 *)(tile + 16 * HD + l * 2 * G);
      ks[0] = bits_h2(z.x); ks[1] = bits_h2(z.y);
    } else {
      const uint2 x = *(const uint2 *)kp, y = *(const uint2 *)vp;
      kw[0] = x.x; kw[1] = x.y;
      vw[0] = y.x; vw[1] = y.y;
      ks[0] = bits_h2(*(const uint32_t *)(tile + 16 * HD + l * 2 * G));
    }
    const uint2 z = *(const uint2 *)(tile + 17 * HD + ((l * G >> 4) * 16 + 4 * hq) * 2);
    vs[0] = bits_h2(z.x); vs[1] = bits_h2(z.y);
  };
  const Const4 kc = constants();
  // Where not every row sees all of the 64 tokens, what no row sees or is not there counts as zero, and so
  // do NaN groups, which are marked. (Elsewhere a NaN reaches every row by itself.)
  uint32_t bad = 0, mark = 0;
  auto edge = [&](int t0) {
    bad = 0;
    mark = in ? 0 : 2;
    if (in && t0 >= see_lo && t0 + 64 <= see_hi) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int tt = t0 + 16 * wave + 4 * hq + i;
      const _Float16 d = vs[i >> 1][i & 1];
      const bool is = in && tt >= all_lo && tt < all_hi, num = d == d;
      if (is && !num) bad |= 1u << i;
      vs[i >> 1][i & 1] = is && num ? d : (_Float16)0.0f;
    }
    if (__builtin_amdgcn_ballot_w64(bad != 0)) mark |= 1;
  };
  auto store = [&](Rows4<HD> &b) {
    const h2v o0 = {(_Float16)-1032.0f, (_Float16)-1032.0f}, o1 = {(_Float16)-72.0f, (_Float16)-72.0f};
    const int t = 16 * wave + l;
#pragma unroll
    for (int g = 0; g < G; g++) {
      const _Float16 d1 = ks[g >> 1][g & 1];
      const h2v d = {d1, d1};
      const uint32_t w = kw[g], w8 = w >> 8;
      const h2v x[4] = {(bits_h2((w & kc.lo) | kc.e0) + o0) * d, (bits_h2((w & kc.hi) | kc.e1) + o1) * d,
                        (bits_h2((w8 & kc.lo) | kc.e0) + o0) * d, (bits_h2((w8 & kc.hi) | kc.e1) + o1) * d};
      b.k[t][(4 * g + hq) ^ key_mix<HD>(t)] = __builtin_bit_cast(h8v, x);
    }
    // four tokens of this lane's channels: 8 bytes of each channel's row
    const int chunk = 2 * wave + (hq & 1), half = hq >> 1;
#pragma unroll
    for (int c = 0; c < NC / 2; c++) {
      h2v e[2], d[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if constexpr (HD == 128) value_pairs<HD>(vw[2 * i], vw[2 * i + 1], c, vs[i], kc, e[i], d[i]);
        else value_pairs<HD>(vw[i], 0u, c, vs[i], kc, e[i], d[i]);
      }
#pragma unroll
      for (int p = 0; p < 2; p++) {
        const int ch = l * NC + 2 * c + p;
        const uint2 x = p ? make_uint2(__builtin_bit_cast(uint32_t, d[0]), __builtin_bit_cast(uint32_t, d[1]))
                          : make_uint2(__builtin_bit_cast(uint32_t, e[0]), __builtin_bit_cast(uint32_t, e[1]));
        ((uint2 *)&b.v[ch][chunk ^ value_mix(ch)])[half] = x;
      }
    }
    if (lane == 0) b.flag[wave] = mark;
    if (mark & 1) {  // (rare) the 16 tokens' bits of each group
      const int span = 16 / G;  // lanes of l that share a group
#pragma unroll
      for (int g = 0; g < G; g++) {
        uint32_t w = l == g * span ? bad << (4 * hq) : 0;
        w |= (uint32_t)__shfl_xor((int)w, 16);
        w |= (uint32_t)__shfl_xor((int)w, 32);
        if (lane == g * span) ((uint16_t *)&b.nans[g])[wave] = (uint16_t)w;
      }
    } else if (lane < G) {
      ((uint16_t *)&b.nans[lane])[wave] = 0;
    }
  };

  // NB blocks of 32 tokens at once: two let the matrix cores work on one block while the other's
  // probabilities are made, but do not fit the registers where queries have two parts
  constexpr int NB = QP == 2 ? 1 : 2;
  // A lane's chunks: the permutations leave what the step k, the block u and the group g add to a chunk's
  // number an exclusive-or as well, so one base serves them all.
  //   keys: (32 u + col) HD / 8 + (2 k + h ^ key_mix);   values: (32 g + col) 8 + (4 u + 2 k + h ^ value_mix ^ 2 g)
  const int kat = col * (HD / 8) + (h ^ key_mix<HD>(col)), vat = col * 8 + (h ^ value_mix(col));
  for (int c = blockIdx.z; c < chunks; c += gridDim.z) {
    const int begin = from + c * a.rchunk, end = min(all_hi, begin + a.rchunk);
    if (begin >= end) break;
    base = -1;
    load(begin);
    edge(begin);
    store(buf[0]);  // (a chunk before this one ended with a barrier)
    load(begin + 64);      // (tiles behind the last are not there)
    __syncthreads();
    int at = 0;
    for (int t0 = begin; t0 < end; t0 += 64, at ^= 1) {
      edge(t0 + 64);
      const Rows4<HD> &b = buf[at];
      const h8v *bk = &b.k[0][0], *bv = &b.v[0][0];
      const uint4 flag = *(const uint4 *)b.flag;
      const uint32_t gone = (flag.x >> 1) | (flag.y & 2) | (flag.z & 2) << 1 | (flag.w & 2) << 2;
      const bool masks = t0 < see_lo || t0 + 64 > see_hi || gone, nans = ((flag.x | flag.y | flag.z | flag.w) & 1) != 0;
#pragma unroll
      for (int u0 = 0; u0 < 2; u0 += NB) {
        f16v s[NB];
#pragma unroll
        for (int u = 0; u < NB; u++) {
#pragma unroll
          for (int i = 0; i < 16; i++) s[u][i] = 0.0f;
#pragma unroll
          for (int k = 0; k < KS; k++) {
            const h8v kf = bk[(kat ^ 2 * k) + (u0 + u) * 32 * (HD / 8)];
            s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[k], s[u], 0, 0, 0);
            if (QP == 2) s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[k], s[u], 0, 0, 0);
          }
        }
        if (u0 == 0) store(buf[at ^ 1]);  // the next tile's codes become values while the products run
        if (u0 == 0) load(t0 + 128);
        if (masks) {
#pragma unroll
          for (int u = 0; u < NB; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const int q = 32 * (u0 + u) + 8 * (i >> 2) + 4 * h + (i & 3), t = t0 + q;
              const bool hide = (bool)((int)(t < lo) | (int)(t >= hi) | (int)(gone >> (q >> 4) & 1));
              s[u][i] = hide ? -__builtin_inff() : s[u][i];
            }
        }
        float mt = s[0][0];
#pragma unroll
        for (int u = 0; u < NB; u++)
#pragma unroll
          for (int i = 0; i < 16; i++) mt = fmaxf(mt, s[u][i]);
        mt = max32(mt);
        if (__builtin_amdgcn_ballot_w64((mt - m) * unlift > P_SLACK)) {
          const float mn = fmaxf(m, mt), f = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * unlift);
          m = mn;
          far = __builtin_amdgcn_ballot_w64(p_far(m * unlift)) != 0;
          sum *= f;
#pragma unroll
          for (int g = 0; g < G; g++) o[g] *= f;
        }
        if (__builtin_expect(nans, 0)) {
#pragma unroll
          for (int u = 0; u < NB; u++)
#pragma unroll
            for (int g = 0; g < G; g++) {
              const uint32_t bits = (uint32_t)(b.nans[g] >> (32 * (u0 + u) + 4 * h));
              bool hit = false;
#pragma unroll
              for (int i = 0; i < 16; i++) hit |= (bits >> (8 * (i >> 2) + (i & 3)) & 1) && !(s[u][i] == -__builtin_inff());
              if (max32(hit ? 1.0f : 0.0f) > 0.0f)
#pragma unroll
                for (int i = 0; i < 16; i++) o[g][i] = __builtin_nanf("");
            }
        }
        float ref = m == -__builtin_inff() ? 0.0f : P_LIFT - m * unlift;  // (kept, it would cost a register too many)
        if (__builtin_expect(far, 0)) {
          const float off = p_far(m * unlift) ? m : 0.0f;
          ref = p_ref(m * unlift);
#pragma unroll
          for (int u = 0; u < NB; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[u][i] -= off;
        }
#pragma unroll
        for (int u = 0; u < NB; u++) {
          h2v p1[8], p2[8];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[u][i], unlift, ref)), y = __builtin_amdgcn_exp2f(fmaf(s[u][i + 1], unlift, ref));
            p1[i / 2] = half_pair(x, y);
            if (PP == 2) {
              p2[i / 2] = half_rest(x, y, p1[i / 2]);
              sum += x + y;
            } else {  // the sum of what the products take, two at a time
              sum = __builtin_amdgcn_fdot2(p1[i / 2], h2v{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
            }
          }
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const h2v q1[4] = {p1[4 * k], p1[4 * k + 1], p1[4 * k + 2], p1[4 * k + 3]}, q2[4] = {p2[4 * k], p2[4 * k + 1], p2[4 * k + 2], p2[4 * k + 3]};
            const h8v ph = __builtin_bit_cast(h8v, q1), pl = __builtin_bit_cast(h8v, q2);
#pragma unroll
            for (int g = 0; g < G; g++) {
              const h8v vf = bv[(vat ^ (2 * k ^ (2 * g & 7)) ^ 4 * (u0 + u)) + 256 * g];
              o[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, ph, o[g], 0, 0, 0);
              if (PP == 2) o[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl, o[g], 0, 0, 0);
            }
          }
        }
      }
      __syncthreads();
    }
  }
  sum = add32(sum);
  if (r >= rows) return;
  // element i of a block is channel 8 (i / 4) + 4 h + i % 4
  if (min(chunks, (int)gridDim.z) == 1) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    E *dst = (E *)a.out + (int64_t)(j.q0 + tok) * a.ld_out + (head * a.group + r % a.group) * HD + 4 * h;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float x[4] = {o[g][i] * inv, o[g][i + 1] * inv, o[g][i + 2] * inv, o[g][i + 3] * inv};
        put_if<R, 4>(a.ovec, dst + 32 * g + 2 * i, x);
      }
    return;
  }
  const int64_t row = (((int64_t)job * a.n_kv + head) * gridDim.z + blockIdx.z) * ROWS_BM + 32 * wave + col;
  float *dst = a.rpart + row * HD + 4 * h;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < 16; i += 4) *(float4 *)(dst + 32 * g + 2 * i) = make_float4(o[g][i], o[g][i + 1], o[g][i + 2], o[g][i + 3]);
  if (h == 0) ((float2 *)(a.rpart + (int64_t)gridDim.x * gridDim.z * ROWS_BM * HD))[row] = make_float2(m * unlift, sum);
}

// The chunks of a row together, a wave a row: sixteen lanes have a row's channels, each of the four
// quarters of the wave takes every fourth chunk. Workgroups below few_jobs * 4 have four of k_kv4_attn's
// rows, the others 16 of k_kv4_rows' (fewer workgroups where a job has no rows at all).
constexpr int JOIN_ROWS = 4;  // k_kv4_rows' rows a wave
template <int HD, class R>
__device__ __forceinline__ void join_row(const Kv4Attn &a, const Job4 &j, bool many, int job, int row, int splits, int jobs);

template <int HD, class R>
__global__ __launch_bounds__(256) void k_kv4_join(const Kv4Attn a, int few_jobs, int few_splits, int many_splits) {
  const bool many = (int)blockIdx.x >= few_jobs * 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Job4 j;
  if (many) {
    constexpr int PER = ROWS_BM / (4 * JOIN_ROWS);
    const int at = blockIdx.x - few_jobs * 4, job = at / PER, row = at % PER * (4 * JOIN_ROWS) + wave * JOIN_ROWS;
    if (many_splits == 1 || !job_of<ROWS_BM>(a, job, j) || j.nq * a.group <= a.few) return;
    for (int i = 0; i < JOIN_ROWS; i++) join_row<HD, R>(a, j, true, job, row + i, many_splits, (int)(gridDim.x - few_jobs * 4) / PER);
  } else {
    const int job = blockIdx.x / 4;
    if (few_splits == 1 || !few_job(a, job, j)) return;
    join_row<HD, R>(a, j, false, job, blockIdx.x % 4 * 4 + wave, few_splits, few_jobs);
  }
}

template <int HD, class R>
__device__ __forceinline__ void join_row(const Kv4Attn &a, const Job4 &j, bool many, int job, int row, int splits, int jobs) {
  typedef typename R::E E;
  constexpr int NC = HD / 16, U = 4;
  const int head = blockIdx.y, part = threadIdx.x & 15, quarter = threadIdx.x >> 4 & 3, bm = many ? ROWS_BM : 16;
  const int chunk = many ? a.rchunk : a.chunk, step = many ? 64 : 32;
  const int rows = j.nq * a.group, rr = j.r0 + row;
  if (rr >= rows) return;
  const int last = min(j.r0 + bm - 1, rows - 1) / a.group, first = j.r0 / a.group;
  const int all_hi = min(j.n - j.nq + last + 1, j.n), from = (a.window > 0 ? max(j.n - j.nq + first + 1 - a.window, 0) : 0) & -step;
  const int n = min(all_hi > from ? (all_hi - from + chunk - 1) / chunk : 1, splits);
  if (n == 1) return;
  const float *whole = many ? a.rpart : a.part;
  const int64_t at = ((int64_t)job * a.n_kv + head) * splits * bm + row;
  const float2 *ms = (const float2 *)(whole + (int64_t)jobs * a.n_kv * splits * bm * HD) + at;
  const float *src = whole + at * HD + part * NC;
  float m = -__builtin_inff(), total = 0.0f, v[NC] = {};
  for (int c0 = quarter; c0 < n; c0 += 4 * U) {  // U chunks' loads at a time
    float2 x[U];
    float4 y[U][NC / 4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = min(c0 + 4 * u, n - 1);
      x[u] = ms[(int64_t)c * bm];
#pragma unroll
      for (int i = 0; i < NC / 4; i++) y[u][i] = *(const float4 *)(src + (int64_t)c * bm * HD + 4 * i);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; u++) mn = fmaxf(mn, x[u].x);  // (a chunk twice does no harm here)
    const float f0 = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    total *= f0;
#pragma unroll
    for (int i = 0; i < NC; i++) v[i] *= f0;
    m = mn;
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (c0 + 4 * u >= n) continue;
      const float f = x[u].x == m ? 1.0f : __builtin_amdgcn_exp2f(x[u].x - m);
      total = fmaf(f, x[u].y, total);
#pragma unroll
      for (int i = 0; i < NC / 4; i++) {
        v[4 * i] = fmaf(f, y[u][i].x, v[4 * i]);
        v[4 * i + 1] = fmaf(f, y[u][i].y, v[4 * i + 1]);
        v[4 * i + 2] = fmaf(f, y[u][i].z, v[4 * i + 2]);
        v[4 * i + 3] = fmaf(f, y[u][i].w, v[4 * i + 3]);
      }
    }
  }
  const float mm = max32(max16(m)), f = m == mm ? 1.0f : __builtin_amdgcn_exp2f(m - mm);
  total = add32(add16(total * f));
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int i = 0; i < NC; i++) v[i] = add32(add16(v[i] * f)) * inv;
  if (quarter) return;
  E *dst = (E *)a.out + (int64_t)(j.q0 + rr / a.group) * a.ld_out + (head * a.group + rr % a.group) * HD + part * NC;
  put_if<R, NC>(a.ovec, dst, v);
}

// How the work is split: jobs (an odd number, so that neighbouring key heads and chunks of a sequence
// go to other XCDs: workgroups go around the eight of them in order), chunks of a sequence (at most)
// and tokens a chunk. Chunks are as long as leaves about `wgs` workgroups, a multiple of `step`.
//   KV4_WGS: 64 sequences of up to 16K (32 heads over 4) took 107 / 99 / 109 us with 4096 / 2048 / 1024
//   workgroups; where that makes chunks of less than 512 tokens (four tiles a wave), half of it, which is
//   what is resident at a time: a verify of 9 rows over twelve sequences of up to 2050 tokens (16 heads
//   over 8 of 64) 18 / 16 us with 2048 / 1024.
//   KV4_RWGS, k_kv4_rows': two a CU. Its chunks have KV4_RLEAST tokens at least, four steps: a launch
//   whose sequences all turn out to be k_kv4_attn's costs as many rounds of empty workgroups as it has
//   chunks (shared memory lets two of them onto a CU).
constexpr int KV4_WGS = 2048, KV4_RWGS = 512, KV4_RLEAST = 256;
struct Split4 { int64_t jobs; int splits, chunk; };
static Split4 split_of(int64_t jobs, int64_t busy, int64_t span, int wgs, int step, int least) {  // busy: jobs with rows, all key heads
  Split4 r;
  r.jobs = jobs | 1;
  auto chunk_for = [&](int64_t n) {
    const int64_t want = n > busy ? n / busy : 1;
    return std::max<int64_t>(((span + want - 1) / want + step - 1) / step * step, least);
  };
  int64_t chunk = chunk_for(wgs);
  if (wgs == KV4_WGS && chunk < 512) chunk = std::min<int64_t>(512, chunk_for(wgs / 2));
  chunk = std::min<int64_t>(chunk, 1 << 20);
  r.chunk = (int)chunk;
  r.splits = (int)std::max<int64_t>((span + chunk - 1) / chunk, 1);
  return r;
}
// The same under a window, of which a job of `tokens` new tokens walks no more than the window, those
// and a tile: shorter chunks, but no more of them than without (the scratch is for so many; a workgroup
// takes a second chunk where there are more).
static Split4 split_window(int64_t jobs, int64_t busy, int max_kv, int window, int tokens, int wgs, int step, int least) {
  Split4 all = split_of(jobs, busy, max_kv, wgs, step, least);
  if (window <= 0) return all;
  const Split4 r = split_of(jobs, busy, std::min<int64_t>(max_kv, (int64_t)window + tokens + 64), wgs, step, least);
  all.chunk = r.chunk;
  all.splits = std::min(all.splits, r.splits);
  return all;
}
// Both kernels' shares. Sequences with more rows than KV4_FEW rows (new tokens times query heads a
// key head) are k_kv4_rows'; where there are no more new tokens than sequences that launch is spared and
// k_kv4_attn takes all.
// A single sequence of that many rows is k_kv4_rows' alone, however many of them q_start leaves it:
// without the launches that would have nothing to do a 2048-row prompt takes 137 us instead of 139.
struct Plan4 { Split4 few, many; bool both, alone; int64_t few_floats, many_floats; };
static Plan4 plan_of(int hd, int group, int n_kv, int rows, int n_seq, int max_kv, int window) {
  Plan4 p{};
  const int64_t all = (int64_t)rows * group, each = (all + n_seq - 1) / n_seq;
  p.both = rows > n_seq && all > KV4_FEW;
  p.alone = p.both && n_seq == 1;
  if (p.alone) p.few = {0, 1, 128};
  else if (p.both) p.few = split_window((int64_t)n_seq * (KV4_FEW / 16), (each > 16 ? 2 : 1) * (int64_t)n_seq * n_kv, max_kv, window, 16 / group + 2, KV4_WGS, 128, 128);
  else p.few = split_window(all / 16 + n_seq, (each + 15) / 16 * n_seq * n_kv, max_kv, window, 16 / group + 2, KV4_WGS, 128, 128);
  if (p.few.splits > 1) p.few_floats = p.few.jobs * n_kv * p.few.splits * 16 * (hd + 2);
  if (p.both) {
    p.many = split_window(all / ROWS_BM + n_seq, (all / ROWS_BM + 1) * n_kv, max_kv, window, ROWS_BM / group + 2, KV4_RWGS, 64, KV4_RLEAST);
    if (p.many.splits > 1) p.many_floats = p.many.jobs * n_kv * p.many.splits * ROWS_BM * (hd + 2);
  }
  return p;
}
int64_t kv4_attention_ws(int hd, int group, int n_kv, int rows, int n_seq, int max_kv) {
  const Plan4 p = plan_of(hd, group, n_kv, rows, n_seq, max_kv, 0);
  return 4 * (p.few_floats + p.many_floats);
}

template <int HD, class R>
static hipError_t launch_attention(Kv4Attn &a, const Plan4 &p, hipStream_t s) {
  constexpr int QP = sizeof(typename R::E) == 4 ? 2 : 1, PP = std::is_same<R, RowBF16>::value ? 1 : 2;
  const unsigned nk = (unsigned)a.n_kv;
  a.few = p.alone ? 0 : p.both ? KV4_FEW : INT32_MAX;
  a.chunk = p.few.chunk;
  a.rchunk = p.many.chunk;
  a.rpart = a.part + p.few_floats;
  constexpr int ES = sizeof(typename R::E);
  a.qvec = (uintptr_t)a.q % 16 == 0 && a.ld_q * ES % 16 == 0;
  a.ovec = (uintptr_t)a.out % 16 == 0 && a.ld_out * ES % 16 == 0;
  if (!p.alone) hipLaunchKernelGGL((k_kv4_attn<HD, R, QP, PP>), dim3((unsigned)p.few.jobs, nk, p.few.splits), dim3(256), 0, s, a);
  if (p.both) {
    constexpr unsigned bytes = 2 * sizeof(Rows4<HD>);
    static std::atomic<uint64_t> set{0};  // devices on which the kernel has been allowed that much shared memory
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev > 63 || !(set.load() >> dev & 1)) {
      e = hipFuncSetAttribute((const void *)k_kv4_rows<HD, R, QP, PP>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
      if (e != hipSuccess) return e;
      if (dev < 64) set |= 1ull << dev;
    }
    hipLaunchKernelGGL((k_kv4_rows<HD, R, QP, PP>), dim3((unsigned)p.many.jobs * nk, 1, p.many.splits), dim3(256), bytes, s, a);
  }
  const unsigned f = p.few.splits > 1 ? (unsigned)p.few.jobs : 0, m = p.both && p.many.splits > 1 ? (unsigned)p.many.jobs : 0;
  if (f || m) hipLaunchKernelGGL((k_kv4_join<HD, R>), dim3(f * 4 + m * (ROWS_BM / (4 * JOIN_ROWS)), nk), dim3(256), 0, s, a, (int)f, p.few.splits, p.many.splits);
  return hipGetLastError();
}

hipError_t launch_kv4_attention(Kv4Attn a, int hd, int type, int max_kv, hipStream_t s) {
  const Plan4 p = plan_of(hd, a.group, a.n_kv, a.rows, a.n_seq, max_kv, a.window);
#define CALL(H, R) return launch_attention<H, R>(a, p, s)
  KV4_BY_TYPE(hd, type, CALL)
#undef CALL
}

}  // namespace spx
